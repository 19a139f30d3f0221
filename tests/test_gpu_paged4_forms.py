"""GPU checks of attention over pages of 4 bits in every form of its kernel of few rows
(paged4_variants, whose forms a test without a GPU checks)."""
import math

import pytest
import torch

from paged4_cases import Plain4, Run4
from paged4_variants import CALLS, MISSING, MISSING_WINDOWS, PAGE, STALE, UNSEEN, UNSEEN_WINDOWS
from test_gpu_paged import _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def _run(c, seed):
    """The call's sequences, appended in two steps; the batch of the second."""
    before, new = [n - m for n, m in zip(c.lengths, c.new)], list(c.new)
    run = Run4(c.kv_heads, c.d, PAGE, [before, new], seed=seed)
    run.append(before)
    return run, run.append(new)


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_attend(call):
    run, batch = _run(call, CALLS.index(call))
    print(call, flush=True)
    run.attend(call.heads, list(call.new), batch, window=call.window, sinks=call.sinks)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("heads,n,length,form", UNSEEN)
def test_unseen_rows_do_not_reach_a_row(heads, n, length, form, d, bad):
    """Infinities and NaN among keys and values that a row does not see: later positions of
    its own chunk, positions that the window has left, and stale ones past the length."""
    kv_heads, stale = 2, STALE
    k, v = (_rows(torch.Generator().manual_seed(d + n + i), length + stale, kv_heads, d) for i in (0, 1))
    rows = {0: 77, 1: length - 1000}  # one left by the windows, one at their edge; then the chunk's last
    k[rows[0], 0, 5] = v[rows[0], 0, 5] = bad
    v[rows[1], 1, 50] = bad
    k[length - 1, 0, d - 1] = v[length - 1, 1, d - 1] = bad
    k[length:], v[length:] = bad, bad
    run = Run4(kv_heads, d, PAGE, [[length + stale]])
    run.append([length + stale], k, v)
    run.lengths = [length]
    batch = run.batch([n])
    q = _rows(run.g, n, heads, d, std=1.5)
    pos = torch.arange(length - n, length)
    for window, sinks in UNSEEN_WINDOWS:
        got = run.cache.attend(q.cuda(), batch, scale=0.1, window=window, sinks=sinks)
        got = got.double().cpu().view(n, kv_heads, -1)
        kc, vc = k[:length].clone(), v[:length].clone()
        for head in (0, 1):
            for row in (rows[head], length - 1):
                kc[row, head], vc[row, head] = 0, 0
        clean = Plain4(torch.bfloat16, kv_heads, d, 1)
        clean.append(kc, vc, [length])
        ref, bound = (x.view(n, kv_heads, -1) for x in clean.attend(q, [n], 0.1, window, sinks))
        for head in (0, 1):
            sees = torch.zeros(n, dtype=torch.bool)
            for row in (rows[head], length - 1):
                sees |= (pos >= row) & ((pos - row < (window or math.inf)) | torch.tensor(row < sinks))
            assert ((got[:, head] - ref[:, head]).abs() <= bound[:, head])[~sees].all()
            assert not torch.isfinite(got[:, head][sees]).all(-1).any()


@pytest.mark.parametrize("heads,n,length,form", MISSING)
@pytest.mark.parametrize("d", [64, 96, 128])
def test_pages_missing_inside(heads, n, length, form, d):
    """Pages that are not there between pages that are, alone and as a step's every block."""
    run = Run4(2, d, PAGE, [[length - n], [n]])
    run.append([length - n])
    run.append([n])
    missing = [0, 3, 4, 7, 8, 9, 10, 13, 16]
    run.tables = [[-1 if i in missing else p for i, p in enumerate(run.tables[0])]]
    gone = [(0, PAGE * i, PAGE * i + PAGE) for i in missing]
    for window, sinks in MISSING_WINDOWS:
        run.attend(heads, [n], run.batch([n]), window=window, sinks=sinks, gone=gone)


def test_the_same_in_a_batch():
    """A sequence's rows do not depend on its neighbours, where the form is one."""
    run = Run4(2, 96, PAGE, [[1999, 1300, 801], [1, 1, 1]])
    run.append([1999, 1300, 801])
    run.append([1, 1, 1])
    q = _rows(run.g, 3, 8, 96, std=1.5)
    for window, sinks in ((None, 0), (1000, 70)):
        got = run.attend(8, [1, 1, 1], run.batch([1, 1, 1]), window=window, sinks=sinks, q=q)
        tables, lengths = run.tables, run.lengths
        for i in (0, 1):
            run.tables, run.lengths = [tables[i]], [lengths[i]]
            one = run.cache.attend(q[i:i + 1].cuda(), run.batch([1]), scale=96 ** -0.5, window=window,
                                   sinks=sinks)
            assert torch.equal(one, got[i:i + 1])
        run.tables, run.lengths = tables, lengths
