"""GPU checks of the paged KV cache in 4 bits (append, read) and of attention over it
against plain forms in 64 bits (paged4_cases)."""
import math

import pytest
import torch

from paged4_cases import E2M1, Plain4, Run4, stored
from test_gpu_paged import _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------

# chunk edges inside a block, at its edge and past it; inside a byte's two positions; a
# sequence without new rows; single tokens; pages of one block and of several
@pytest.mark.parametrize("kv_heads,d,page,steps", [
    (2, 96, 64, [[1, 1], [1, 31], [1, 0], [1, 1]]),
    (1, 64, 32, [[33, 0, 95], [32, 5, 1], [0, 64, 33]]),
    (3, 128, 128, [[257], [1], [63], [64]]),
    (2, 96, 96, [[100, 96, 3, 29], [1, 1, 1, 3]]),
    (1, 64, 32, [[1]] * 40),
])
def test_append_and_read(kv_heads, d, page, steps):
    run = Run4(kv_heads, d, page, steps)
    for new in steps:
        print(f"append {new} after {run.lengths}", flush=True)
        batch = run.append(new)
    longest = max(run.lengths) + 5
    key, value = run.cache.read(batch, longest)
    assert key.shape == value.shape == (len(run.lengths), kv_heads, longest, d)
    for i, n in enumerate(run.lengths):
        for got, want in ((key[i], run.plain.k[i]), (value[i], run.plain.v[i])):
            assert torch.equal(got[:, :n].double().cpu(), want.transpose(0, 1))
            assert not got[:, n:].any()
    room = [torch.full((len(run.lengths), kv_heads, 2 * longest, d), 7.0, dtype=torch.bfloat16,
                       device="cuda") for _ in range(2)]
    run.cache.read(batch, 40, out=tuple(x[:, :, 3:43] for x in room))
    for x, y in zip(room, (key, value)):
        n = min(40, longest)
        assert torch.equal(x[:, :, 3:3 + n], y[:, :, :n])
        assert (x[:, :, :3] == 7).all() and (x[:, :, 43:] == 7).all()


def test_the_layout():
    """Where each value and byte lies."""
    d, page = 96, 64
    run = Run4(2, d, page, [[64]])
    batch = run.append([64])
    key, value = run.cache.read(batch, 64)
    at = run.tables[0][0]
    signs = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6])
    for pages, got, is_key in ((run.cache.key, key, True), (run.cache.value, value, False)):
        byte = pages.view(torch.uint8)[at].cpu()  # [heads, blocks, 16 d]
        code = torch.stack((byte % 16, byte // 16), -1).flatten(-2).view(2, 2, 4, 16, 2, d // 32, 8)
        for head, p, w in ((0, 0, 0), (1, 37, 95), (0, 21, 40), (1, 63, 17), (0, 14, 70), (1, 9, 33)):
            b, q = p // 32, p % 32
            if is_key:
                n, c, s, g, e = q // 16, q % 16, w // 32, w // 8 % 4, w % 8
                x = run.cache.key_exponent[at, head, b].view(16, 2, d // 32)[c, n, s]
                z = code[head, b, g, c, n, s, e]
            else:
                u, o, c, g, e = w // 32, w // 16 % 2, w % 16, q // 4 % 4, q // 16 * 4 + q % 4
                x = run.cache.value_exponent[at, head, p]
                z = code[head, b, g, c, o, u, e]
            assert signs[int(z)] * 2.0 ** (int(x) - 127) == got[0, head, p, w].item()


def test_append_leaves_the_rest():
    """Other positions, pages and rows of no sequence stay as they are; a page id
    outside the cache and positions past the table take nothing."""
    from parrot import PagedBatch, PagedKVCache
    for first in (0, 1, 30, 31):
        cache = PagedKVCache(6, 64, 2, 96, E2M1)
        g = torch.Generator().manual_seed(3)
        for x in (cache.key, cache.value):
            x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, generator=g))
        for x in (cache.key_exponent, cache.value_exponent):
            x.copy_(torch.randint(110, 140, x.shape, generator=g))
        k, v = _rows(g, 80, 2, 96), _rows(g, 80, 2, 96)
        # rows 0-2 nobody's, then 40 at first .. over pages 4 and 1, 20 on pages that are
        # not there, 7 of which 5 lie past the table; the rest nobody's
        batch = PagedBatch(i32([[4, 1], [-1, 6], [3, -1]]), i32([first + 40, 100, 133]),
                           i32([3, 43, 63, 70]))
        every = PagedBatch(i32([[0], [1], [2], [3], [4], [5]]), i32([64] * 6), i32([0] * 7))
        before = [x.view(torch.uint8).clone() for x in cache._tensors]
        whole = cache.read(every, 64)
        cache.append(k.cuda(), v.cuda(), batch)
        after = cache.read(every, 64)
        for x, y, rows, group in ((whole[0], after[0], k, 32), (whole[1], after[1], v, 96)):
            want = x.clone()
            new = stored(rows[3:43], group).transpose(0, 1).to(torch.bfloat16).cuda()
            n = 64 - first
            want[4, :, first:first + 40] = new[:, :n]
            want[1, :, :max(40 - n, 0)] = new[:, n:]
            assert torch.equal(y, want)
        there = [4, 1] if first + 40 > 64 else [4]
        for x, y in zip(before, cache._tensors):
            changed = (x != y.view(torch.uint8)).flatten(1).any(1)
            assert changed.nonzero()[:, 0].tolist() == sorted(there)


def test_rows_of_every_size():
    """Zeros, the smallest and largest numbers, halves of steps, single large values,
    groups of one row that differ, and rows that hold a NaN or an infinity."""
    d = 64
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(d), torch.full((d,), -0.0), torch.full((d,), 1e-40),
            torch.full((d,), 3.3e38), torch.linspace(-8, 8, d), torch.linspace(-7, 7, d),
            torch.arange(d) / 4.0, torch.arange(d) / 9.25, torch.arange(d) * 2.0 ** -120,
            2.0 ** torch.arange(-63.0, 1), torch.linspace(-3.3e38, 3.3e38, d),
            torch.cat((torch.randn(32, generator=g) * 1e-6, torch.randn(32, generator=g) * 1e6))]
    for p in range(-120, 121, 6):
        rows.append(torch.randn(d, generator=g).clamp(-3, 3) * 2.0 ** p)
    # just under and over where the power steps, and the rounding of what is near it
    for top in (6.0, 6.5, 6.96875, 7.0, 7.03125, 8.0, 3.5, 3.515625, 1.75, 1.7578125, 5.0, 2.5):
        x = torch.randn(d, generator=g) * 0.3 * top
        x = x.clamp(-top, top)
        x[7] = -top
        rows.append(x)
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.randn(d, generator=g)
        x[11] = bad
        rows.append(x)
    rows = torch.stack(rows).bfloat16()[:, None]
    run = Run4(1, d, 64, [[len(rows)]])
    batch = run.append([len(rows)], rows, rows.flip(0))
    for got, x, group in zip(run.cache.read(batch, len(rows)), (rows, rows.flip(0)), (32, d)):
        got, want = got[0, 0].double().cpu(), stored(x, group)[:, 0]
        assert torch.equal(got.isnan(), want.isnan()) and want.isnan().any()
        assert group == d or want[-1].isnan().sum() == 32
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_append_rope():
    """Rotated first, quantised then: as append of the rows that a cache in bf16 holds."""
    from parrot import PagedKVCache
    run = Run4(2, 96, 64, [[70, 33]])
    run.lengths = [70, 33]
    batch = run.batch([70, 33])
    k, v, q = (_rows(run.g, 103, h, 96).cuda() for h in (2, 2, 8))
    angle = torch.arange(128.0)[:, None] * 10000.0 ** (-torch.arange(0, 96, 2) / 96)
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    plain = PagedKVCache(run.cache.key.shape[0], 64, 2, 96)
    want = plain.append_rope(q, k, v, batch, cos, sin)
    assert torch.equal(run.cache.append_rope(q, k, v, batch, cos, sin), want)
    key, value = plain.read(batch, 70)
    for got, x, group in zip(run.cache.read(batch, 70), (key, value), (32, 96)):
        assert torch.equal(got.double(), stored(x, group))


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 96), (4, 4, 64), (12, 2, 128), (5, 1, 64), (16, 1, 128)])
@pytest.mark.parametrize("page,steps", [(64, [[1, 1, 0], [1, 1, 1]]), (32, [[33, 0, 95], [32, 5, 1], [0, 64, 33]]),
                                        (96, [[100, 96, 3], [1, 1, 3]]), (128, [[257, 600, 0], [1, 40, 7]])])
def test_append_rope_in_steps(heads, kv_heads, d, page, steps):
    """Chunks at every offset of a block, tables shorter than the positions, rows of a packed
    projection and rows of nobody: keys as append stores what a cache in bf16 rotated,
    values and queries as they are there."""
    from parrot import PagedBatch, PagedKVCache
    run = Run4(kv_heads, d, page, steps)
    plain = PagedKVCache(run.cache.key.shape[0], page, kv_heads, d)
    angle = torch.arange(300.0)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    for new in steps:
        run.lengths = [a + b for a, b in zip(run.lengths, new)]
        batch = run.batch(new)
        rows = sum(new)
        packed = _rows(run.g, rows + 4, heads + 2 * kv_heads, d).cuda()
        packed[rows:] = math.nan  # (nobody's)
        q, k, v = packed.split((heads, kv_heads, kv_heads), 1)
        print(f"{new} after {run.lengths}", flush=True)
        want = plain.append_rope(q, k, v, batch, cos, sin)
        got = run.cache.append_rope(q, k, v, batch, cos, sin)
        assert torch.equal(got[:rows], want[:rows])
        longest = max(run.lengths)
        key, value = plain.read(batch, longest)
        for got, x, group in zip(run.cache.read(batch, longest), (key, value), (32, d)):
            assert torch.equal(got.double(), stored(x, group))
    # into a captured graph, replayed for other rows
    new = [1] * len(run.lengths)
    batch = PagedBatch(batch.table, batch.lengths, i32(range(len(new) + 1)))
    q, k, v = (_rows(run.g, len(new), h, d).cuda() for h in (heads, kv_heads, kv_heads))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run.cache.append_rope(q, k, v, batch, cos, sin)
    for _ in range(3):
        for x in (q, k, v):
            x.copy_(_rows(run.g, *x.shape))
        graph.replay()
        assert torch.equal(out, plain.append_rope(q, k, v, batch, cos, sin))
        key, value = plain.read(batch, longest)
        for got, x, group in zip(run.cache.read(batch, longest), (key, value), (32, d)):
            assert torch.equal(got.double(), stored(x, group))
        torch.zeros(1 << 20, device="cuda").sum().item()  # eager work in between


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

LAYOUTS = [(8, 2, 96), (4, 4, 64), (6, 2, 128), (16, 1, 64), (5, 1, 96)]


@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("steps,window,sinks", [
    ([[1]], None, 0),                                   # a first token alone
    ([[31, 32, 33, 64], [1, 1, 1, 1]], None, 0),        # single tokens past block edges
    ([[200, 7, 0, 65], [3, 0, 9, 40]], 50, 0),          # ragged chunks, one sequence idle
    ([[300, 500], [1, 2]], 100, 5),                     # sinks far from the window
    ([[130, 97], [33, 64]], 40, 70),                    # more sinks than window
    ([[70]], 1, 0), ([[70]], 1, 33), ([[90]], 64, 30),  # one key; sinks that join the window
])
def test_attend(heads, kv_heads, d, steps, window, sinks):
    print(f"attend {heads}/{kv_heads} of {d}, {steps}, window {window} + {sinks}", flush=True)
    run = Run4(kv_heads, d, 64, steps, seed=len(steps) + d)
    for new in steps:
        batch = run.append(new)
        run.attend(heads, new, batch, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 16, 96), (16, 16, 64), (32, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 0), (70, 40), (1, 0)])
def test_attend_many_rows(heads, kv_heads, d, window, sinks):
    """Tiles of 128 rows: many sequences with ragged chunks after ragged contexts."""
    g = torch.Generator().manual_seed(d)
    first = torch.randint(0, 200, (24,), generator=g).tolist()
    then = torch.randint(40, 260, (24,), generator=g).tolist()
    then[3] = 0
    run = Run4(kv_heads, d, 64, [first, then])
    run.append(first)
    batch = run.append(then)
    run.attend(heads, then, batch, window=window, sinks=sinks)


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("steps,page,window,sinks", [
    ([[3000, 900], [1, 1]], 32, None, 0),       # long contexts, split over workgroups
    ([[3000, 900], [1, 6]], 256, 2048, 4),
    ([[1500], [200]], 96, None, 0),             # a chunk over a context
    ([[700, 333], [513, 260]], 64, 300, 40),    # hundreds of rows
])
def test_attend_long(d, steps, page, window, sinks):
    run = Run4(2, d, page, steps, seed=page)
    for new in steps:
        print(f"attend {new} after {run.lengths}", flush=True)
        batch = run.append(new)
        run.attend(8, new, batch, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,d", [(8, 64), (16, 96), (64, 128)])
@pytest.mark.parametrize("new,window,sinks", [([1, 1, 1, 1], None, 0), ([1, 1, 0, 1], 4064, 0),
                                              ([1, 1, 1, 1], 4032, 20)])
def test_attend_long_of_many_heads(heads, d, new, window, sinks):
    """Splits of as many keys as eight wavefronts take, beside sequences that need none."""
    run = Run4(8, d, 64, [[4130, 700, 4099, 0], new])
    for now in ([4130, 700, 4099, 0], new):
        batch = run.append(now)
    run.attend(heads, new, batch, window=window, sinks=sinks)


def test_attend_scales_and_strides():
    """Negative and large scales; rows of a packed projection, strides that the kernels do
    not read in place, an offset that is not aligned."""
    run = Run4(2, 64, 32, [[77, 40]])
    packed = _rows(run.g, 117, 10, 64).cuda()
    run.lengths = [77, 40]
    batch = run.batch([77, 40])
    run.cache.append(packed[:, 6:8], packed[:, 8:], batch)
    run.plain.append(packed[:, 6:8].cpu(), packed[:, 8:].cpu(), [77, 40])
    for scale in (0.125, -0.125, 3.0, 1e-3):
        q = packed[:, :6]
        got = run.cache.attend(q, batch, scale=scale)
        ref, bound = run.plain.attend(q.cpu(), [77, 40], scale)
        assert ((got.double().cpu() - ref).abs() <= bound).all()
        for other in (q.contiguous(), q.transpose(0, 1).contiguous().transpose(0, 1),
                      torch.empty(117 * 384 + 1, dtype=q.dtype, device="cuda")[1:]
                      .view(117, 6, 64).copy_(q)):
            assert torch.equal(run.cache.attend(other, batch, scale=scale), got)


@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (73, 1), (73, 128)])
def test_rows_without_keys(n, copies):
    """More new rows than positions, lengths of zero, pages that are not there: 0 where a
    row sees nothing, and rows of no sequence left as they are."""
    from parrot import PagedBatch
    run = Run4(2, 96, 32, [[64]])
    run.append([64])
    rows = 3 * n * copies
    q = _rows(run.g, rows + 5, 8, 96).cuda()
    table = [run.tables[0], [9999, -7], run.tables[0]] * copies
    starts = i32(range(0, rows + 1, n))
    for length in (0, 4):
        for kw in ({}, {"window": 8, "sinks": 1}):
            out = torch.full((rows + 5, 768), 3.0, dtype=torch.bfloat16, device="cuda")
            batch = PagedBatch(i32(table), i32([length, 50, 0] * copies), starts)
            run.cache.attend(q, batch, scale=0.125, out=out, **kw)
            assert (out[rows:] == 3).all()
            y = out[:rows].view(copies, 3, n, 768)
            assert not y[:, 1:].any() and not y[:, 0, :max(n - length, 0)].any()
            some = min(n, length)
            if some == 0:
                continue
            part = Plain4(torch.bfloat16, 2, 96, 1)
            part.k, part.v = [run.plain.k[0][:length]], [run.plain.v[0][:length]]
            for i in (0, copies - 1):
                at = (3 * i + 1) * n
                ref, bound = part.attend(q[at - some:at].cpu(), [some], 0.125, kw.get("window"),
                                         kw.get("sinks", 0))
                assert ((y[i, 0, n - some:].double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("n,copies", [(1, 1), (2, 1), (6, 1), (75, 1), (75, 40), (1, 100)])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_a_cache_without_pages(d, n, copies):
    """Nothing is stored, so nothing is read: 0 everywhere."""
    from parrot import PagedBatch, PagedKVCache
    cache = PagedKVCache(0, 32, 2, d, E2M1)
    b = copies
    batch = PagedBatch(i32([[0, -1, 5, 2 ** 31 - 1] * 20] * b), i32([1200 + n] * b),
                       i32(range(0, n * b + 1, n)))
    rows = torch.ones(n * b, 12, d, dtype=torch.bfloat16, device="cuda")
    cache.append(rows[:, :2], rows[:, 2:4], batch)
    assert not cache.attend(rows[:, 4:], batch, scale=0.1).any()
    assert not any(x.any() for x in cache.read(batch, 70))


@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (75, 1), (75, 40)])
def test_pages_missing_inside(n, copies):
    """Pages that are not there between pages that are: their positions are not seen, in
    tiles of 16, 32 and 128 rows."""
    run = Run4(2, 96, 32, [[900], [n]])
    run.append([900])
    run.append([n])
    missing = [3, 6, 7, 12, 13, 14, 20, 25]
    run.tables = [[-1 if i in missing else p for i, p in enumerate(run.tables[0])]]
    gone = [(0, 32 * i, 32 * i + 32) for i in missing]
    q = _rows(run.g, n, 8, 96)
    for window in (None, 300):
        ref, bound = run.plain.attend(q, [n], 96 ** -0.5, window, 40, gone)
        run.tables, run.lengths = run.tables * copies, run.lengths * copies
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), run.batch([n] * copies),
                               scale=96 ** -0.5, window=window, sinks=40)
        run.tables, run.lengths = run.tables[:1], run.lengths[:1]
        got = got.double().cpu().view(copies, n, -1)
        assert torch.equal(got, got[:1].expand_as(got))
        assert ((got[0] - ref).abs() <= bound).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("last", [73, 100, 110, 118, 150])
@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (15, 1), (73, 1), (73, 128)])
def test_unseen_rows_do_not_reach_a_row(bad, last, n, copies):
    """Infinities and NaN among keys and values that a row does not see: later positions
    of its own chunk, positions the window has left, and stale ones past the length."""
    run = Run4(2, 96, 64, [[150]])
    k, v = _rows(run.g, 150, 2, 96), _rows(run.g, 150, 2, 96)
    k[77, 0, 5] = v[77, 0, 5] = bad
    v[101, 1, 50] = bad
    run.append([150], k, v)
    run.lengths = [last]
    run.tables, run.lengths = run.tables * copies, run.lengths * copies
    batch = run.batch([n] * copies)
    q = _rows(run.g, n, 8, 96, std=1.5)
    for window, sinks in ((20, 0), (20, 3), (None, 0)):
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), batch, scale=0.1, window=window,
                               sinks=sinks).view(copies, n, 2, 4, 96)
        assert torch.equal(got.view(torch.int16), got[:1].view(torch.int16).expand_as(got))
        got = got[0].double().cpu()
        kc, vc = k[:last].clone(), v[:last].clone()
        for head, row in ((0, 77), (1, 101)):
            if row < last:
                kc[row, head], vc[row, head] = 0 if row == 77 else kc[row, head], 0
        clean = Plain4(torch.bfloat16, 2, 96, 1)
        clean.append(kc, vc, [last])
        ref, bound = clean.attend(q, [n], 0.1, window, sinks)
        ref, bound = ref.view(n, 2, 4, 96), bound.view(n, 2, 4, 96)
        pos = torch.arange(last - n, last)
        for head, row in ((0, 77), (1, 101)):
            sees = (pos >= row) & (pos < row + (window or last))
            assert ((got[:, head] - ref[:, head]).abs() <= bound[:, head])[~sees].all()
            assert not torch.isfinite(got[:, head][sees]).all(-1).any()


@pytest.mark.parametrize("n,copies", [(1, 1), (15, 1), (73, 1), (73, 128)])
def test_largest_rows(n, copies):
    """Keys and values up to the largest bf16 numbers, zeros among them: scores by queries
    as small, values where a row sees one key."""
    run = Run4(2, 64, 32, [[150]])
    g = run.g
    large = torch.randint(-3, 4, (150, 2, 64), generator=g) / 3 * 3.3e38
    large[::3] = torch.randint(-2, 3, (50, 2, 64), generator=g) * 2.0 ** 126
    large[1::5] = torch.randint(-1, 2, (30, 2, 64), generator=g) * 2.0 ** 127
    large, usual = large.bfloat16(), _rows(g, 150, 2, 64)
    q = (torch.randint(-3, 4, (n, 8, 64), generator=g) * 2.0 ** -125).bfloat16()
    for k, v, kw in ((large, usual, {}), (large, usual, {"window": 40, "sinks": 3}),
                     (usual, large, {"window": 1}), (large, large, {"window": 1})):
        run.lengths = [0]
        run.plain = Plain4(torch.bfloat16, 2, 64, 1)
        run.append([150], k, v)
        lengths, tables = run.lengths, run.tables
        run.tables, run.lengths = tables * copies, lengths * copies
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), run.batch([n] * copies), scale=0.1,
                               **kw).view(copies, n, -1)
        run.tables, run.lengths = tables, lengths
        assert torch.equal(got, got[:1].expand_as(got))
        ref, bound = run.plain.attend(q, [n], 0.1, kw.get("window"), kw.get("sinks", 0))
        assert ((got[0].double().cpu() - ref).abs() <= bound).all(), kw


@pytest.mark.parametrize("new", [5, 40, 2000])
@pytest.mark.parametrize("window,sinks", [(1000, 0), (1000, 5), (300, 0), (None, 0)])
def test_tables_shorter_than_the_lengths(new, window, sinks):
    """Positions past the table are not stored: no row sees them, and the last rows'
    window may hold nothing else."""
    run = Run4(2, 96, 64, [[3200]])
    run.append([3200])
    run.tables = [run.tables[0][:32]]
    run.attend(8, [new], run.batch([new]), window=window, sinks=sinks, gone=[(0, 2048, 3200)])


def test_far_pages():
    """Pages past 2^31 and 2^32 values and bytes."""
    from parrot import PagedBatch, PagedKVCache
    page, d = 128, 128
    pages = (1 << 33) // (2 * page * d) + 300
    cache = PagedKVCache(pages, page, 2, d, E2M1)
    g = torch.Generator().manual_seed(1)
    k, v, q = _rows(g, 300, 2, d), _rows(g, 300, 2, d), _rows(g, 300, 4, d)
    batch = PagedBatch.from_lists([[pages - 1, 0, pages // 2]], [300], [300])
    cache.append(k.cuda(), v.cuda(), batch)
    plain = Plain4(torch.bfloat16, 2, d, 1)
    plain.append(k, v, [300])
    for n in (1, 12, 300):
        one = PagedBatch(batch.table, batch.lengths, i32([0, n]))
        got = cache.attend(q[:n].cuda(), one, scale=0.1)
        ref, bound = plain.attend(q[:n], [n], 0.1)
        assert ((got.double().cpu() - ref).abs() <= bound).all()
    key, value = cache.read(batch, 300)
    assert torch.equal(key[0].double().cpu(), plain.k[0].transpose(0, 1))
    assert torch.equal(value[0].double().cpu(), plain.v[0].transpose(0, 1))
    del cache
    torch.cuda.empty_cache()


def test_shared_pages():
    """Sequences that begin with the same pages."""
    run = Run4(2, 64, 32, [[160, 0, 0], [1, 7, 100]])
    run.append([160, 0, 0])
    run.tables = [run.tables[0], *(run.tables[0][:5] + t for t in run.tables[1:])]
    run.lengths = [160] * 3
    for x in (run.plain.k, run.plain.v):
        x[1:] = [x[0], x[0]]
    for new in ([1, 7, 0], [0, 0, 100]):
        batch = run.append(new)
        run.attend(8, new, batch, window=120, sinks=33)
    key, _ = run.cache.read(batch, 160)
    assert torch.equal(key[0], key[1]) and torch.equal(key[0], key[2])


@pytest.mark.parametrize("heads,kv_heads,others,new,length", [
    (8, 2, 400, 1, 8400), (16, 2, 260, 6, 8400), (32, 32, 31, 128, 3000)])
def test_shares_of_many_blocks(heads, kv_heads, others, new, length):
    """One long sequence among so many that no tile's keys are split."""
    steps = [[length] + [0] * others, [new] * (others + 1)]
    run = Run4(kv_heads, 64, 32, steps)
    for now in steps:
        batch = run.append(now)
    run.attend(heads, steps[-1], batch)


def test_a_cache_takes_its_own_memory_only():
    from parrot import PagedKVCache
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    cache = PagedKVCache(4096, 64, 2, 128, E2M1)
    size = sum(x.numel() * x.element_size() for x in cache._tensors)
    assert size == 4096 * 64 * 2 * (64 + 64 + 4 + 1)
    assert torch.cuda.max_memory_allocated() - before <= size + 4096
    assert not cache.key.view(torch.uint8).any() and not cache.value.view(torch.uint8).any()


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------

def test_captured_steps_on_a_stream():
    """Append and attention captured once, replayed for growing sequences: every replay as
    the eager calls."""
    from parrot import PagedBatch
    run = Run4(2, 96, 64, [[600, 90]] + [[1, 1]] * 12)
    run.append([600, 90])
    k, v, q = (torch.zeros(2, h, 96, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 8))
    lengths = i32(run.lengths)
    batch = PagedBatch(run.batch([1, 1]).table, lengths, i32([0, 1, 2]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        lengths.add_(1)
        run.cache.append(k, v, batch)
        out = run.cache.attend(q, batch, scale=0.1, window=400, sinks=8)
    side = torch.cuda.Stream()
    for i in range(10):
        new = [_rows(run.g, 2, h, 96) for h in (2, 2, 8)]
        with torch.cuda.stream(side):
            for x, y in zip((k, v, q), new):
                x.copy_(y)
            graph.replay()
        side.synchronize()
        run.plain.append(*new[:2], [1, 1])
        run.lengths = [n + 1 for n in run.lengths]
        ref, bound = run.plain.attend(new[2], [1, 1], 0.1, 400, 8)
        assert ((out.double().cpu() - ref).abs() <= bound).all(), i
        assert torch.equal(out, run.cache.attend(new[2].cuda(), run.batch([1, 1]), scale=0.1,
                                                 window=400, sinks=8))
        torch.zeros(1 << 20, device="cuda").sum().item()  # eager work in between


def test_two_streams():
    """The same cache read from two streams at once gives what one stream gives."""
    run = Run4(2, 96, 64, [[2500, 1800], [1, 1]])
    run.append([2500, 1800])
    batch = run.append([1, 1])
    qs = [_rows(run.g, 2, 8, 96).cuda() for _ in range(2)]
    want = [run.cache.attend(q, batch, scale=0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(run.cache.attend(q, batch, scale=0.1))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


def test_a_layer_over_four_bits():
    """LocalGQA.extend over pages of 4 bits is its projections around the cache's calls."""
    from parrot import ModelConfig, PagedBatch, PagedKVCache, hip_moe
    from parrot.model import LocalGQA, _rope_tables
    cfg = ModelConfig(moe_backend="grouped_hip", depth_backend="hip", collect_router_stats=False)
    torch.manual_seed(0)
    layer = LocalGQA(cfg).cuda().bfloat16().eval()
    x = torch.randn(40, cfg.dim, device="cuda", dtype=torch.bfloat16)
    batch = PagedBatch.from_lists([[1], [0]], [25, 15], [25, 15])
    caches = [PagedKVCache(2, 32, 2, 96, E2M1) for _ in range(2)]
    y = layer.extend(x, caches[0], batch, sinks=2)
    heads = (cfg.n_heads, cfg.n_kv_heads, cfg.n_kv_heads)
    qkv = hip_moe.proj(x, layer._qkv_fragments(), sum(heads) * 96).view(40, sum(heads), 96)
    cos, sin = _rope_tables(cfg, x.new_empty(0, dtype=torch.float32))
    q = caches[1].append_rope(*qkv.split(heads, 1), batch, cos, sin)
    a = caches[1].attend(q, batch, scale=96 ** -0.5, window=cfg.window_size, sinks=2)
    assert torch.equal(y, layer._project_out(a, None)) and y.any()
