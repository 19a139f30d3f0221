"""GPU checks of token sampling (temperature, top-k, top-p, min-p by given
uniform numbers) against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def _draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, probability) of one row in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(x.argmax()), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    kept = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        kept = kept[:k]
    if p < 1:
        mass = np.cumsum(w[kept])
        before = np.concatenate(([0.0], mass[:-1]))
        kept = kept[(before < p * mass[-1]) | (np.arange(len(kept)) == 0)]
    kept = kept[w[kept] >= min(m, 1.0)]
    kept = np.sort(kept)
    reach = np.cumsum(w[kept])
    i = min(int(np.searchsorted(reach, u * reach[-1], side="right")), len(kept) - 1)
    return int(kept[i]), w[kept[i]] / reach[-1]


def _check(x, u, **kw):
    from parrot import hip_moe
    gpu = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    token, prob = hip_moe.sample(x.cuda(), u.cuda(), **gpu)
    assert token.shape == prob.shape == (*x.shape[:-1], 1) and token.dtype == torch.int64
    flat = x.reshape(-1, x.shape[-1]).double().numpy()
    names = {"t": "temperature", "k": "top_k", "p": "top_p", "m": "min_p"}
    for r in range(len(flat)):
        args = {a: (kw[n][r].item() if isinstance(kw[n], torch.Tensor) else kw[n])
                for a, n in names.items() if n in kw}
        want, share = _draw(flat[r], u.flatten()[r].double().item(), **args)
        assert token.flatten()[r].item() == want, (r, args)
        # one rounding to fp32 (2^-24), and weights rounded to 2^-41 of the largest
        # at 2^20 tokens, each share of the sum at most half of one off
        assert abs(prob.flatten()[r].item() - share) <= 2.0 ** -23 * share + 2.0 ** -30
    return token


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 1025, 4096, 4099, 9000, 16381, 20000, 30001, 32768,
                                   50001, 200000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sample(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    rows = 12
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    u = torch.rand(rows, generator=g)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
    print(f"sample {rows} x {vocab} {dtype}", flush=True)
    _check(x, u)
    _check(x, u, temperature=0.7, top_k=50, top_p=0.9)
    _check(x, u, temperature=pick([0.0, 0.3, 1.0, 2.0, 50.0]),
           top_k=pick([0, 1, 2, 40, 1000, vocab, 2 ** 31 - 1]).to(torch.int32),
           top_p=pick([1.0, 0.99, 0.9, 0.5, 1e-6, 0.0]), min_p=pick([0.0, 0.05, 0.3, 1.0]))


def test_ties():
    """Equal logits go by their index at every border."""
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-3, 4, (40, 5000), generator=g).float()
    u = torch.rand(40, generator=g)
    _check(x, u, temperature=0.0)
    for kw in ({"top_k": 1}, {"top_k": 700}, {"top_p": 0.3}, {"top_k": 900, "top_p": 0.5},
               {"top_k": 900, "top_p": 0.5, "min_p": 0.3}, {"min_p": 1.0}, {"top_p": 0.999}):
        _check(x, u, **kw)
    same = torch.zeros(8, 4097)
    _check(same, torch.rand(8, generator=g), top_k=333, top_p=0.7)
    _check(same, torch.rand(8, generator=g))


@pytest.mark.parametrize("vocab", [2000, 12002, 25001])
def test_ties_of_other_lengths(vocab):
    """As above, and fewer logits above -infinity than are asked for."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randint(-3, 4, (12, vocab), generator=g).float()
    x[3, 40:] = -math.inf
    x[4, :-40] = -math.inf
    u = torch.rand(12, generator=g)
    for kw in ({}, {"top_k": 700}, {"top_p": 0.3}, {"top_k": 900, "top_p": 0.5, "min_p": 0.3},
               {"top_p": 0.9999, "temperature": 0.02}, {"top_p": 0.999, "temperature": 100.0}):
        _check(x, u, **kw)


def test_borders_of_uniform():
    """u of 0 is the first kept token, the largest u below 1 the last."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3001, generator=g)
    for u in (0.0, 1 - 2.0 ** -24, 0.5, 2.0 ** -149):
        for kw in ({}, {"top_k": 5}, {"top_p": 0.8}):
            _check(x, torch.full((4,), u), **kw)


@pytest.mark.parametrize("vocab", [777, 3001, 6000, 12001, 20002, 29000, 40001])
def test_infinite_and_missing_logits(vocab):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, vocab, generator=g)
    x[0, ::2] = -math.inf
    x[1, ::3] = math.nan
    x[2, 5:] = -math.inf
    x[3] = -math.inf
    x[4] = math.nan
    x[5, [3, 100, 500]] = math.inf
    x[6] = torch.finfo(torch.float32).min
    x[7, 1:] = torch.finfo(torch.float32).min
    x[8] = x[8] * 1e37
    u = torch.rand(9, generator=g)
    for kw in ({}, {"top_k": 10}, {"top_p": 0.9}, {"temperature": 0.0}, {"min_p": 0.2},
               {"temperature": 0.01, "top_p": 0.5}, {"top_k": 400, "top_p": 0.99, "min_p": 0.01}):
        _check(x, u, **kw)


@pytest.mark.parametrize("vocab", [100, 1000, 3001, 6000, 12001, 29000, 40001])
@pytest.mark.parametrize("temperature", [1e-290, 1e-306, 1e-310, 5e-324])
def test_tiny_temperatures(vocab, temperature):
    """The smallest positive numbers: the largest logits alone are drawn from, alike."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, vocab, generator=g)
    x[1, [1, 50, 90]] = 9.0
    x[2] = 0.0
    x[2, ::2] = 2.0 ** -149
    x[3, [7, 80]] = math.inf
    u = torch.rand(4, generator=g)
    for kw in ({}, {"top_k": 2}, {"top_k": 600}, {"top_p": 0.4}, {"min_p": 1.0}):
        _check(x, u, temperature=temperature, **kw)


@pytest.mark.parametrize("vocab", [100, 1000, 3001, 6000, 12001, 29000, 40001])
def test_parameters_that_are_not_numbers(vocab):
    """As sample_torch has them: a NaN counts as no restriction, a temperature of 0, a
    uniform number of 0; at an infinite temperature every logit is alike, the largest
    and the smallest too."""
    from parrot import hip_moe
    from parrot.model import sample_torch
    g = torch.Generator().manual_seed(7)
    x = torch.randn(6, vocab, generator=g) * 4
    x[1, vocab // 2:] = -math.inf
    u = torch.rand(6, generator=g)
    nan, inf, one = (torch.full((6,), v) for v in (math.nan, math.inf, 1.0))
    # the largest numbers; infinities (which numpy's form above does not take at an
    # infinite temperature)
    ends = (torch.rand(6, vocab, generator=g) - 0.5) * 6.8e38
    cases = [(x, u, {"temperature": nan}), (x, u, {"temperature": inf}), (x, u, {"top_p": nan}),
             (x, u, {"min_p": nan, "top_k": 20}), (x, nan, {"top_k": 9}), (x, one, {"top_k": 9}),
             (x, u, {"temperature": inf, "top_k": 600, "top_p": 0.5})]
    for y in (ends, ends.nan_to_num()):
        cases += [(y, torch.rand(6, generator=g), {"temperature": math.inf, **kw})
                  for kw in ({}, {"top_k": 20}, {"top_p": 0.5})]
    for y, v, kw in cases:
        want = sample_torch(y, v, **kw)
        token, prob = hip_moe.sample(y.cuda(), v.cuda(), **{
            n: p.cuda() if isinstance(p, torch.Tensor) else p for n, p in kw.items()})
        assert torch.equal(token.cpu(), want[0]), kw
        assert ((prob.cpu() - want[1]).abs() <= 2.0 ** -23 * want[1] + 2.0 ** -30).all()


def test_numbers_below_zero():
    """A temperature below 0 takes the largest, a top_k below 0 is none, as numbers and
    as tensors."""
    g = torch.Generator().manual_seed(8)
    x, u = torch.randn(5, 3000, generator=g), torch.rand(5, generator=g)
    for t in (-0.5, -math.inf, torch.full((5,), -2.0)):
        _check(x, u, temperature=t)
    for k in (-1, -2 ** 31, torch.full((5,), -7, dtype=torch.int32)):
        _check(x, u, top_k=k)


@pytest.mark.parametrize("vocab", [5, 1500, 5000, 40000])
def test_uniform_numbers_outside_their_range(vocab):
    """Below 0 the first token that was kept, from 1 on the last."""
    from parrot import hip_moe
    x = torch.zeros(6, vocab)
    x[:, 1], x[:, 2], x[:, 3] = 5.0, 1.0, 6.0
    u = torch.tensor([-1.0, -math.inf, -0.0, 1.0, 2.0, math.inf])
    for kw in ({"top_k": 2}, {"min_p": 0.3}):
        token, _ = hip_moe.sample(x.cuda(), u.cuda(), **kw)
        assert token.flatten().tolist() == [1, 1, 1, 3, 3, 3]


def test_numbers_are_taken_in_64_bits():
    """0.1 of 40 equal weights is four of them; as fp32, in a tensor, a fifth."""
    x, u = torch.zeros(3, 40), torch.tensor([0.0, 0.5, 0.99])
    for p, kept in ((0.1, 4), (torch.full((3,), 0.1), 5)):
        token = _check(x, u, top_p=p)
        assert token.flatten().tolist() == [int(kept * v) for v in (0.0, 0.5, 0.99)]


def test_a_row_does_not_depend_on_the_others():
    from parrot import hip_moe
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(300, 32768, generator=g) * 0.55).cuda()
    u = torch.rand(300, generator=g).cuda()
    token, prob = hip_moe.sample(x, u, temperature=0.9, top_p=0.95)
    one, p1 = hip_moe.sample(x[17:18], u[17:18], temperature=0.9, top_p=0.95)
    assert torch.equal(token[17:18], one) and torch.equal(prob[17:18], p1)
    again, p2 = hip_moe.sample(x, u, temperature=0.9, top_p=0.95)
    assert torch.equal(token, again) and torch.equal(prob, p2)


def test_strides_shapes_and_out():
    from parrot import hip_moe
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 5, 700, generator=g)
    u = torch.rand(3, 5, generator=g)
    want = _check(x, u, top_k=30)
    wide = torch.randn(15, 1001, generator=g).cuda()
    wide[:, 3:703] = x.view(15, 700).cuda()
    assert torch.equal(hip_moe.sample(wide[:, 3:703], u.cuda().view(-1), top_k=30)[0].flatten(),
                       want.flatten())
    turned = x.view(15, 700).cuda().t().contiguous().t()
    assert torch.equal(hip_moe.sample(turned, u.cuda().view(-1), top_k=30)[0].flatten(),
                       want.flatten())
    out = torch.zeros(3, 5, dtype=torch.int64, device="cuda")
    got, _ = hip_moe.sample(x.cuda(), u.cuda(), top_k=30, out=out)
    assert torch.equal(out, want.view(3, 5)) and got.data_ptr() == out.data_ptr()
    assert hip_moe.sample(x[:0].cuda(), u[:0].cuda())[0].shape == (0, 5, 1)


def test_frequencies():
    """Shares of tokens over evenly spaced u are their probabilities."""
    from parrot import hip_moe
    x = torch.tensor([0.3, -1.0, 2.0, 0.5, 0.5, -3.0])
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    token, _ = hip_moe.sample(x.expand(n, 6).contiguous().cuda(), u.cuda())
    share = torch.bincount(token.flatten().cpu(), minlength=6) / n
    assert ((share - x.double().softmax(0)).abs() <= 1.0 / n).all()


def test_captured():
    from parrot import hip_moe
    g = torch.Generator().manual_seed(5)
    x, u = torch.empty(6, 32768, device="cuda"), torch.empty(6, device="cuda")
    x.zero_(), u.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        token, prob = hip_moe.sample(x, u, temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
    for _ in range(5):
        x.copy_(torch.randn(6, 32768, generator=g) * 2)
        u.copy_(torch.rand(6, generator=g))
        graph.replay()
        want, p = hip_moe.sample(x, u, temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
        assert torch.equal(token, want) and torch.equal(prob, p)
