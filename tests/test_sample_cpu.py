"""Sampling on the pytorch backend against the definition written out in numpy, and
generation that draws its tokens (no GPU)."""
import math

import numpy as np
import pytest
import torch

from conftest import tiny_model_config


def _draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
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
    kept = np.sort(kept[w[kept] >= min(m, 1.0)])
    reach = np.cumsum(w[kept])
    i = min(int(np.searchsorted(reach, u * reach[-1], side="right")), len(kept) - 1)
    return int(kept[i]), w[kept[i]] / reach[-1]


def test_sample_torch():
    from parrot.model import sample_torch
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 300, generator=g) * 3
    x[3, ::2] = -math.inf
    x[4] = -math.inf
    x[5, ::3] = math.nan
    x[6] = torch.randint(0, 3, (300,), generator=g).float()
    x[7, [4, 9]] = math.inf
    u = torch.rand(40, generator=g)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (40,), generator=g)]  # noqa: E731
    for kw in (dict(), dict(temperature=0.5, top_k=7, top_p=0.8, min_p=0.05),
               dict(temperature=pick([0.0, 0.7, 2.0]), top_k=pick([0, 1, 5, 500]).int(),
                    top_p=pick([1.0, 0.9, 0.0]), min_p=pick([0.0, 0.1, 1.0]))):
        token, prob = sample_torch(x, u, **kw)
        for r in range(40):
            value = lambda n, v: (  # noqa: E731
                kw[n][r].item() if isinstance(kw.get(n), torch.Tensor) else kw.get(n, v))
            args = dict(t=value("temperature", 1.0), k=value("top_k", 0), p=value("top_p", 1.0),
                        m=value("min_p", 0.0))
            want, share = _draw(x[r].numpy(), u[r].double().item(), **args)
            assert token[r].item() == want, (r, args)
            assert abs(prob[r].item() - share) <= 1e-6


def test_parameters_that_are_not_numbers():
    """A NaN counts as no restriction, a temperature of 0, a uniform number of 0; an
    infinite temperature makes every logit alike; a uniform number of 1 is the last
    that was kept."""
    from parrot.model import sample_torch
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 200, generator=g) * 4
    x[:, 150:] = -math.inf
    u = torch.rand(6, generator=g)
    nan, inf = torch.full((6,), math.nan), torch.full((6,), math.inf)
    for kw, same in (({"temperature": nan}, {"temperature": 0.0}), ({"top_p": nan}, {"top_p": 1.0}),
                     ({"min_p": nan, "top_k": 20}, {"min_p": 0.0, "top_k": 20})):
        for got, want in zip(sample_torch(x, u, **kw), sample_torch(x, u, **same)):
            assert torch.equal(got, want), kw
    for got, want in zip(sample_torch(x, nan, top_k=9), sample_torch(x, 0 * u, top_k=9)):
        assert torch.equal(got, want)
    token, prob = sample_torch(x, u, temperature=inf)
    assert torch.equal(token[:, 0], (u.double() * 150).floor().long())
    assert torch.equal(prob, torch.full((6, 1), 1 / 150))
    token, _ = sample_torch(x, torch.ones(6), top_k=9)
    assert torch.equal(token[:, 0], x.topk(9).indices.amax(-1))


def test_decode_sample_on_the_pytorch_backend():
    from parrot import Parrot
    from parrot.model import sample_torch
    torch.manual_seed(0)
    model = Parrot(tiny_model_config()).eval()
    ids = torch.randint(0, model.config.vocab_size, (2, 9))
    u = torch.rand(5, 2)
    _, state = model.prefill(ids)
    _, other = model.prefill(ids)
    token = ids[:, -1:]
    for i in range(5):
        logits, other = model.decode_step(token, other)
        want = sample_torch(logits[:, -1], u[i], temperature=0.8, top_k=10, top_p=0.9)[0]
        token, state = model.decode_sample(token, state, u[i], temperature=0.8, top_k=10,
                                           top_p=0.9)
        assert token.shape == (2, 1) and torch.equal(token, want)
    greedy, _ = model.decode_sample(token, state, u[0], temperature=0.0)
    best, _ = model.decode_next(token, other)
    assert torch.equal(greedy, best)


def test_hip_sample_refuses_cpu_tensors():
    from parrot import hip_moe
    with torch.no_grad(), pytest.raises(RuntimeError):
        hip_moe.sample(torch.zeros(2, 5), torch.zeros(2))


def test_sample_parameters():
    """A temperature of 0 or less and a top_k of 0 or less are numbers like any other, as
    in a tensor and on the pytorch backend."""
    from parrot import hip_moe
    from parrot.model import sample_torch

    def sample(**kw):  # as far as its arguments' checks, which come before the launch
        parameter, given = hip_moe._sample_parameter, {}
        with pytest.MonkeyPatch.context() as patch, torch.no_grad():
            patch.setattr(hip_moe, "_require", lambda *_: None)
            patch.setattr(hip_moe, "_on", lambda _: (_ for _ in ()).throw(InterruptedError))
            patch.setattr(hip_moe, "_sample_parameter", lambda x, what, *a: given.setdefault(
                what, parameter(x, what, *a)))
            with pytest.raises(InterruptedError):
                hip_moe.sample(torch.zeros(2, 5), torch.zeros(2), **kw)
        return given
    assert sample(temperature=-0.5)["temperature"] == (None, -0.5)
    assert sample(temperature=math.inf)["temperature"] == (None, math.inf)
    for k in (-1, -2 ** 31, 0, 2 ** 31 - 1):
        assert sample(top_k=k)["top_k"] == (None, k)
    for bad in ({"temperature": math.nan}, {"top_k": 2 ** 31}, {"top_k": -2 ** 31 - 1},
                {"top_p": -0.1}, {"top_p": 1.1}, {"top_p": math.nan}, {"min_p": 2.0},
                {"min_p": math.nan}, {"min_p": -1.0}):
        with pytest.raises(RuntimeError):
            sample(**bad)
    x, u = torch.randn(3, 50, generator=torch.Generator().manual_seed(0)), torch.full((3,), 0.7)
    assert torch.equal(sample_torch(x, u, temperature=-0.5)[0][:, 0], x.argmax(-1))
    assert torch.equal(sample_torch(x, u, top_k=-1)[0], sample_torch(x, u)[0])


def test_a_row_of_nan_draws_a_token():
    """Logits that are all NaN draw a token that the next step takes."""
    from parrot import Parrot
    torch.manual_seed(0)
    model = Parrot(tiny_model_config()).eval()
    ids = torch.randint(0, model.config.vocab_size, (2, 9))
    _, state = model.prefill(ids)
    with torch.no_grad():
        model.final_norm.weight.fill_(math.nan)
    token = ids[:, -1:]
    for kw in ({}, {"temperature": 0.0}, {"top_k": 3}):
        token, state = model.decode_sample(token, state, torch.tensor([0.2, 0.9]), **kw)
        assert not token.any() and token.shape == (2, 1)


def test_drawn_tokens_land_in_the_given_tensor():
    """decode_step's output tensor takes drawn tokens as it does greedy ones."""
    from parrot import Parrot
    torch.manual_seed(0)
    model = Parrot(tiny_model_config()).eval()
    ids = torch.randint(0, model.config.vocab_size, (2, 9))
    u, out = torch.tensor([0.3, 0.6]), torch.full((2, 1), -7)
    _, state = model.prefill(ids)
    want, _ = model.decode_sample(ids[:, -1:], state, u, temperature=0.9)
    _, state = model.prefill(ids)
    got, _ = model.decode_step(ids[:, -1:], state, _next_token_only=True, _out=out,
                               _draw=(u, {"temperature": 0.9}))
    assert got is out and torch.equal(out, want)


def test_numbers_are_taken_in_64_bits():
    """0.1 of 40 equal weights is four of them, as the definition and the kernel have it;
    rounded to fp32 it would be a fifth."""
    from parrot.model import sample_torch
    x, u = torch.zeros(3, 40), torch.tensor([0.0, 0.5, 0.99])
    for p, kept in ((0.1, 4), (torch.full((3,), 0.1), 5)):
        token, prob = sample_torch(x, u, top_p=p)
        assert token.flatten().tolist() == [int(kept * v) for v in (0.0, 0.5, 0.99)]
        assert torch.equal(prob, torch.full((3, 1), 1 / kept))
    token, prob = sample_torch(torch.tensor([[0.0, -1.0]]), torch.zeros(1), temperature=0.3)
    assert prob.item() == torch.tensor(1 / (1 + math.exp(-1 / 0.3))).item()


def test_uniform_numbers_outside_their_range():
    """Below 0 the first token that was kept, from 1 on the last, never one that was not."""
    from parrot.model import sample_torch
    x = torch.tensor([[0.0, 5.0, 1.0, 6.0, 2.0]]).expand(6, 5)
    u = torch.tensor([-1.0, -math.inf, -0.0, 1.0, 2.0, math.inf])
    token, prob = sample_torch(x, u, top_k=2)
    assert token.flatten().tolist() == [1, 1, 1, 3, 3, 3]
    share = 1 / (1 + math.exp(-1.0))
    assert (prob.flatten() - torch.tensor([1 - share] * 3 + [share] * 3)).abs().max() <= 1e-6
