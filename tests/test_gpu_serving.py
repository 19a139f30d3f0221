"""GPU checks of the paged cache, attention over it and sampling as a program runs
them together: RoPE at ragged positions, a layer extended over paged sequences,
generation that draws its tokens, eagerly and from a captured graph."""
import pytest
import torch

from conftest import tiny_model_config
from paged_cases import stored

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float8_e4m3fn, torch.int8]


def _hip_config(**kw):
    from parrot import ModelConfig
    return ModelConfig(moe_backend="grouped_hip", depth_backend="hip", collect_router_stats=False,
                       **kw)


def _layer(cfg, seed=0):
    from parrot.model import LocalGQA
    torch.manual_seed(seed)
    with torch.device("cuda"):
        layer = LocalGQA(cfg).bfloat16().eval()
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0.0, 0.04)
    return layer


@pytest.mark.parametrize("dtype", TYPES)
def test_append_rope(dtype):
    """Keys and queries rotated at ragged positions: the bits of the RoPE launch
    whose rows have one first position, then stored as any keys are; rows of no
    page and past the table have their queries rotated all the same."""
    from parrot import PagedBatch, PagedKVCache, hip_moe
    from parrot.model import _rope_tables
    cfg = _hip_config()
    heads, hk, d = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    g = torch.Generator().manual_seed(1)
    news, lengths = [5, 40, 1, 33], [5, 100, 2000, 80]
    qkv = torch.randn(sum(news), heads + 2 * hk, d, generator=g).bfloat16().cuda()
    cos, sin = _rope_tables(cfg, qkv.new_empty(0, dtype=torch.float32))
    cache = PagedKVCache(40, 64, hk, d, dtype)
    tables = [[3], [7, 1], list(range(8, 40)), [0]]  # the last one's second page is missing
    with torch.no_grad():
        batch = PagedBatch.from_lists(tables, lengths, news)
        q, k, v = qkv.split((heads, hk, hk), dim=1)
        got = cache.append_rope(q, k, v, batch, cos, sin)
        keys, values = cache.read(batch, 2000)
        at = 0
        for i, (n, length) in enumerate(zip(news, lengths)):
            rows = qkv[at:at + n].reshape(1, n, -1)
            qr, kr, vr = hip_moe.rope_qkv(rows, cos, sin, heads, hk, d, length - n, False)
            assert torch.equal(got[at:at + n], qr[0].transpose(0, 1))
            kept = min(length, 64 * len(tables[i])) - (length - n)  # rows that have a page
            for x, y in ((keys, kr), (values, vr)):
                want = stored(y[0, :, :kept].cpu(), dtype)
                assert torch.equal(x[i, :, length - n:length - n + kept].double().cpu(), want)
            at += n


def _attended(layer, x, positions_first, window, sinks, dtype):
    """A layer's output for one sequence x [t, dim] in float64, keys and values as a
    cache of ``dtype`` stores the bf16 ones."""
    from parrot.model import _apply_rope
    c = layer.cfg
    t = x.shape[0]
    x64 = x.double()
    w = [getattr(layer, n).weight.double() for n in ("q", "k", "v", "out")]
    q, k, v = ((x64 @ m.T).bfloat16().view(1, t, -1, c.head_dim).transpose(1, 2)
               for m in w[:3])
    q, k = (_apply_rope(c, y.double(), 0).bfloat16() for y in (q, k))
    k, v = (stored(y[0].cpu(), dtype).cuda() for y in (k, v))
    rep = c.n_heads // c.n_kv_heads
    s = torch.matmul(q[0].double(), k.repeat_interleave(rep, 0).transpose(1, 2).contiguous())
    i, j = torch.arange(t, device="cuda")[:, None], torch.arange(t, device="cuda")
    seen = (j <= i) & ((j > i - window) | (j < sinks))
    p = (s * c.head_dim ** -0.5).masked_fill(~seen, -float("inf")).softmax(-1)
    y = torch.matmul(p, v.repeat_interleave(rep, 0)).transpose(0, 1).reshape(t, -1)
    return y @ w[3].T


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sinks", [0, 5])
def test_layer_extended_in_chunks(dtype, sinks):
    """Three sequences fed to a layer in chunks, then token by token, as the layer
    over each whole sequence gives.  A bf16 pipeline rounds q, k, v (2^-8 each, and
    a quantised key or value may round to the other side of a step where its bf16
    differs in the last bit), P, y and the output: the error's norm stays within
    three per cent of the output's, and the HIP prefill's own is of that size."""
    from parrot import PagedBatch, PagedKVCache
    cfg = _hip_config(window_size=100)
    layer = _layer(cfg)
    g = torch.Generator().manual_seed(2)
    lengths = [150, 37, 301]
    xs = [torch.randn(n, cfg.dim, generator=g).bfloat16().cuda() for n in lengths]
    cache = PagedKVCache(20, 32, cfg.n_kv_heads, cfg.head_dim, dtype)
    order = torch.randperm(20, generator=g).tolist()
    tables = [order[:5], order[5:7], order[7:17]]
    done, outs = [0, 0, 0], [[], [], []]
    steps = [[100, 0, 33], [1, 30, 200], [40, 5, 60]] + [[1, 1, 1], [1, 1, 1]] + [[7, 0, 6]]
    with torch.no_grad():
        for new in steps:
            done = [a + b for a, b in zip(done, new)]
            batch = PagedBatch.from_lists(tables, done, new)
            x = torch.cat([x[a - n:a] for x, a, n in zip(xs, done, new)])
            addend = torch.randn(x.shape, generator=g).bfloat16().cuda()
            y = layer.extend(x, cache, batch, sinks=sinks)
            assert torch.equal(layer.extend(x, cache, batch, addend=addend, sinks=sinks),
                               addend + y)
            for out, part in zip(outs, y.split(new)):
                out.append(part)
        assert done == lengths
        for x, out in zip(xs, outs):
            want = _attended(layer, x, 0, cfg.window_size, sinks, dtype)
            got = torch.cat(out).double()
            err = ((got - want).norm() / want.norm()).item()
            print(f"relative error {err:.2e}", flush=True)
            assert err < 3e-2
            if sinks == 0 and dtype == torch.bfloat16:
                whole = layer.prefill(x[None])[0][0].double()
                base = ((whole - want).norm() / want.norm()).item()
                print(f"prefill's {base:.2e}", flush=True)
                assert err < 1.2 * base


def test_layer_refuses_pages_past_its_positions():
    """A table may end inside the page that max_seq_len ends in, not behind it."""
    from parrot import PagedBatch, PagedKVCache
    cfg = _hip_config(max_seq_len=100, window_size=50)
    layer = _layer(cfg)
    cache = PagedKVCache(6, 32, cfg.n_kv_heads, cfg.head_dim)
    x = torch.randn(3, cfg.dim, device="cuda").bfloat16()
    with torch.no_grad():
        layer.extend(x, cache, PagedBatch.from_lists([[0, 1, 2, 3]], [100], [3]))
        with pytest.raises(ValueError, match="max_seq_len"):
            layer.extend(x, cache, PagedBatch.from_lists([[0, 1, 2, 3, 4]], [131], [3]))


def _model(seed=0, **kw):
    from parrot import Parrot
    torch.manual_seed(seed)
    cfg = tiny_model_config(moe_backend="grouped_hip", depth_backend="hip",
                            collect_router_stats=False, **kw)
    return Parrot(cfg).cuda().bfloat16().eval()


def test_generation_that_draws():
    """decode_sample draws from decode_step's logits; a captured graph gives the
    same tokens, its parameters and numbers read at every replay."""
    from parrot import hip_moe
    from parrot.decode_graph import DecodeGraph
    model = _model()
    ids = torch.randint(0, model.config.vocab_size, (3, 20),
                        generator=torch.Generator().manual_seed(1)).cuda()
    g = torch.Generator().manual_seed(2)
    us = torch.rand(12, 3, generator=g).cuda()
    kw = dict(temperature=torch.tensor([0.7, 1.3, 0.0], device="cuda"), top_k=20, top_p=0.9)
    with torch.inference_mode():
        logits, state = model.prefill(ids)
        first = logits[:, -1].argmax(-1, keepdim=True)
        token, drawn = first, []
        for u in us:
            token, state = model.decode_sample(token, state, u, **kw)
            drawn.append(token)
        # by hand
        _, state = model.prefill(ids)
        token = first
        for u, want in zip(us, drawn):
            logits, state = model.decode_step(token, state)
            token = hip_moe.sample(logits[:, -1], u, **kw)[0]
            assert torch.equal(token, want)
        # captured, twice over, with eager work in between
        for _ in range(2):
            _, state = model.prefill(ids)
            temperature = torch.zeros(3, device="cuda")
            graph = DecodeGraph(model, state, sampling={**kw, "temperature": temperature})
            temperature.copy_(kw["temperature"])
            token = first
            for u, want in zip(us, drawn):
                token = graph.step(token, u)
                torch.zeros(1000, device="cuda").sum().item()
                assert torch.equal(token, want)
        assert torch.equal(torch.cat(drawn, 1)[2], _greedy(model, ids, first, 12)[2])
        with pytest.raises(ValueError):
            graph.step(token)
        with pytest.raises(ValueError):
            graph.step(token, us[0, :2])
        with pytest.raises(RuntimeError):
            DecodeGraph(model, state, logits=True, sampling=kw)


@pytest.mark.parametrize("batch,kw", [(3, {}), (17, {}), (3, {"residual": "standard"})])
def test_rows_of_nan_draw_a_token(batch, kw):
    """Logits that are all NaN draw token 0, eagerly and captured, also where the next
    step's embedding is looked up by itself (more than 16 sequences, no depth mixes)."""
    from parrot.decode_graph import DecodeGraph
    model = _model(**kw)
    ids = torch.randint(0, model.config.vocab_size, (batch, 20),
                        generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.linspace(0, 0.9, batch, device="cuda")
    with torch.inference_mode():
        _, state = model.prefill(ids)
        weight = model.final_norm.weight.clone()
        model.final_norm.weight.fill_(float("nan"))
        token = ids[:, -1:].contiguous()
        for _ in range(2):
            token, state = model.decode_sample(token, state, u, top_k=5)
            assert token.shape == (batch, 1) and not token.any()
        graph = DecodeGraph(model, state, sampling=dict(temperature=0.8))
        for _ in range(3):
            token = graph.step(token, u)
            assert not token.any()
        model.final_norm.weight.copy_(weight)
        want, _ = model.decode_sample(token.clone(), state, u, temperature=0.8)
        state.position -= 1
        state.position_device.sub_(1)
        assert torch.equal(graph.step(token, u), want) and (want >= 0).all()


@pytest.mark.parametrize("rows,vocab,dim", [(1, 300, 768), (16, 32768, 768), (5, 1001, 200)])
def test_greedy_rows_of_nan(rows, vocab, dim):
    """A row whose logits are all NaN gives token 0, the others theirs."""
    from parrot import hip_moe
    g = torch.Generator().manual_seed(3)
    h = torch.randn(rows, dim, generator=g).bfloat16().cuda()
    w = torch.randn(vocab, dim, generator=g).bfloat16().cuda()
    with torch.no_grad():
        want = hip_moe.vocab_argmax(h, w)
        h[rows // 2] = float("nan")
        want[rows // 2] = 0
        assert torch.equal(hip_moe.vocab_argmax(h, w), want)


@pytest.mark.parametrize("batch,kw", [(3, {}), (17, {}), (3, {"residual": "standard"})])
def test_greedy_steps_of_nan(batch, kw):
    """Greedy tokens of logits that are all NaN are tokens that the next step takes."""
    from parrot.decode_graph import DecodeGraph
    model = _model(**kw)
    ids = torch.randint(0, model.config.vocab_size, (batch, 20),
                        generator=torch.Generator().manual_seed(1)).cuda()
    with torch.inference_mode():
        _, state = model.prefill(ids)
        model.final_norm.weight.fill_(float("nan"))
        token = ids[:, -1:].contiguous()
        for _ in range(2):
            token, state = model.decode_next(token, state)
            assert not token.any()
        graph = DecodeGraph(model, state)
        for _ in range(3):
            token = graph.step(token)
            assert not token.any()


@pytest.mark.parametrize("batch,kw", [(3, {}), (17, {}), (3, {"residual": "standard"})])
def test_captured_ids_outside_the_vocabulary(batch, kw):
    """A captured step takes ids outside the embedding as its nearest row, such as the
    -1 that hip_moe.sample writes into a graph's ids for a row of NaN."""
    from parrot import hip_moe
    from parrot.decode_graph import DecodeGraph
    model = _model(**kw)
    vocab = model.config.vocab_size
    ids = torch.randint(0, vocab, (batch, 20), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.inference_mode():
        _, state = model.prefill(ids)
        graph = DecodeGraph(model, state, logits=True)
        u = torch.zeros(batch, device="cuda")
        nothing = torch.full((batch, vocab), float("nan"), device="cuda")

        def step(token):
            state.position = 20
            state.position_device.fill_(20)
            return graph.step(token).clone()
        for far, near in ((-1, 0), (vocab, vocab - 1), (2 ** 40, vocab - 1)):
            want = step(torch.full((batch, 1), near, device="cuda"))
            assert torch.equal(step(torch.full((batch, 1), far, device="cuda")), want)
            if far == -1:
                hip_moe.sample(nothing, u, out=graph.ids)
                assert (graph.ids == -1).all() and torch.equal(step(graph.ids), want)


def _greedy(model, ids, token, steps):
    _, state = model.prefill(ids)
    out = []
    for _ in range(steps):
        token, state = model.decode_next(token, state)
        out.append(token)
    return torch.cat(out, 1)


def test_layer_refusals():
    from parrot import PagedBatch, PagedKVCache
    cfg = _hip_config()
    layer = _layer(cfg)
    cache = PagedKVCache(4, 32, cfg.n_kv_heads, cfg.head_dim)
    batch = PagedBatch.from_lists([[0]], [3], [3])
    x = torch.randn(3, cfg.dim, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):  # gradients
        layer.extend(x, cache, batch)
    with torch.no_grad():
        for bad in ((x[None], cache, batch), (x.float(), cache, batch),
                    (x, PagedKVCache(4, 32, 1, cfg.head_dim), batch),
                    (x, cache, PagedBatch.from_lists([[0]], [3], [3], device="cpu"))):
            with pytest.raises(RuntimeError):
                layer.extend(*bad)
        assert layer.extend(x[:0], cache, batch).shape == (0, cfg.dim)
