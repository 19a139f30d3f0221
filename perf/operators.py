"""Operators of generation over a paged KV cache, timed against their plain forms.

Three things a serving loop does between the model's projections: it writes the
keys and values of new tokens into pages (in bf16, or quantised to 8 bits as
they are written) and reads sequences back; it attends from a chunk of new
tokens, one or thousands of them, over those pages, through a sliding window
with a few first tokens that stay visible; and it draws the next tokens from
the logits with temperature, top-k, top-p and min-p.

Sizes are those of the default ModelConfig (8 query heads on 2 of 96, window
2048, 4096 positions, 32768 tokens) and, in between, other head layouts, page
sizes and lengths.

A page holds ``page`` positions of every kv head, in blocks of 32 positions in
MFMA fragment order: K of a block as [2][d / 32][4][16][8] (position 16 n + c,
dimension 32 s + 8 g + e at [n][s][g][c][e]), V as [d / 16][4][16][2][4]
(position 16 h + 4 g + j, dimension 16 t + c at [t][g][c][h][j]).  An 8-bit page
holds q with the value q 2^(x - 127), x being the byte of its position and head:
the smallest power of two that brings the row's largest magnitude inside the
type's range.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
BF16 = torch.bfloat16
VOCAB = 32768
TYPES = {"bf16": BF16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# the type's largest magnitude as m 2^k with 0.5 <= m < 1
LARGEST = {"e4m3": (0.875, 9), "int8": (127 / 128, 7)}


def _package():
    path = os.path.join(os.getcwd(), "parrot-h200-worker_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _keep(name, batch, new, context, page, kv_heads, head_dim, dtype, ragged):
    return {"name": name, "kind": "keep", "batch": batch, "new": new, "context": context,
            "page": page, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "ragged": ragged}


def _attend(name, batch, new, context, page, heads, kv_heads, head_dim, dtype, window, sinks,
            ragged):
    return {"name": name, "kind": "attend", "batch": batch, "new": new, "context": context,
            "page": page, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # a decode step's row of one sequence, and the sequence read back (a
        # conversation handed to a contiguous cache)
        _keep("keep_1_after_500", 1, 1, 500, 64, 2, 96, "int8", False),
        # a ragged batch of short chunks behind earlier ones
        _keep("keep_7_ragged", 7, 77, 400, 32, 4, 64, "e4m3", True),
        # prompts that fill the context, quantised and read back
        _keep("keep_4x4096", 4, 4096, 0, 128, 2, 96, "e4m3", False),
        # one token after a short prompt: latency
        _attend("attend_1_after_128", 1, 1, 128, 64, 8, 2, 96, "bf16", 2048, 0, False),
        # a served batch of conversations, windowed, the first tokens visible
        _attend("attend_32_windowed", 32, 1, 4000, 64, 8, 2, 96, "e4m3", 2048, 4, True),
        # a few long documents, everything visible
        _attend("attend_8_after_32000", 8, 1, 32000, 128, 8, 2, 96, "e4m3", 0, 0, False),
        # short ragged chunks (speculated tokens) over long contexts, wide heads
        _attend("attend_5_speculated", 5, 6, 9000, 32, 16, 2, 128, "int8", 0, 0, True),
        # a chunk of a prompt after earlier chunks
        _attend("attend_512_after_3500", 3, 512, 3500, 64, 8, 2, 96, "bf16", 2048, 4, True),
        # whole prompts in one chunk
        _attend("attend_4x4096", 4, 4096, 0, 128, 8, 2, 96, "bf16", 2048, 0, False),
        _attend("attend_2x4096_quantised", 2, 4096, 0, 64, 8, 8, 64, "int8", 0, 0, False),
        # the next token of one conversation, and of a served batch whose
        # requests each bring their own parameters
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "mixed": False},
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": VOCAB, "mixed": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["keep", "attend", "attend", "attend", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log_int(rng, 1, 64), "vocab": _log_int(rng, 100, VOCAB),
                "mixed": rng.random() < 0.7}
    heads, kv_heads, head_dim = rng.choice([(8, 2, 96), (8, 2, 96), (8, 8, 64), (16, 2, 128),
                                            (12, 4, 64), (4, 1, 96), (6, 2, 128)])
    batch = _log_int(rng, 1, 32)
    case = {"kind": kind, "batch": batch}
    if kind == "keep":
        total = _log_int(rng, 2, max(2, 8192 // batch))
        case["new"] = _log_int(rng, 1, total)
        case["context"] = total - case["new"]
    elif rng.random() < 0.5:  # single tokens and short chunks over a context
        case["new"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
        case["context"] = _log_int(rng, 1, max(1, 65536 // batch))
    else:
        total = _log_int(rng, 9, max(9, 8192 // batch))
        case["new"] = _log_int(rng, 9, total)
        case["context"] = total - case["new"]
    case.update(page=rng.choice([32, 64, 64, 128]), heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=rng.choice(["bf16", "e4m3", "int8"]),
                ragged=rng.random() < 0.5)
    if kind == "attend":
        case["window"] = rng.choice([0, 2048, rng.randint(1, 1000)])
        case["sinks"] = rng.choice([0, 4, rng.randint(1, 70)])
    else:
        del case["heads"]
    return case


def _counts(case):
    """New rows and whole lengths of each sequence, from the case alone."""
    b, new, context = case["batch"], case["new"], case["context"]
    if not case["ragged"]:
        return [new] * b, [context + new] * b
    rng = random.Random("%d %d %d" % (b, new, context))
    news = [rng.randint(max(1, new // 2), new) for _ in range(b)]
    return news, [n + rng.randint(context // 3, context) for n in news]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device=DEVICE) * std


def _keys(gen, kv_heads, d):
    """Channel scales of keys: most alike, a few several times as large."""
    return 0.55 * torch.exp(0.5 * torch.randn(kv_heads, d, generator=gen, device=DEVICE))


def _exponent(amax, dtype):
    m, k = LARGEST[dtype]
    frac, exp = torch.frexp(amax)
    e = torch.where(frac <= m, exp - k, exp - k + 1)
    return torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 120)


def _quantised(x, dtype):
    """(q, byte) of rows x [..., d]."""
    x = x.float()
    e = _exponent(x.abs().amax(-1), dtype)
    y = torch.ldexp(x, -e.unsqueeze(-1))
    y = y.to(torch.float8_e4m3fn) if dtype == "e4m3" else y.round().to(torch.int8)
    return y, (e + 127).to(torch.uint8)


def _place(d, device):
    """Where dimension w of position p of a 32-position block lies, [32, d]: K, V."""
    p = torch.arange(32, device=device)[:, None]
    w = torch.arange(d, device=device)[None, :]
    k = ((((p // 16) * (d // 32) + w // 32) * 4 + w // 8 % 4) * 16 + p % 16) * 8 + w % 8
    v = (((w // 16) * 4 + p // 4 % 4) * 16 + w % 16) * 8 + p // 16 * 4 + p % 4
    return k, v


def _batch(case, gen, seed):
    news, lengths = _counts(case)
    page = case["page"]
    width = max((n + page - 1) // page for n in lengths)
    pages = case["batch"] * width + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE)[:case["batch"] * width]
    i32 = dict(dtype=torch.int32, device=DEVICE)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    return {"starts": torch.tensor(starts, **i32), "lengths": torch.tensor(lengths, **i32),
            "table": order.view(case["batch"], width).to(torch.int32), "rows": starts[-1],
            "longest": max(lengths), "most": max(news), "pages": pages}


def _pages(case, gen, s):
    """Every page full of rows, as earlier appends left them."""
    hk, d, page, n = case["kv_heads"], case["head_dim"], case["page"], s["pages"]
    keys = _keys(gen, hk, d)
    for name, at, channel in (("key", 0, keys[:, None]), ("value", 1, 0.55)):
        rows = (_normal(gen, n, hk, page, d) * channel).to(BF16)
        if case["dtype"] != "bf16":
            rows, s[name + "_exponent"] = _quantised(rows, case["dtype"])
        place = _place(d, DEVICE)[at].flatten()
        flat = rows.view(torch.uint8 if rows.element_size() == 1 else torch.int16)
        flat = flat.view(n, hk, page // 32, 32 * d)
        out = torch.empty_like(flat)
        out[..., place] = flat
        s[name] = out.view(TYPES[case["dtype"]])
    return keys


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(gen, rows, vocab, std=2.0)
        # a trained model's head: a few tokens far above the rest, on some rows
        lift = torch.randint(0, vocab, (rows, 8), generator=gen, device=DEVICE)
        logits.scatter_add_(1, lift, _normal(gen, rows, 8, std=4.0).abs())
        s["logits"] = logits
        s["uniform"] = torch.rand(rows, generator=gen, device=DEVICE)
        pick = lambda values: torch.tensor(values, device=DEVICE)[  # noqa: E731
            torch.randint(0, len(values), (rows,), generator=gen, device=DEVICE)]
        if case["mixed"]:
            s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3])
            s["top_k"] = pick([0, 0, 1, 20, 50, 300]).to(torch.int32)
            s["top_p"] = pick([1.0, 1.0, 0.95, 0.9, 0.5])
            s["min_p"] = pick([0.0, 0.0, 0.0, 0.02, 0.1])
        else:
            s["temperature"], s["top_p"], s["min_p"] = (
                torch.full((rows,), x, device=DEVICE) for x in (0.8, 0.95, 0.0))
            s["top_k"] = torch.full((rows,), 50, dtype=torch.int32, device=DEVICE)
        return s
    s.update(_batch(case, gen, seed))
    channel = _pages(case, gen, s)
    hk, d, rows = case["kv_heads"], case["head_dim"], s["rows"]
    if case["kind"] == "keep":
        # views of a packed projection's output
        packed = _normal(gen, rows, 2, hk, d)
        packed[:, 0] *= channel
        packed[:, 1] *= 0.55
        packed = packed.to(BF16)
        s["k"], s["v"] = packed[:, 0], packed[:, 1]
    else:
        h = case["heads"]
        packed = _normal(gen, rows, h + 2 * hk, d, std=1.5).to(BF16)
        s["q"] = packed[:, :h]
        s["scale"] = d ** -0.5
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    with torch.no_grad():
        if own:
            return _run_own(state)
        if state["kind"] == "sample":
            return _sample_plain(state)
        if state["kind"] == "keep":
            return _keep_plain(state)
        return _attend_plain(state)


def _run_own(s):
    if "handles" not in s:  # what a program keeps: the cache over its pages, the batch
        _package()
        from parrot import hip_moe
        from parrot.paged import PagedBatch, PagedKVCache
        if s["kind"] == "sample":
            s["handles"] = hip_moe.sample
        else:
            s["handles"] = (
                PagedKVCache.from_pages(s["key"], s["value"], s.get("key_exponent"),
                                        s.get("value_exponent")),
                PagedBatch(s["table"], s["lengths"], s["starts"]))
    if s["kind"] == "sample":
        return s["handles"](s["logits"], s["uniform"], temperature=s["temperature"],
                            top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    cache, batch = s["handles"]
    if s["kind"] == "keep":
        cache.append(s["k"], s["v"], batch)
        return cache.read(batch, s["longest"])
    return cache.attend(s["q"], batch, scale=s["scale"], window=s["window"] or None,
                        sinks=s["sinks"])


def _rows_of(s):
    """Sequence and position of every new row."""
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    start, end = s["starts"][seq], s["starts"][seq + 1]
    return seq, (s["lengths"][seq] - end + row).long(), row - start


def _read_plain(s, longest):
    """Keys and values [b, Hk, longest, d] of the batch, in fp32."""
    b, width = s["table"].shape
    hk, d, page = s["kv_heads"], s["head_dim"], s["page"]
    got = []
    for name, at in (("key", 0), ("value", 1)):
        x = s[name][s["table"].long()].float()  # [b, width, Hk, blocks, 32 d]
        x = x[..., _place(d, DEVICE)[at].flatten()].view(b, width, hk, page, d)
        if s["dtype"] != "bf16":
            e = s[name + "_exponent"][s["table"].long()].int() - 127
            x = torch.ldexp(x, e.unsqueeze(-1))
        x = x.transpose(1, 2).reshape(b, hk, width * page, d)[:, :, :longest]
        there = torch.arange(x.shape[2], device=DEVICE) < s["lengths"][:, None]
        got.append(torch.where(there[:, None, :, None], x, torch.zeros_like(x)))
    return got


def _keep_plain(s):
    d, page = s["head_dim"], s["page"]
    seq, position, _ = _rows_of(s)
    at_page = s["table"][seq, position // page].long()[:, None, None]
    head = torch.arange(s["kv_heads"], device=DEVICE)[None, :, None]
    block = (position % page // 32)[:, None, None]
    for name, x, place in (("key", s["k"], _place(d, DEVICE)[0]),
                           ("value", s["v"], _place(d, DEVICE)[1])):
        if s["dtype"] != "bf16":
            x, byte = _quantised(x, s["dtype"])
            s[name + "_exponent"][at_page[..., 0], head[..., 0],
                                  (position % page)[:, None]] = byte
        pages = s[name]
        if s["dtype"] == "e4m3":  # bytes are moved
            x, pages = x.view(torch.uint8), pages.view(torch.uint8)
        pages[at_page, head, block, place[position % 32][:, None, :]] = x
    return [x.to(BF16) for x in _read_plain(s, s["longest"])]


def _attend_plain(s):
    b, h, hk, d = s["batch"], s["heads"], s["kv_heads"], s["head_dim"]
    rep, most = h // hk, s["most"]
    k, v = _read_plain(s, s["longest"])
    seq, position, index = _rows_of(s)
    q = torch.zeros(b, most, h, d, device=DEVICE)
    q[seq, index] = s["q"].float()
    q = q.view(b, most, hk, rep, d).permute(0, 2, 3, 1, 4).reshape(b, hk, rep * most, d)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    at = torch.zeros(b, most, dtype=torch.long, device=DEVICE)
    at[seq, index] = position
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if s["window"]:
        seen &= (key > at[..., None] - s["window"]) | (key < s["sinks"])
    scores = scores.view(b, hk, rep, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    scores = scores.view(b, hk, rep * most, -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    y = y.view(b, hk, rep, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, h * d)
    return y[seq, index].to(BF16)


def _sample_plain(s):
    """In 64 bits: a border between two tokens is a matter of the last bits."""
    t = s["temperature"].double()[:, None]
    x = s["logits"].double() / torch.where(t > 0, t, torch.ones_like(t))
    rank = torch.arange(x.shape[1], device=DEVICE)
    # the most likely first, equal ones by their index
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp(x - x[:, :1])
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    k = torch.where(t > 0, k, torch.ones_like(k))
    w = torch.where(rank < k, w, torch.zeros_like(w))
    before = torch.cumsum(w, -1) - w
    top_p = s["top_p"].double()[:, None]
    w = torch.where((before < top_p * w.sum(-1, keepdim=True)) | (top_p >= 1), w,
                    torch.zeros_like(w))
    w = torch.where(w >= s["min_p"].double()[:, None], w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)  # by index again
    reach = torch.cumsum(w, -1)
    total = reach[:, -1:]
    token = torch.searchsorted(reach, s["uniform"].double()[:, None] * total, right=True)
    return token, (w.gather(1, token) / total).float()


# ---------------------------------------------------------------------------
# the least work, and the definitions in 64 bits
# ---------------------------------------------------------------------------

def _seen(position, window, sinks):
    """Keys a query at `position` sees."""
    if position < 0:
        return 0
    n = position + 1
    if not window or n <= window:
        return n
    return window + min(sinks, n - window)


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * 32, "flops": 4 * n}
    news, lengths = _counts(case)
    hk, d = case["kv_heads"], case["head_dim"]
    stored = 2 * hk * (2 * d if case["dtype"] == "bf16" else d + 1)  # a position, K and V
    if case["kind"] == "keep":
        new, old = sum(news), sum(lengths) - sum(news)
        return {"bytes": new * (4 * hk * d + stored) + old * stored +
                case["batch"] * max(lengths) * 4 * hk * d, "flops": 6 * new * hk * d}
    window, sinks = case["window"], case["sinks"]
    pairs = read = 0
    for n, length in zip(news, lengths):
        pairs += sum(_seen(p, window, sinks) for p in range(length - n, length))
        first = max(0, length - n - window + 1) if window else 0
        read += length - first + min(sinks if window else 0, first)
    return {"bytes": read * stored + sum(news) * 4 * case["heads"] * d,
            "flops": 4 * d * case["heads"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _sample_exact(s)
    hk, d, page = case["kv_heads"], case["head_dim"], case["page"]
    news, lengths = _counts(case)
    rows = {"key": [], "value": []}  # of each sequence, [length, Hk, d]
    for i, length in enumerate(lengths):
        table = s["table"][i, :(length + page - 1) // page].long()
        for name in rows:
            x = s[name][table].double().view(len(table), hk, page // 32, -1)
            if name == "key":  # [n][s][g][c][e]
                x = x.view(*x.shape[:3], 2, d // 32, 4, 16, 8).permute(0, 2, 3, 6, 1, 4, 5, 7)
            else:  # [t][g][c][h][j]
                x = x.view(*x.shape[:3], d // 16, 4, 16, 2, 4).permute(0, 2, 6, 4, 7, 1, 3, 5)
            x = x.reshape(len(table) * page, hk, d)
            if case["dtype"] != "bf16":
                e = s[name + "_exponent"][table].double() - 127
                x = x * torch.exp2(e).transpose(1, 2).reshape(-1, hk, 1)
            rows[name].append(x[:length])
    if case["kind"] == "keep":
        return _keep_exact(case, s, rows, news, lengths)
    h, rep = case["heads"], case["heads"] // hk
    window = case["window"] or (1 << 40)
    out, at = [], 0
    for i, (n, length) in enumerate(zip(news, lengths)):
        q = s["q"][at:at + n].double()
        at += n
        pos = torch.arange(length - n, length, device=DEVICE)[:, None]
        key = torch.arange(length, device=DEVICE)
        seen = (key <= pos) & ((key > pos - window) | (key < case["sinks"]))
        y = torch.empty_like(q)
        for head in range(h):
            z = (q[:, head] @ rows["key"][i][:, head // rep].T.contiguous()) * d ** -0.5
            p = z.masked_fill(~seen, -math.inf).softmax(-1)
            y[:, head] = p @ rows["value"][i][:, head // rep].contiguous()
        out.append(y.view(n, h * d))
    return torch.cat(out)


def _keep_exact(case, s, rows, news, lengths):
    got, at = [], 0
    for name, x in (("key", s["k"]), ("value", s["v"])):
        y = torch.zeros(case["batch"], case["kv_heads"], max(lengths), case["head_dim"],
                        dtype=torch.float64, device=DEVICE)
        at = 0
        for i, (n, length) in enumerate(zip(news, lengths)):
            new = x[at:at + n].double()
            at += n
            if case["dtype"] != "bf16":
                m, k = LARGEST[case["dtype"]]
                step = torch.exp2(torch.ceil(torch.log2(
                    new.abs().amax(-1, keepdim=True) / (m * 2.0 ** k))).clamp(-100, 120))
                z = new / step
                if case["dtype"] == "int8":
                    new = torch.round(z) * step
                else:  # 3 bits behind the leading one, down to 2^-9
                    ulp = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
                    new = torch.round(z / ulp) * ulp * step
            y[i, :, :length] = torch.cat((rows[name][i][:length - n], new)).transpose(0, 1)
        got.append(y)
    return got


def _sample_exact(s):
    got = []
    for x, u, t, k, p, m in zip(*(s[n].double().cpu().numpy() for n in (
            "logits", "uniform", "temperature", "top_k", "top_p", "min_p"))):
        if t == 0:
            got.append(1.0)
            continue
        w = np.exp(x / t - (x / t).max())
        order = np.argsort(-w, kind="stable")
        kept = order[:int(k)] if k else order
        if p < 1:
            mass = np.cumsum(w[kept])
            kept = kept[np.concatenate(([0.0], mass[:-1])) < p * mass[-1]]
        kept = np.sort(kept[w[kept] >= m])
        reach = np.cumsum(w[kept])
        i = int(np.searchsorted(reach, u * reach[-1], side="right"))
        got.append(w[kept[i]] / reach[-1])
    return None, torch.tensor(got, dtype=torch.float64)[:, None]
