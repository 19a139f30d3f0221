"""A paged KV cache in 4 bits, and its pages handed out on the GPU, timed against plain forms.

Three more things that a serving loop does: it keeps keys and values in pages of
4 bits (quantised as they are written, read back as rows); it attends from a
chunk of new tokens, one or thousands of them, over those pages; and it hands
the pages out, on the GPU and from the requests' lengths alone: the page
tables, the rows' starts, positions and slots of a step, and the pages of
tokens that are taken back.

Sizes are those of the default ModelConfig (8 query heads on 2 of 96, window
2048, 4096 positions) and, in between, other head layouts, page sizes and
lengths.

A page holds ``page`` positions of every kv head, in blocks of 32 positions.  A
block's values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), eight
to a word, the first in the lowest bits, in records of d / 16 words, one for
each g < 4 and c < 16: K [g][c][n][s], position 16 n + c, dimensions 32 s + 8 g
to 32 s + 8 g + 7; V [g][c][o][u], dimension 32 u + 16 o + c, positions 4 g to
4 g + 3 and 16 + 4 g to 16 + 4 g + 3.  A value is q 2^(x - 127); the byte x is
one for 32 dimensions of a key ([16][2][d / 32] of a block: [c][n][s]) and one
for a whole value row.  2^(x - 127) is the power of two that leaves the largest
magnitude of those values above 3.5 and not above 7 (what is above 6 becomes 6).
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
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _package():
    path = os.path.join(os.getcwd(), "parrot-h200-worker_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _keep(name, batch, new, context, page, kv_heads, head_dim, ragged):
    return {"name": name, "kind": "keep", "batch": batch, "new": new, "context": context,
            "page": page, "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged}


def _attend(name, batch, new, context, page, heads, kv_heads, head_dim, window, sinks, ragged):
    return {"name": name, "kind": "attend", "batch": batch, "new": new, "context": context,
            "page": page, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "window": window, "sinks": sinks, "ragged": ragged}


def _pool(name, batch, new, context, page, pages, ragged):
    return {"name": name, "kind": "pool", "batch": batch, "new": new, "context": context,
            "page": page, "pages": pages, "ragged": ragged}


def listed():
    return [
        # a decode step's row of one sequence, and the sequence read back (a
        # conversation handed to a contiguous cache)
        _keep("keep_1_after_500", 1, 1, 500, 64, 2, 96, False),
        # a ragged batch of short chunks behind earlier ones
        _keep("keep_7_ragged", 7, 77, 400, 32, 4, 64, True),
        # prompts that fill the context, quantised and read back
        _keep("keep_4x4096", 4, 4096, 0, 128, 2, 96, False),
        # one token after a short prompt: latency
        _attend("attend_1_after_128", 1, 1, 128, 64, 8, 2, 96, 2048, 0, False),
        # a served batch of conversations, windowed, the first tokens visible
        _attend("attend_32_windowed", 32, 1, 4000, 64, 8, 2, 96, 2048, 4, True),
        # a few long documents, everything visible: what 4 bits are for
        _attend("attend_8_after_32000", 8, 1, 32000, 128, 8, 2, 96, 0, 0, False),
        # short ragged chunks (speculated tokens) over long contexts, wide heads
        _attend("attend_5_speculated", 5, 6, 9000, 32, 16, 2, 128, 0, 0, True),
        # a chunk of a prompt after earlier chunks
        _attend("attend_512_after_3500", 3, 512, 3500, 64, 8, 2, 96, 2048, 4, True),
        # whole prompts in one chunk
        _attend("attend_2x4096", 2, 4096, 0, 64, 8, 8, 64, 0, 0, False),
        # a step of a few conversations: one more token each, taken back
        _pool("pool_8_step", 8, 1, 4000, 64, 4096, False),
        # a served batch whose draft of a few tokens is turned down
        _pool("pool_32_speculated", 32, 6, 4000, 32, 8192, True),
        # a server filled with prompts, and emptied
        _pool("pool_400_admitted", 400, 4096, 0, 64, 40000, True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["keep", "attend", "attend", "attend", "pool"])
    if kind == "pool":
        batch = _log_int(rng, 1, 400)
        new = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
        context = rng.choice([0, rng.randint(1, 4096), rng.randint(1, 4096)])
        page = rng.choice([32, 64, 64, 128])
        most = batch * ((new + context + page - 1) // page)
        # from pools that are nearly empty to some that cannot hold the step
        pages = min(40000, max(64, int(most * rng.choice([0.9, 1.15, 1.5, 3.0]))))
        return {"kind": kind, "batch": batch, "new": new, "context": context, "page": page,
                "pages": pages, "ragged": rng.random() < 0.7}
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
                head_dim=head_dim, ragged=rng.random() < 0.5)
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


def _quantised(x, group):
    """(q as 4 bits in bytes, byte) of rows x [..., d], one byte for `group` of them."""
    x = x.float().unflatten(-1, (-1, group))
    frac, exp = torch.frexp(x.abs().amax(-1))  # 0.5 <= frac < 1
    e = torch.where(frac <= 0.875, exp - 3, exp - 2).clamp(-100, 125)
    e = torch.where(frac > 0, e, torch.full_like(e, -100))
    y = torch.ldexp(x, -e.unsqueeze(-1))
    # the nearest of the eight magnitudes; between two the one whose last bit is 0
    size, code = y.abs(), torch.zeros(y.shape, dtype=torch.uint8, device=y.device)
    for i in range(1, 8):
        border = (E2M1[i - 1] + E2M1[i]) / 2
        code += (size >= border) if i % 2 == 0 else (size > border)
    code |= torch.signbit(x).to(torch.uint8) << 3
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _place(d, device):
    """Where dimension w of position p of a 32-position block lies, [32, d]: K, V."""
    s = d // 32
    p = torch.arange(32, device=device)[:, None]
    w = torch.arange(d, device=device)[None, :]
    k = (((w // 8 % 4 * 16 + p % 16) * 2 + p // 16) * s + w // 32) * 8 + w % 8
    v = (((p // 4 % 4 * 16 + w % 16) * 2 + w // 16 % 2) * s + w // 32) * 8 + p // 16 * 4 + p % 4
    return k, v


def _place_exponents(d, device):
    """Where the byte of group s of key p of a block lies, [32, d / 32]."""
    p = torch.arange(32, device=device)[:, None]
    return (p % 16 * 2 + p // 16) * (d // 32) + torch.arange(d // 32, device=device)[None, :]


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
        code, byte = _quantised(rows, d if at else 32)
        code = code.view(n, hk, page // 32, 32 * d)
        out = torch.empty_like(code)
        out[..., _place(d, DEVICE)[at].flatten()] = code
        s[name] = out[..., ::2] | out[..., 1::2] << 4
        if at:
            s["value_exponent"] = byte.view(n, hk, page)
        else:
            byte = byte.view(n, hk, page // 32, d)  # [position][group]
            s["key_exponent"] = torch.empty_like(byte)
            s["key_exponent"][..., _place_exponents(d, DEVICE).flatten()] = byte
    return keys


def _prepare_pool(case, gen, s):
    """Sequences of their old lengths on pages in no order; of the other pages some hold
    what is kept for later requests (used once or, shared, more often), the rest are
    free.  A pool that is too small for the old lengths holds as many sequences as it
    can; the others are empty."""
    news, lengths = _counts(case)
    page, pages = case["page"], case["pages"]
    width = max((n + page - 1) // page for n in lengths)
    order = torch.randperm(pages, generator=gen, device=DEVICE).cpu().tolist()
    table, old, at = [], [], 0
    for n, length in zip(news, lengths):
        need = (length - n + page - 1) // page
        if at + need > pages:
            need, length = 0, n
        table.append(order[at:at + need] + [-1] * (width - need))
        old.append(length - n)
        at += need
    i32 = dict(dtype=torch.int32, device=DEVICE)
    s["table"] = torch.tensor(table, **i32)
    s["lengths"] = torch.tensor(old, **i32)
    s["old"] = torch.tensor(old, **i32)
    s["starts"] = torch.zeros(case["batch"] + 1, **i32)
    s["new_rows"] = torch.tensor(news, **i32)
    s["rows"] = sum(news)
    s["uses"] = torch.zeros(pages, **i32)
    s["uses"][torch.tensor(order[:at], dtype=torch.long, device=DEVICE)] = 1
    kept = order[at:at + pages // 10 + 1]
    s["uses"][torch.tensor(kept, dtype=torch.long, device=DEVICE)] = torch.randint(
        1, 4, (len(kept),), generator=gen, device=DEVICE, dtype=torch.int32)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "pool":
        return _prepare_pool(case, gen, s)
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
        if state["kind"] == "pool":
            return _pool_plain(state)
        if state["kind"] == "keep":
            return _keep_plain(state)
        return _attend_plain(state)


def _run_own(s):
    if "handles" not in s:  # what a program keeps: the cache or the pool, and the batch
        _package()
        from parrot.paged import PagedBatch, PagedKVCache, PagePool
        batch = PagedBatch(s["table"], s["lengths"], s["starts"])
        if s["kind"] == "pool":
            s["handles"] = PagePool.from_uses(s["uses"], s["page"]), batch
        else:
            fp4 = torch.float4_e2m1fn_x2
            s["handles"] = PagedKVCache.from_pages(
                s["key"].view(fp4), s["value"].view(fp4), s["key_exponent"],
                s["value_exponent"]), batch
    cache, batch = s["handles"]
    if s["kind"] == "pool":
        slots, positions = cache.extend(batch, s["new_rows"], s["rows"])
        cache.release(batch, s["old"])
        return slots, positions, s["starts"], s["lengths"], s["table"], s["uses"]
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
    values = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=DEVICE)
    table = s["table"].long()
    got = []
    for name, at in (("key", 0), ("value", 1)):
        x = s[name][table]  # [b, width, Hk, blocks, 16 d]
        x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
        x = values[x[..., _place(d, DEVICE)[at].flatten()].long()].view(b, width, hk, page, d)
        e = s[name + "_exponent"][table].int() - 127
        if at:
            x = torch.ldexp(x, e.unsqueeze(-1))
        else:
            e = e[..., _place_exponents(d, DEVICE).flatten()].view(b, width, hk, page, d // 32, 1)
            x = torch.ldexp(x.unflatten(-1, (-1, 32)), e).flatten(-2)
        x = x.transpose(1, 2).reshape(b, hk, width * page, d)[:, :, :longest]
        there = torch.arange(x.shape[2], device=DEVICE) < s["lengths"][:, None]
        got.append(torch.where(there[:, None, :, None], x, torch.zeros_like(x)))
    return got


def _keep_plain(s):
    d, page = s["head_dim"], s["page"]
    seq, position, _ = _rows_of(s)
    at_page = s["table"][seq, position // page].long()[:, None]
    head = torch.arange(s["kv_heads"], device=DEVICE)[None, :]
    block, p = (position % page // 32)[:, None], position % 32
    for name, x, at in (("key", s["k"], 0), ("value", s["v"], 1)):
        code, byte = _quantised(x, d if at else 32)
        if at:
            s["value_exponent"][at_page, head, (position % page)[:, None]] = byte[..., 0]
        else:
            s["key_exponent"][at_page[..., None], head[..., None], block[..., None],
                              _place_exponents(d, DEVICE)[p][:, None, :]] = byte
        pages = torch.stack((s[name] & 15, s[name] >> 4), -1).flatten(-2)
        pages[at_page[..., None], head[..., None], block[..., None],
              _place(d, DEVICE)[at][p][:, None, :]] = code
        s[name].copy_(pages[..., ::2] | pages[..., 1::2] << 4)
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


def _pool_plain(s):
    """New rows for the sequences in order, each on the lowest free pages; then back to
    the old lengths."""
    page, rows, table, lengths = s["page"], s["rows"], s["table"], s["lengths"]
    b, width = table.shape
    column = torch.arange(width, device=DEVICE)
    n, old = s["new_rows"].long().clamp_min(0), lengths.long()
    n = torch.where(old + n <= width * page, n, torch.zeros_like(n))
    have = (old + page - 1) // page
    need = (old + n + page - 1) // page - have
    free = (s["uses"] <= 0).nonzero()[:, 0]
    taken = need.cumsum(0)
    fits = (n.cumsum(0) <= rows) & ((need == 0) | (taken <= len(free)))
    n, need = n * fits, need * fits
    first = taken - need
    rank = first[:, None] + column - have[:, None]
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    got = free[rank[fresh]]
    table[fresh] = got.to(torch.int32)
    s["uses"][got] = 1
    s["starts"][1:] = n.cumsum(0).to(torch.int32)
    lengths += n.to(torch.int32)
    # the rows' places
    row = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    there = seq < b
    seq = seq.clamp_max(b - 1)
    position = lengths[seq].long() - s["starts"][seq + 1] + row
    position = torch.where(there, position, torch.zeros_like(position))
    slot = table[seq, position // page].long() * page + position % page
    gone = torch.full_like(slot, -1)
    slots, positions = torch.where(there, slot, gone), torch.where(there, position, gone)
    # taken back
    to = torch.minimum(s["old"], lengths)
    back = (column >= ((to + page - 1) // page)[:, None]) & (table >= 0)
    s["uses"].index_add_(0, table[back], torch.full((1,), -1, dtype=torch.int32,
                                                    device=DEVICE).expand(int(back.sum())))
    table.masked_fill_(back, -1)
    lengths.copy_(to)
    return slots, positions.to(torch.int32), s["starts"], lengths, table, s["uses"]


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
    news, lengths = _counts(case)
    if case["kind"] == "pool":
        page, rows = case["page"], sum(news)
        need = sum((length + page - 1) // page - (length - n + page - 1) // page
                   for n, length in zip(news, lengths))
        # lengths there and back, starts, old lengths; slots and positions; the pool,
        # and each page's table entry and use, there and back
        return {"bytes": 28 * case["batch"] + 12 * rows + 4 * case["pages"] + 32 * need,
                "flops": 4 * rows}
    hk, d = case["kv_heads"], case["head_dim"]
    stored = hk * (d + d // 32 + 1)  # a position, K and V
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
    if case["kind"] == "pool":
        return _pool_exact(s)
    hk, d, page = case["kv_heads"], case["head_dim"], case["page"]
    news, lengths = _counts(case)
    rows = {"key": [], "value": []}  # of each sequence, [length, Hk, d]
    for i, length in enumerate(lengths):
        table = s["table"][i, :(length + page - 1) // page].long()
        n = len(table)
        for name in rows:
            x = s[name][table].view(n, hk, page // 32, 4, 16, 2, d // 32, 4).int()
            x = torch.stack((x % 16, x // 16), -1).flatten(-2)  # [g][c][n][s][e], [g][c][o][u][e]
            size = x % 8
            # one bit behind the leading one; below 1 in halves
            size = torch.where(size < 2, size.double() / 2,
                               (1 + size.double() % 2 / 2) * torch.exp2((size // 2 - 1).double()))
            x = torch.where(x >= 8, -size, size)
            e = s[name + "_exponent"][table].double() - 127
            if name == "key":
                x = x.permute(0, 2, 5, 4, 1, 6, 3, 7)  # [.., block, n, c, Hk, s, g, e]
                e = e.view(n, hk, page // 32, 16, 2, d // 32, 1, 1).permute(0, 2, 4, 3, 1, 5, 6, 7)
            else:
                x = x.unflatten(-1, (2, 4))  # [p, Hk, block, g, c, o, u, h, j]
                x = x.permute(0, 2, 7, 3, 8, 1, 6, 5, 4)  # [.., block, h, g, j, Hk, u, o, c]
                e = e.view(n, hk, page // 32, 2, 4, 4, 1, 1, 1).permute(0, 2, 3, 4, 5, 1, 6, 7, 8)
            rows[name].append((x * torch.exp2(e)).reshape(n * page, hk, d)[:length])
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
    got = []
    for name, x, group in (("key", s["k"], 32), ("value", s["v"], case["head_dim"])):
        y = torch.zeros(case["batch"], case["kv_heads"], max(lengths), case["head_dim"],
                        dtype=torch.float64, device=DEVICE)
        at = 0
        for i, (n, length) in enumerate(zip(news, lengths)):
            new = x[at:at + n].double().unflatten(-1, (-1, group))
            at += n
            step = torch.exp2(torch.ceil(torch.log2(
                new.abs().amax(-1, keepdim=True) / 7.0)).clamp(-100, 125))
            z = new / step
            # one bit behind the leading one, down to 0.5, up to 6
            ulp = torch.exp2(torch.floor(torch.log2(z.abs().clamp(1.0, 6.0))) - 1)
            z = (torch.round(z / ulp) * ulp).clamp(-6.0, 6.0)
            new = (z * step).flatten(-2)
            y[i, :, :length] = torch.cat((rows[name][i][:length - n], new)).transpose(0, 1)
        got.append(y)
    return got


def _pool_exact(s):
    page, rows, width = s["page"], s["rows"], s["table"].shape[1]
    table, uses = s["table"].cpu().numpy().copy(), s["uses"].cpu().numpy().copy()
    old, news = s["lengths"].cpu().tolist(), s["new_rows"].cpu().tolist()
    free = [p for p in range(len(uses)) if uses[p] == 0]
    starts, slots, positions = [0], [], []
    asked_rows = asked_pages = at = 0
    for i, (length, n) in enumerate(zip(old, news)):
        if length + n > width * page:
            starts.append(starts[-1])
            continue
        have = -(-length // page)
        need = -(-(length + n) // page) - have
        asked_rows, asked_pages = asked_rows + n, asked_pages + need
        if asked_rows > rows or (need and asked_pages > len(free)):
            starts.append(starts[-1])
            continue
        pages = list(table[i, :have]) + free[at:at + need]
        at += need
        for p in range(length, length + n):
            slots.append(int(pages[p // page]) * page + p % page)
            positions.append(p)
        starts.append(starts[-1] + n)
    rest = [-1] * (rows - len(slots))
    # (taken back: lengths, table and uses are as they were)
    return (np.array(slots + rest, dtype=np.int64), np.array(positions + rest, dtype=np.int32),
            np.array(starts, dtype=np.int32), np.array(old, dtype=np.int32), table, uses)
