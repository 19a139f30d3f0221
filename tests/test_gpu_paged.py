"""GPU checks of the paged KV cache (append, read) and of attention over it
against plain forms in 64 bits (paged_cases)."""
import itertools
import math

import pytest
import torch

from paged_cases import Plain, stored

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float8_e4m3fn, torch.int8]
NAMES = {torch.bfloat16: "bf16", torch.float8_e4m3fn: "e4m3", torch.int8: "int8"}


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def _rows(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g) * std).bfloat16()


def _tables(g, lengths, page, spare=2):
    """Pages in no order, and how many there are."""
    need = [(n + page - 1) // page for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n])
        at += n
    return tables, sum(need) + spare


class Run:
    """Sequences in a cache and in the plain form, appended to in steps."""

    def __init__(self, dtype, kv_heads, d, page, steps, seed=0):
        """steps: lists of new rows per sequence."""
        from parrot import PagedKVCache
        self.g = torch.Generator().manual_seed(seed)
        self.lengths = [0] * len(steps[0])
        total = [sum(s) for s in zip(*steps)]
        self.tables, pages = _tables(self.g, total, page)
        self.cache = PagedKVCache(pages, page, kv_heads, d, dtype)
        self.plain = Plain(dtype, kv_heads, d, len(total))
        self.kv_heads, self.d = kv_heads, d

    def batch(self, new):
        from parrot import PagedBatch
        return PagedBatch.from_lists(self.tables, self.lengths, new)

    def append(self, new, k=None, v=None):
        n = sum(new)
        k = _rows(self.g, n, self.kv_heads, self.d) if k is None else k
        v = _rows(self.g, n, self.kv_heads, self.d) if v is None else v
        self.lengths = [a + b for a, b in zip(self.lengths, new)]
        batch = self.batch(new)
        self.cache.append(k.cuda(), v.cuda(), batch)
        self.plain.append(k, v, new)
        return batch

    def attend(self, heads, new, batch, scale=None, window=None, sinks=0, q=None, gone=()):
        q = _rows(self.g, sum(new), heads, self.d, std=1.5) if q is None else q
        scale = self.d ** -0.5 if scale is None else scale
        got = self.cache.attend(q.cuda(), batch, scale=scale, window=window, sinks=sinks)
        ref, bound = self.plain.attend(q, new, scale, window, sinks, gone)
        off = (got.double().cpu() - ref).abs()
        assert torch.isfinite(got).all()
        worst = (off / bound.clamp_min(1e-30)).max().item() if off.numel() else 0.0
        print(f"worst error {worst:.3f} of the bound", flush=True)
        assert (off <= bound + 1e-30).all()
        return got


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------

# chunk edges inside a block, at its edge and past it; a sequence without new
# rows; single tokens; pages of one block and of several
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("kv_heads,d,page,steps", [
    (2, 96, 64, [[1, 1], [1, 31], [1, 0], [1, 1]]),
    (1, 64, 32, [[33, 0, 95], [32, 5, 1], [0, 64, 33]]),
    (3, 128, 128, [[257], [1], [63], [64]]),
    (2, 96, 96, [[100, 96, 3, 29], [1, 1, 1, 3]]),
])
def test_append_and_read(dtype, kv_heads, d, page, steps):
    run = Run(dtype, kv_heads, d, page, steps)
    for new in steps:
        print(f"append {NAMES[dtype]} {new} after {run.lengths}", flush=True)
        batch = run.append(new)
    longest = max(run.lengths) + 5
    key, value = run.cache.read(batch, longest)
    assert key.shape == value.shape == (len(run.lengths), kv_heads, longest, d)
    for i, n in enumerate(run.lengths):
        for got, want in ((key[i], run.plain.k[i]), (value[i], run.plain.v[i])):
            assert torch.equal(got[:, :n].double().cpu(), want.transpose(0, 1))
            assert not got[:, n:].any()
    # fewer positions than there are, into a slice of a longer cache
    room = [torch.full((len(run.lengths), kv_heads, 2 * longest, d), 7.0, dtype=torch.bfloat16,
                       device="cuda") for _ in range(2)]
    run.cache.read(batch, 40, out=tuple(x[:, :, 3:43] for x in room))
    for x, y in zip(room, (key, value)):
        n = min(40, longest)
        assert torch.equal(x[:, :, 3:3 + n], y[:, :, :n])
        assert (x[:, :, :3] == 7).all() and (x[:, :, 43:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_append_leaves_the_rest(dtype):
    """Other positions, pages and rows of no sequence stay as they are; a page id
    outside the cache and positions past the table take nothing."""
    from parrot import PagedBatch, PagedKVCache
    cache = PagedKVCache(6, 64, 2, 96, dtype)
    for x in (cache.key, cache.value):
        x.view(torch.uint8).fill_(0x31)
    for x in (cache.key_exponent, cache.value_exponent):
        if x is not None:
            x.fill_(0x77)
    g = torch.Generator().manual_seed(3)
    k, v = _rows(g, 80, 2, 96), _rows(g, 80, 2, 96)
    # rows 0-2 nobody's, then 40 at 30 .. 69 over pages 4 and 1, 20 on pages that
    # are not there, 7 of which 5 lie past the table; the rest nobody's
    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = PagedBatch(i32([[4, 1], [-1, 6], [3, -1]]), i32([70, 100, 133]), i32([3, 43, 63, 70]))
    before = [x.clone() for x in (cache.key, cache.value)]
    whole = cache.read(PagedBatch(i32([[0], [1], [2], [3], [4], [5]]), i32([64] * 6),
                                  i32([0] * 7)), 64)
    cache.append(k.cuda(), v.cuda(), batch)
    after = cache.read(PagedBatch(i32([[0], [1], [2], [3], [4], [5]]), i32([64] * 6),
                                  i32([0] * 7)), 64)
    for x, y, rows in ((whole[0], after[0], k), (whole[1], after[1], v)):
        want = x.clone()
        new = stored(rows[3:43], dtype).transpose(0, 1).to(torch.bfloat16).cuda()
        want[4, :, 30:] = new[:, :34]
        want[1, :, :6] = new[:, 34:]
        assert torch.equal(y, want)
    for x, y in zip(before, (cache.key, cache.value)):
        changed = (x.view(torch.uint8) != y.view(torch.uint8)).flatten(1).any(1).tolist()
        assert changed == [False, True, False, False, True, False]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=NAMES.get)
def test_rows_of_every_size(dtype):
    """Zeros, the smallest and largest numbers, halves of steps, single large
    values, and rows that hold a NaN or an infinity."""
    d = 64
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(d), torch.full((d,), -0.0), torch.full((d,), 1e-40),
            torch.full((d,), 3.3e38), torch.linspace(-448, 448, d), torch.linspace(-127, 127, d),
            torch.arange(d) / 2.0, torch.arange(d) * 2.0 ** -120, 2.0 ** torch.arange(-63.0, 1)]
    for p in range(-30, 31, 6):
        rows.append(torch.randn(d, generator=g) * 2.0 ** p)
    # just under and over the powers at which the scale steps
    for top in (448.0, 449.0, 450.0, 127.0, 127.5, 128.0, 1.75, 1.7578125, 1.984375, 1.9921875):
        x = torch.randn(d, generator=g) * 0.3 * top
        x = x.clamp(-top, top)
        x[7] = -top
        rows.append(x)
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.randn(d, generator=g)
        x[11] = bad
        rows.append(x)
    rows = torch.stack(rows).bfloat16()[:, None]
    run = Run(dtype, 1, d, 64, [[len(rows)]])
    batch = run.append([len(rows)], rows, rows.flip(0))
    for got, x in zip(run.cache.read(batch, len(rows)), (rows, rows.flip(0))):
        got, want = got[0, 0].double().cpu(), stored(x, dtype)[:, 0]
        assert torch.equal(got.isnan(), want.isnan()) and want.isnan().any()
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

LAYOUTS = [(8, 2, 96), (4, 4, 64), (6, 2, 128), (16, 1, 64), (5, 1, 96)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("steps,window,sinks", [
    ([[1]], None, 0),                                   # a first token alone
    ([[31, 32, 33, 64], [1, 1, 1, 1]], None, 0),        # single tokens past block edges
    ([[200, 7, 0, 65], [3, 0, 9, 40]], 50, 0),          # ragged chunks, one sequence idle
    ([[300, 500], [1, 2]], 100, 5),                     # sinks far from the window
    ([[130, 97], [33, 64]], 40, 70),                    # more sinks than window
    ([[70]], 1, 0), ([[70]], 1, 33), ([[90]], 64, 30),  # one key; sinks that join the window
])
def test_attend(dtype, heads, kv_heads, d, steps, window, sinks):
    print(f"attend {NAMES[dtype]} {heads}/{kv_heads} of {d}, {steps}, window {window} + {sinks}",
          flush=True)
    run = Run(dtype, kv_heads, d, 64, steps, seed=len(steps) + d)
    for new in steps:
        batch = run.append(new)
        run.attend(heads, new, batch, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 16, 96), (16, 16, 64), (32, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 0), (70, 40), (1, 0)])
def test_attend_many_rows(dtype, heads, kv_heads, d, window, sinks):
    """Tiles of 128 rows: many sequences with ragged chunks after ragged contexts."""
    g = torch.Generator().manual_seed(d)
    first = torch.randint(0, 200, (24,), generator=g).tolist()
    then = torch.randint(40, 260, (24,), generator=g).tolist()
    then[3] = 0
    run = Run(dtype, kv_heads, d, 64, [first, then])
    run.append(first)
    batch = run.append(then)
    run.attend(heads, then, batch, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("steps,page,window,sinks", [
    ([[3000, 900], [1, 1]], 32, None, 0),       # long contexts, split over workgroups
    ([[3000, 900], [1, 6]], 256, 2048, 4),
    ([[1500], [200]], 96, None, 0),             # a chunk over a context
    ([[700, 333], [513, 260]], 64, 300, 40),    # hundreds of rows
])
def test_attend_long(dtype, steps, page, window, sinks):
    run = Run(dtype, 2, 96, page, steps, seed=page)
    for new in steps:
        print(f"attend {NAMES[dtype]} {new} after {run.lengths}", flush=True)
        batch = run.append(new)
        run.attend(8, new, batch, window=window, sinks=sinks)


def test_attend_scales_and_strides():
    """Negative and large scales; rows of a packed projection, strides that the
    kernels do not read in place, an offset that is not aligned."""
    run = Run(torch.bfloat16, 2, 64, 32, [[77, 40]])
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


def test_rows_without_keys():
    """More new rows than positions, lengths of zero, pages that are not there: 0
    where a row sees nothing, and rows of no sequence left as they are."""
    from parrot import PagedBatch
    run = Run(torch.bfloat16, 1, 64, 32, [[64, 64, 10]])
    run.append([64, 64, 10])
    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    table = [run.tables[0], run.tables[1], run.tables[2] + [-1]]
    q = _rows(run.g, 30, 2, 64)
    for kw in ({}, {"window": 8, "sinks": 1}):
        # 12 rows of which the last 4 have positions; 5 rows of an empty sequence;
        # 6 whose pages are not there; 3 rows of nobody
        table_t = i32([table[0], [9999, -7], table[2]])
        batch = PagedBatch(table_t, i32([4, 0, 10]), i32([0, 12, 17, 23]))
        out = torch.full((30, 128), 3.0, dtype=torch.bfloat16, device="cuda")
        got = run.cache.attend(q.cuda(), batch, scale=0.125, out=out, **kw)
        assert got is out
        assert not got[:8].any() and not got[12:17].any() and (got[23:] == 3).all()
        part = Plain(torch.bfloat16, 1, 64, 1)
        part.k, part.v = [run.plain.k[0][:4]], [run.plain.v[0][:4]]
        ref, bound = part.attend(q[8:12], [4], 0.125, kw.get("window"), kw.get("sinks", 0))
        assert ((got[8:12].double().cpu() - ref).abs() <= bound).all()
        gone = PagedBatch(i32([[9999, -7], [-1, -1]]), i32([40, 64]), i32([0, 12, 20]))
        out.fill_(3.0)
        run.cache.attend(q.cuda(), gone, scale=0.125, out=out, **kw)
        assert not out[:20].any() and (out[20:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_pages_given_back(dtype):
    """Pages that the window has left are not read: their ids may name nothing."""
    run = Run(dtype, 2, 96, 32, [[500], [1]])
    run.append([500])
    batch = run.append([1])
    q = _rows(run.g, 1, 8, 96)
    want = run.attend(8, [1], batch, window=100, sinks=20, q=q)
    run.tables = [[p if i < 1 or i >= 12 else -1 for i, p in enumerate(run.tables[0])]]
    assert torch.equal(run.attend(8, [1], run.batch([1]), window=100, sinks=20, q=q), want)
    # ... and where the window does reach them, they are not seen
    run.tables = [[p if i != 14 else run.cache.key.shape[0] for i, p in enumerate(run.tables[0])]]
    run.attend(8, [1], run.batch([1]), window=100, sinks=20, q=q, gone=[(0, 448, 480)])


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("last", [73, 100, 110, 118, 150])
# tiles of 16 rows, of 32, and (many sequences with many rows) of 128
@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (15, 1), (73, 1), (73, 128)])
def test_unseen_rows_do_not_reach_a_row(dtype, bad, last, n, copies):
    """Infinities and NaN among keys and values that a row does not see: later
    positions of its own chunk, positions the window has left (in a block that it
    still covers), and stale ones past the length.  copies: sequences of the same
    pages, to all of which the same must come out."""
    run = Run(dtype, 2, 96, 64, [[150]])
    k, v = _rows(run.g, 150, 2, 96), _rows(run.g, 150, 2, 96)
    k[77, 0, 5] = v[77, 0, 5] = bad
    v[101, 1, 50] = bad
    run.append([150], k, v)
    # a sequence of the first `last` positions, of which n are its new rows
    run.lengths = [last]
    run.tables, run.lengths = run.tables * copies, run.lengths * copies
    batch = run.batch([n] * copies)
    q = _rows(run.g, n, 8, 96, std=1.5)
    for window, sinks in ((20, 0), (20, 3), (None, 0)):
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), batch, scale=0.1, window=window,
                               sinks=sinks).view(copies, n, 2, 4, 96)
        assert torch.equal(got.view(torch.int16), got[:1].view(torch.int16).expand_as(got))
        got = got[0].double().cpu()
        # the same without the bad rows
        kc, vc = k[:last].clone(), v[:last].clone()
        for head, row in ((0, 77), (1, 101)):
            if row < last:
                kc[row, head], vc[row, head] = 0 if row == 77 else kc[row, head], 0
        clean = Plain(dtype, 2, 96, 1)
        clean.append(kc, vc, [last])
        ref, bound = clean.attend(q, [n], 0.1, window, sinks)
        ref, bound = ref.view(n, 2, 4, 96), bound.view(n, 2, 4, 96)
        pos = torch.arange(last - n, last)
        for head, row in ((0, 77), (1, 101)):
            sees = (pos >= row) & (pos < row + (window or last))
            assert ((got[:, head] - ref[:, head]).abs() <= bound[:, head])[~sees].all()
            # and where a row does see it, it is not finite either (all of the
            # row's, or that value's dimension)
            assert not torch.isfinite(got[:, head][sees]).all(-1).any()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (75, 1), (75, 40)])  # tiles as above
def test_pages_missing_inside(dtype, n, copies):
    """Pages that are not there between pages that are, at either block of a pair, one
    and several at a time: their positions are not seen."""
    run = Run(dtype, 2, 96, 32, [[900], [n]])
    run.append([900])
    run.append([n])
    missing = [3, 6, 7, 12, 13, 14, 20, 25]
    run.tables = [[-1 if i in missing else p for i, p in enumerate(run.tables[0])]]
    gone = [(0, 32 * i, 32 * i + 32) for i in missing]
    q = _rows(run.g, n, 8, 96)
    for window in (None, 300):
        want = run.attend(8, [n], run.batch([n]), window=window, sinks=40, q=q, gone=gone)
        if copies == 1:
            continue
        run.tables, run.lengths = run.tables * copies, run.lengths * copies
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), run.batch([n] * copies),
                               scale=96 ** -0.5, window=window, sinks=40)
        run.tables, run.lengths = run.tables[:1], run.lengths[:1]
        got = got.double().cpu().view(copies, n, -1)
        assert torch.equal(got, got[:1].expand_as(got))
        ref, bound = run.plain.attend(q, [n], 96 ** -0.5, window, 40, gone)
        assert ((got[0] - ref).abs() <= bound).all()
        assert ((got[0] - want.double().cpu()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_shared_pages(dtype):
    """Sequences that begin with the same pages."""
    run = Run(dtype, 2, 64, 32, [[160, 0, 0], [1, 7, 100]])
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
    (8, 2, 400, 1, 8400),    # tiles of 16 rows: 263 blocks, every fourth by one wavefront
    (16, 2, 260, 6, 8400),   # of 32
    (32, 32, 31, 128, 3000),  # of 128: 98 blocks
])
def test_shares_of_many_blocks(heads, kv_heads, others, new, length):
    """One long sequence among so many that no tile's keys are split: more blocks than
    are looked up at once."""
    print(f"{length} keys, {new} new rows, {others} other sequences", flush=True)
    steps = [[length] + [0] * others, [new] * (others + 1)]
    run = Run(torch.int8, kv_heads, 64, 32, steps)
    for now in steps:
        batch = run.append(now)
    run.attend(heads, steps[-1], batch)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,copies", [(1, 1), (6, 1), (75, 1), (75, 40)])
def test_tables_of_no_pages_and_endless_windows(dtype, n, copies):
    """Tables without a column hold nothing; a window and sinks as large as they get
    hide nothing."""
    from parrot import PagedBatch
    run = Run(dtype, 2, 64, 32, [[90], [n]])
    run.append([90])
    batch = run.append([n])
    q = _rows(run.g, n, 8, 64)
    want = run.attend(8, [n], batch, scale=0.1, q=q)
    many = q.cuda().repeat(copies, 1, 1)
    batch = PagedBatch.from_lists(run.tables * copies, run.lengths * copies, [n] * copies)
    for kw in ({"window": 2 ** 31 - 1}, {"window": 2 ** 40, "sinks": 2 ** 40},
               {"window": 1, "sinks": 2 ** 31 - 1}):
        got = run.cache.attend(many, batch, scale=0.1, **kw).view(copies, n, -1)
        ref, bound = run.plain.attend(q, [n], 0.1)
        assert ((got.double().cpu() - ref).abs() <= bound).all() and want.shape == got.shape[1:]
    none = PagedBatch.from_lists([[]] * copies, [90 + n] * copies, [n] * copies)
    before = [x.clone() for x in run.cache.read(run.batch([n]), 90 + n)]
    run.cache.append(many[:, :2], many[:, 2:4], none)
    assert not run.cache.attend(many, none, scale=0.1).any()
    assert not any(x.any() for x in run.cache.read(none, 50))
    for x, y in zip(before, run.cache.read(run.batch([n]), 90 + n)):
        assert torch.equal(x, y)


def test_far_pages():
    """Pages past 2^31 and 2^32 elements and bytes."""
    from parrot import PagedBatch, PagedKVCache
    page, d = 128, 128
    pages = (1 << 32) // (2 * page * d) + 300
    for dtype in (torch.int8, torch.bfloat16):
        print(f"far pages {NAMES[dtype]}", flush=True)
        cache = PagedKVCache(pages, page, 2, d, dtype)
        g = torch.Generator().manual_seed(1)
        k, v, q = _rows(g, 300, 2, d), _rows(g, 300, 2, d), _rows(g, 300, 4, d)
        tables = [[pages - 1, 0, pages // 2]]
        batch = PagedBatch.from_lists(tables, [300], [300])
        cache.append(k.cuda(), v.cuda(), batch)
        plain = Plain(dtype, 2, d, 1)
        plain.append(k, v, [300])
        got = cache.attend(q.cuda(), batch, scale=0.1)
        ref, bound = plain.attend(q, [300], 0.1)
        assert ((got.double().cpu() - ref).abs() <= bound).all()
        key, value = cache.read(batch, 300)
        assert torch.equal(key[0].double().cpu(), plain.k[0].transpose(0, 1))
        assert torch.equal(value[0].double().cpu(), plain.v[0].transpose(0, 1))
        del cache
        torch.cuda.empty_cache()


def test_many_sequences():
    """More sequences than a wavefront has lanes, most of them without new rows."""
    g = torch.Generator().manual_seed(2)
    first = torch.randint(0, 40, (150,), generator=g).tolist()
    then = torch.randint(0, 3, (150,), generator=g).tolist()
    run = Run(torch.float8_e4m3fn, 1, 64, 32, [first, then])
    for new in (first, then):
        batch = run.append(new)
        run.attend(2, new, batch, window=17, sinks=2)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("heads,kv_heads,d,new,length,window,sinks,copies", [
    (8, 2, 96, 5, 4096, 2048, 0, 64), (8, 2, 96, 5, 4096, 2048, 0, 36),
    (8, 2, 96, 1025, 4096, 2048, 0, 4), (8, 2, 96, 465, 1465, 1000, 0, 1),
    (8, 8, 64, 337, 1337, 1024, 0, 16), (16, 2, 128, 1172, 1172, 1000, 0, 1),
    (8, 2, 64, 1025, 3000, 1024, 70, 4),
])
def test_split_windows_with_short_last_tiles(dtype, heads, kv_heads, d, new, length, window, sinks,
                                             copies):
    """A sequence's last tile spans fewer positions than the others and sees fewer of
    the window's blocks, in calls that split the keys.  copies: sequences of the same
    pages, to all of which the same must come out."""
    print(f"{copies} x {new} of {length}, {heads} on {kv_heads} of {d}, window {window} + {sinks}",
          flush=True)
    run = Run(dtype, kv_heads, d, 64, [[length]])
    run.append([length])
    q = _rows(run.g, new, heads, d, std=1.5)
    run.tables, run.lengths = run.tables * copies, run.lengths * copies
    got = run.cache.attend(q.cuda().repeat(copies, 1, 1), run.batch([new] * copies), scale=d ** -0.5,
                           window=window, sinks=sinks).view(copies, new, -1)
    assert torch.equal(got, got[:1].expand_as(got))
    ref, bound = run.plain.attend(q, [new], d ** -0.5, window, sinks)
    assert ((got[0].double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("new", [5, 40, 2000])
@pytest.mark.parametrize("window,sinks", [(1000, 0), (1000, 5), (300, 0), (None, 0)])
def test_tables_shorter_than_the_lengths(dtype, new, window, sinks):
    """Positions past the table are not stored: no row sees them, and the last rows'
    window may hold nothing else."""
    run = Run(dtype, 2, 96, 64, [[3200]])
    run.append([3200])
    run.tables = [run.tables[0][:32]]
    run.attend(8, [new], run.batch([new]), window=window, sinks=sinks, gone=[(0, 2048, 3200)])


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
# tiles of 16 rows, of 32, and of 128, as above
@pytest.mark.parametrize("n,copies", [(1, 1), (15, 1), (73, 1), (73, 128)])
def test_largest_rows(dtype, n, copies):
    """Keys and values up to the largest bf16 numbers, zeros among them: scores by
    queries as small, values where a row sees one key."""
    run = Run(dtype, 2, 64, 32, [[150]])
    g = run.g
    large = torch.randint(-3, 4, (150, 2, 64), generator=g) / 3 * 3.3e38
    large[::3] = torch.randint(-2, 3, (50, 2, 64), generator=g) * 2.0 ** 126
    large[1::5] = torch.randint(-1, 2, (30, 2, 64), generator=g) * 2.0 ** 127
    large, usual = large.bfloat16(), _rows(g, 150, 2, 64)
    assert torch.isfinite(large).all()
    q = (torch.randint(-3, 4, (n, 8, 64), generator=g) * 2.0 ** -125).bfloat16()
    for k, v, kw in ((large, usual, {}), (large, usual, {"window": 40, "sinks": 3}),
                     (usual, large, {"window": 1}), (large, large, {"window": 1})):
        run.lengths = [0]
        run.plain = Plain(dtype, 2, 64, 1)
        run.append([150], k, v)
        lengths, tables = run.lengths, run.tables
        run.tables, run.lengths = tables * copies, lengths * copies
        got = run.cache.attend(q.cuda().repeat(copies, 1, 1), run.batch([n] * copies), scale=0.1,
                               **kw).view(copies, n, -1)
        run.tables, run.lengths = tables, lengths
        assert torch.equal(got, got[:1].expand_as(got))
        ref, bound = run.plain.attend(q, [n], 0.1, kw.get("window"), kw.get("sinks", 0))
        assert ((got[0].double().cpu() - ref).abs() <= bound).all(), kw


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_a_cache_takes_its_own_memory_only(dtype):
    """No tensor beside the four that are kept is made, not for a moment either."""
    from parrot import PagedKVCache
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    cache = PagedKVCache(4096, 64, 2, 128, dtype)
    size = sum(x.numel() * x.element_size() for x in (
        cache.key, cache.value, cache.key_exponent, cache.value_exponent) if x is not None)
    assert torch.cuda.max_memory_allocated() - before <= size + 4096
    assert not cache.key.view(torch.uint8).any() and not cache.value.view(torch.uint8).any()


def test_read_refuses_outputs_that_it_cannot_write():
    """Of another shape, type or device, strides that are not multiples of 4, one place for
    two positions."""
    run = Run(torch.int8, 2, 64, 32, [[40, 9]])
    batch = run.append([40, 9])
    good = torch.empty(2, 2, 40, 64, dtype=torch.bfloat16, device="cuda")
    run.cache.read(batch, 40, out=(good, good.clone()))
    for bad in (good[:, :, :39], good.float(), good.cpu(), good.repeat(1, 1, 1, 2)[..., ::2],
                torch.empty(2, 2, 40, 66, dtype=torch.bfloat16, device="cuda")[..., :64],
                good[:, :, :1].expand(2, 2, 40, 64), good[:1].expand(2, 2, 40, 64)):
        for pair in ((good, bad), (bad, good)):
            with pytest.raises(RuntimeError):
                run.cache.read(batch, 40, out=pair)


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------

def test_captured_steps():
    """Append and attention captured once, replayed for growing sequences: every
    replay as the eager calls; two graphs at once over two caches."""
    from parrot import PagedBatch
    steps = [[600, 90]] + [[1, 1]] * 12
    runs = [Run(t, 2, 96, 64, steps, seed=i) for i, t in enumerate(TYPES[:2])]
    held = []
    for run in runs:
        run.append([600, 90])
        k, v, q = (torch.empty(2, h, 96, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 8))
        lengths = torch.tensor(run.lengths, dtype=torch.int32, device="cuda")
        batch = PagedBatch(run.batch([1, 1]).table, lengths,
                           torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))

        def step(run=run, k=k, v=v, q=q, lengths=lengths, batch=batch):
            lengths.add_(1)
            run.cache.append(k, v, batch)
            return run.cache.attend(q, batch, scale=0.1, window=400, sinks=8)
        graph = torch.cuda.CUDAGraph()
        for x in (k, v, q):
            x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step()
        held.append((graph, out, k, v, q, batch))
    for i in range(10):
        news = []
        for run, (graph, out, k, v, q, _) in zip(runs, held):
            new = [_rows(run.g, 2, h, 96) for h in (2, 2, 8)]
            for x, y in zip((k, v, q), new):
                x.copy_(y)
            news.append(new)
        for _, (graph, *_) in zip(runs, held):
            graph.replay()
        torch.cuda.synchronize()
        for run, (graph, out, *_), (k, v, q) in zip(runs, held, news):
            run.plain.append(k, v, [1, 1])
            run.lengths = [n + 1 for n in run.lengths]
            ref, bound = run.plain.attend(q, [1, 1], 0.1, 400, 8)
            assert ((out.double().cpu() - ref).abs() <= bound).all(), i
            assert torch.equal(out, run.cache.attend(q.cuda(), run.batch([1, 1]), scale=0.1,
                                                     window=400, sinks=8))
        torch.zeros(1 << 20, device="cuda").sum().item()  # eager work in between


def test_two_streams():
    """The same cache read from two streams at once gives what one stream gives."""
    run = Run(torch.int8, 2, 96, 64, [[2500, 1800], [1, 1]])
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
    for y, w in zip(got, itertools.cycle(want)):
        assert torch.equal(y, w)
