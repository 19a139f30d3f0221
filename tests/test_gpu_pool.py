"""GPU checks of the page pool against a plain form (pool_cases)."""
import random

import pytest
import torch

from pool_cases import PlainPool, pages_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Both:
    """A pool and a batch on the GPU, and the plain form."""

    def __init__(self, uses, page, table, lengths):
        from parrot import PagedBatch, PagePool
        self.plain = PlainPool(uses, page, table, lengths)
        b = len(lengths)
        self.pool = PagePool.from_uses(i32(uses), page)
        self.batch = PagedBatch(i32(table).view(b, -1 if b else 0), i32(lengths),
                                i32([7] * (b + 1)))

    @classmethod
    def filled(cls, rng, b, width, page, pages, most):
        """Sequences of up to `most` positions on pages in no order, some others in use."""
        order = list(range(pages))
        rng.shuffle(order)
        uses, table, lengths = [0] * pages, [], []
        for _ in range(b):
            n = rng.randint(0, most)
            need = pages_of(n, page)
            if need > min(width, len(order)):
                n = need = 0
            row = [order.pop() for _ in range(need)]
            for p in row:
                uses[p] = 1
            table.append(row + [-1] * (width - need))
            lengths.append(n)
        for p in order[:len(order) // 4]:
            uses[p] = rng.randint(1, 3)
        for p in order[len(order) // 4:len(order) // 3]:
            uses[p] = -1
        return cls(uses, page, table, lengths)

    def check(self):
        assert self.batch.lengths.tolist() == self.plain.lengths
        assert self.batch.table.tolist() == self.plain.table
        assert self.pool.uses.tolist() == self.plain.uses

    def extend(self, new, rows):
        want = self.plain.extend(new, rows)
        got = self.pool.extend(self.batch, i32(new), rows)
        assert got[0].dtype == torch.int64 and got[1].dtype == torch.int32
        assert self.batch.starts.tolist() == self.plain.starts
        assert got[1].tolist() == want[1] and got[0].tolist() == want[0]
        self.check()

    def release(self, lengths=None, **kw):
        self.plain.release(lengths, **kw)
        self.pool.release(self.batch, None if lengths is None else i32(lengths), **kw)
        self.check()


# one sequence, a wavefront's number and more, more than a workgroup's, more than LDS holds;
# pools of a few pages and of more than a workgroup reads at once; plenty and too few
@pytest.mark.parametrize("b,width,page,pages,most,new,seed", [
    (1, 4, 32, 7, 40, 30, 0), (1, 1, 64, 1, 0, 64, 1), (3, 5, 96, 40, 300, 90, 2),
    (65, 9, 32, 700, 200, 40, 3), (65, 9, 32, 300, 200, 100, 4), (400, 20, 64, 9000, 1000, 7, 5),
    (1025, 3, 32, 3000, 64, 33, 6), (1025, 3, 32, 700, 40, 33, 7), (5000, 2, 32, 9000, 50, 20, 8),
    (5000, 2, 32, 1500, 10, 60, 9), (70, 130, 32, 5000, 2000, 2000, 10),
    (6, 40, 32, 70001, 900, 300, 11), (40, 700, 64, 140000, 30000, 9000, 12),
])
def test_extend_and_release(b, width, page, pages, most, new, seed):
    rng = random.Random(seed)
    both = Both.filled(rng, b, width, page, pages, most)
    for step in range(6):
        print(f"{b} sequences, {pages} pages, step {step}", flush=True)
        news = [rng.choice([0, 1, rng.randint(-3, new), new]) for _ in range(b)]
        total = sum(max(n, 0) for n in news)
        both.extend(news, rng.choice([total, total + 9, total // 2, max(total - 1, 0)]))
        if step % 3 == 0:  # some tokens turned down, some sequences done
            both.release([rng.choice([0, n, max(n - 1, 0), n + 5, max(n - new, -1)])
                          for n in both.plain.lengths])
        elif step % 3 == 1:
            both.release(window=rng.choice([1, 33, page, 2 * page, 10 ** 12]),
                         sinks=rng.choice([0, 1, page, page + 1]))
        else:
            both.release([max(n - 3, 0) for n in both.plain.lengths], window=rng.randint(1, most + 2),
                         sinks=rng.choice([0, 4]))


def test_edges_of_a_page():
    """Lengths one before, at and past the end of a page and of the table; new rows that
    fill it and pass it."""
    lengths = [0, 31, 32, 33, 63, 64, 95, 96, 96, 96]
    for n in (1, 2, 32, 33, 96, 97):
        table, at = [], 0
        for x in lengths:
            need = pages_of(x, 32)
            table.append(list(range(at, at + need)) + [-1] * (3 - need))
            at += need
        both = Both([1] * at + [0] * 40, 32, table, lengths)
        both.extend([n] * 9 + [0], 1000)
        both.release(lengths)
        both.extend([n] * 9 + [0], 5 * n)
        both.release([0] * 10)
    assert not both.pool.uses.any() and (both.batch.table == -1).all()


def test_numbers_that_do_not_fit():
    """Lengths below 0 and past the table, new rows of 2^31 - 1, ids outside the pool, no
    pages, no columns, no rows, no sequences: bounded, as the plain form has it."""
    both = Both([0, 0, 0], 32, [[-1, -1], [5, -7], [2, 99], [1, -1]], [-5, 40, 9000, 3])
    both.extend([2 ** 31 - 1, 20, 1, 30], 90)
    both.extend([40, 1, 2 ** 31 - 1, -2 ** 31], 2)
    both.release([-1, 2 ** 31 - 1, 8000, 2], window=1)
    both.release([0, 0, 0, 0])
    many = Both([1] * 9 + [0] * 3, 32, [[-1] * 3] * 70, [0] * 70)
    many.extend([2 ** 31 - 1] * 69 + [1], 4)
    many.extend([96] * 70, 2 ** 12)
    for uses, table, lengths in (([], [[-1], [-1]], [0, 0]), ([0, 0], [[], []], [0, 3]),
                                 ([0, 1], [], [])):
        none = Both(uses, 64, table, lengths)
        none.extend([1] * len(lengths), 3)
        none.extend([0] * len(lengths), 0)
        none.release([0] * len(lengths))
        none.release(window=5)


def test_shared_pages():
    """Two sequences on one beginning: its pages are free once both have let go."""
    both = Both([0] * 8, 32, [[-1] * 4] * 3, [0] * 3)
    both.extend([70, 0, 0], 70)
    for form in (both.plain.table, both.batch.table):  # the second begins with two whole pages
        form[1][:2] = form[0][:2]
    both.plain.lengths[1] = 64
    both.batch.lengths[1] = 64
    for p in both.plain.table[0][:2]:
        both.plain.uses[p] += 1
        both.pool.uses[p] += 1
    both.extend([1, 40, 0], 41)
    both.release([0, 104, 0])
    both.extend([0, 0, 120], 120)
    both.release([0, 64, 120])
    both.release([0, 0, 0])
    assert not both.pool.uses.any()


def test_long_tables():
    """Tables of thousands of pages, in one sequence and in a few: rows by the thousand."""
    rng = random.Random(3)
    both = Both.filled(rng, 3, 3000, 32, 12000, 40000)
    both.extend([50000, 20000, 3], 70100)
    both.release(window=4000, sinks=100)
    both.release([n // 2 for n in both.plain.lengths])
    both.extend([9000, 9000, 9000], 27000)


def test_the_same_again():
    """What is handed out depends on the numbers alone."""
    rng = random.Random(4)
    both = Both.filled(rng, 300, 40, 32, 9000, 600)
    new = i32([rng.randint(0, 500) for _ in range(300)])
    state = (both.batch.table, both.batch.lengths, both.pool.uses)
    before, first = [x.clone() for x in state], None
    for _ in range(20):
        for x, y in zip(state, before):
            x.copy_(y)
        got = [*both.pool.extend(both.batch, new, 80000), *(x.clone() for x in state)]
        both.pool.release(both.batch, before[1])
        assert all(torch.equal(x, y) for x, y in zip(state, before)) or \
            (before[2] < 0).any()  # (a use below 0 is 0 after a turn)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


def test_refusals():
    from parrot import PagedBatch, PagePool
    pool = PagePool(9, 32)
    batch = PagedBatch.from_lists([[0], [1]], [5, 6], [1, 1])
    good = i32([1, 1])
    pool.extend(batch, good, 2)
    for bad in (good.long(), i32([1]), i32([1, 1, 1]), i32([[1, 1]]), good.cpu(), i32([1, 0, 1])[::2]):
        with pytest.raises(RuntimeError):
            pool.extend(batch, bad, 2)
        with pytest.raises(RuntimeError):
            pool.release(batch, bad)
    for rows in (-1, (1 << 30) + 1):
        with pytest.raises(RuntimeError):
            pool.extend(batch, good, rows)
    for kw in ({"window": 0}, {"window": -3}, {"sinks": -1}):
        with pytest.raises(RuntimeError):
            pool.release(batch, **kw)
    with pytest.raises(RuntimeError):
        pool.extend(PagedBatch.from_lists([[0], [1]], [5, 6], [1, 1], device="cpu"), good, 2)


# ---------------------------------------------------------------------------
# as a server uses them: a pool, caches of every type and attention in one captured step
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float4_e2m1fn_x2, torch.float8_e4m3fn])
def test_a_captured_loop(dtype):
    """Sequences that grow by one or a few tokens a step, give back what the window has
    left, end and begin again, in one graph that is replayed: each step as the same calls
    on pages that were given by hand."""
    from parrot import PagedBatch, PagedKVCache, PagePool
    b, heads, kv_heads, d, page, width, rows = 3, 8, 2, 96, 32, 40, 24
    window, sinks = 70, 33
    g = torch.Generator().manual_seed(6)
    # (as many pages as the windows need, fewer than the whole sequences would)
    pool, cache = PagePool(30, page), PagedKVCache(30, page, kv_heads, d, dtype)
    batch = PagedBatch(i32([[-1] * width] * b), i32([0] * b), i32([0] * (b + 1)))
    k, v, q = (torch.zeros(rows, h, d, dtype=torch.bfloat16, device="cuda")
               for h in (kv_heads, kv_heads, heads))
    new, keep = i32([0] * b), i32([0] * b)

    def step():
        pool.release(batch, keep)
        places = pool.extend(batch, new, rows)
        cache.append(k, v, batch)
        y = cache.attend(q, batch, scale=0.1, window=window, sinks=sinks)
        pool.release(batch, window=window, sinks=sinks)
        return (y, *places)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    # the same sequences, all of their pages kept
    whole = PagedKVCache(b * width, page, kv_heads, d, dtype)
    tables = [list(range(i * width, (i + 1) * width)) for i in range(b)]
    lengths = [0] * b
    for t in range(60):
        news = [(7 + t) % 9, 1, 0 if t % 5 else 13]
        keeps = [0 if t == 25 else lengths[0], lengths[1] - (t % 4 == 3), lengths[2]]
        lengths = [a + n for a, n in zip(keeps, news)]
        total = sum(news)
        fresh = [torch.randn(rows, h, d, generator=g).bfloat16() for h in (kv_heads, kv_heads, heads)]
        for x, y in zip((k, v, q, new, keep), (*fresh, i32(news), i32(keeps))):
            x.copy_(y)
        graph.replay()
        byhand = PagedBatch.from_lists(tables, lengths, news)
        whole.append(k, v, byhand)
        want = whole.attend(q, byhand, scale=0.1, window=window, sinks=sinks)
        assert torch.equal(out[0][:total], want[:total]), t
        assert batch.lengths.tolist() == lengths
        positions = [p for n, length in zip(news, lengths) for p in range(length - n, length)]
        assert out[2].tolist() == positions + [-1] * (rows - total)
        assert (out[1][:total] >= 0).all()
        # (a window's pages, one for a page half in it, the sinks' two)
        assert int(pool.uses.sum()) <= b * 6 and int((batch.table >= 0).sum()) == int(pool.uses.sum())
        torch.zeros(1 << 20, device="cuda").sum().item()  # eager work in between
    pool.release(batch, i32([0] * b))
    assert not pool.uses.any()


def test_captured_steps_of_many_rows():
    """Steps whose rows a second launch places, of two pools in two graphs that are
    replayed in turn: each as the plain form."""
    rng = random.Random(8)
    sides = []
    for b, width, page, pages, rows in ((60, 90, 32, 5000, 9000), (1100, 3, 64, 3000, 20000)):
        both = Both.filled(rng, b, width, page, pages, 70)
        new, keep = i32([0] * b), i32(both.plain.lengths)

        def step():
            places = both.pool.extend(both.batch, new, rows)
            both.pool.release(both.batch, keep)
            return places
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        sides.append((both, new, keep, rows, graph, out))
    for t in range(6):
        for both, new, keep, rows, graph, out in sides:
            b = len(both.plain.lengths)
            news = [rng.choice([0, 1, rng.randint(2, 400)]) for _ in range(b)]
            keeps = [rng.choice([0, n, n + 9, n + 500]) for n in both.plain.lengths]
            new.copy_(i32(news))
            keep.copy_(i32(keeps))
            torch.zeros(1 << 20, device="cuda").sum().item()  # eager work in between
            graph.replay()
            want = both.plain.extend(news, rows)
            assert both.batch.starts.tolist() == both.plain.starts, t
            assert out[0].tolist() == want[0] and out[1].tolist() == want[1], t
            both.plain.release(keeps)
            both.check()


def test_slots_index_what_lies_by_page():
    """A per-token tensor [pages * page_size, ...] written and read by slots."""
    from parrot import PagedBatch, PagePool
    pool = PagePool(20, 32)
    batch = PagedBatch(i32([[-1] * 4] * 2), i32([0, 0]), i32([0] * 3))
    latents = torch.zeros(20 * 32, 8, device="cuda")
    kept = [[], []]
    for new in ([40, 3], [1, 1], [0, 50], [7, 7]):
        slots, positions = pool.extend(batch, i32(new), sum(new))
        x = torch.randn(sum(new), 8, device="cuda")
        latents[slots] = x
        for i in (0, 1):
            kept[i].append(x[sum(new[:i]):sum(new[:i + 1])])
        for i in (0, 1):
            p = torch.arange(int(batch.lengths[i]), device="cuda")
            at = batch.table[i][p // 32].long() * 32 + p % 32
            assert torch.equal(latents[at], torch.cat(kept[i]))


def test_refused_rows_take_no_memory():
    from parrot import PagedBatch, PagePool
    pool = PagePool(9, 32)
    batch = PagedBatch.from_lists([[0], [1]], [5, 6], [1, 1])
    new = i32([1, 1])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for rows in ((1 << 30) + 1, 1 << 32, (1 << 32) + 2):
        with pytest.raises(RuntimeError, match="rows"):
            pool.extend(batch, new, rows)
    assert torch.cuda.max_memory_allocated() == before
    assert batch.lengths.tolist() == [5, 6] and batch.starts.tolist() == [0, 1, 2]


@pytest.mark.parametrize("one_call", [True, False])
def test_refused_rows_beside_a_window(one_call):
    """Drafts that are turned down after the window has left pages, at lengths around the
    edges where it does: with the positions taken back before their window is released, or
    in the same call, each captured step is the same calls on pages that all stay."""
    from parrot import PagedBatch, PagedKVCache, PagePool
    b, heads, kv_heads, d, page, width, rows = 4, 8, 2, 96, 32, 16, 28
    window, sinks = 70, 33
    g = torch.Generator().manual_seed(16)
    rng = random.Random(16)
    pool, cache = PagePool(40, page), PagedKVCache(40, page, kv_heads, d)
    whole = PagedKVCache(b * width, page, kv_heads, d)
    tables = [list(range(i * width, (i + 1) * width)) for i in range(b)]
    batch = PagedBatch(i32([[-1] * width] * b), i32([0] * b), i32([0] * (b + 1)))
    k, v, q = (torch.zeros(rows, h, d, dtype=torch.bfloat16, device="cuda")
               for h in (kv_heads, kv_heads, heads))
    new, kept = i32([0] * b), i32([0] * b)

    def step():
        pool.extend(batch, new, rows)
        cache.append(k, v, batch)
        y = cache.attend(q, batch, scale=0.1, window=window, sinks=sinks)
        if one_call:
            pool.release(batch, kept, window=window, sinks=sinks)
        else:
            pool.release(batch, kept)
            pool.release(batch, window=window, sinks=sinks)
        return y
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lengths, plain = [0] * b, PlainPool([0] * 40, page, [[-1] * width] * b, [0] * b)
    left = crossed = 0
    while min(lengths) < width * page - 7:
        # drafts of up to 7 tokens, of which some stay; the last sequence never waits
        news = [min(n, width * page - length) for n, length in
                zip([1, 7, rng.randint(1, 7), 6], lengths)]
        keeps = [length + n - rng.randint(0, max(n - 1, 0)) for n, length in zip(news, lengths)]
        keeps[3] = lengths[3] + news[3] - (0 if rng.random() < 0.3 else max(news[3] - 1, 0))
        grown = [n + length for n, length in zip(news, lengths)]
        for n, to in zip(grown, keeps):  # pages that all of the rows would leave, the kept ones not
            crossed += (n - window + 1) // page > max(to - window + 1, 0) // page >= 2
        fresh = [torch.randn(rows, h, d, generator=g).bfloat16() for h in (kv_heads, kv_heads, heads)]
        for x, y in zip((k, v, q, new, kept), (*fresh, i32(news), i32(keeps))):
            x.copy_(y)
        graph.replay()
        byhand = PagedBatch.from_lists(tables, grown, news)
        whole.append(k, v, byhand)
        want = whole.attend(q, byhand, scale=0.1, window=window, sinks=sinks)
        total = sum(news)
        assert torch.equal(out[:total], want[:total]), lengths
        plain.extend(news, rows)
        plain.release(keeps, window=window, sinks=sinks)
        assert batch.lengths.tolist() == plain.lengths == keeps
        assert batch.table.tolist() == plain.table and pool.uses.tolist() == plain.uses
        lengths = keeps
        left += sum(row[2] == -1 for row in plain.table)
    assert left > 0 and crossed > 10


def test_a_step_and_back():
    """extend, then release to the lengths before: the table and the lengths are as they
    were, and so are the uses (of pages that a use below 0 made free, 0 is left)."""
    rng = random.Random(5)
    for negative in (False, True):
        both = Both.filled(rng, 300, 40, 32, 9000, 600)
        if not negative:
            both.pool.uses.clamp_(min=0)
        assert (both.pool.uses < 0).any() == negative
        new = i32([rng.randint(0, 500) for _ in range(300)])
        state = (both.batch.table, both.batch.lengths, both.pool.uses)
        before = [x.clone() for x in state]
        for _ in range(3):
            both.pool.extend(both.batch, new, 80000)
            assert not torch.equal(state[0], before[0]) and not torch.equal(state[1], before[1])
            both.pool.release(both.batch, before[1])
            assert torch.equal(state[0], before[0]) and torch.equal(state[1], before[1])
            assert torch.equal(state[2].clamp_min(0), before[2].clamp_min(0))
            assert negative or torch.equal(state[2], before[2])


def test_pools_and_caches_of_other_sizes():
    """Pages that a cache does not have, or of another size: refused by its calls, where
    rows would be dropped or go astray; taken once a fitting pool has the batch."""
    from parrot import PagedBatch, PagedKVCache, PagePool
    cache = PagedKVCache(6, 64, 2, 96)
    rows = torch.randn(3, 12, 96, device="cuda").bfloat16()
    k, v, q = rows[:, :2], rows[:, 2:4], rows[:, 4:]
    table = torch.ones(64, 48, device="cuda")
    for pool in (PagePool(7, 64), PagePool(6, 32), PagePool(6, 128)):
        batch = PagedBatch(i32([[-1, -1]]), i32([0]), i32([0, 0]))
        pool.extend(batch, i32([3]), 3)
        before = [x.clone() for x in cache._tensors[:2]]
        for call in (lambda: cache.append(k, v, batch), lambda: cache.read(batch, 3),
                     lambda: cache.append_rope(q, k, v, batch, table, table),
                     lambda: cache.attend(q, batch, scale=0.1)):
            with pytest.raises(RuntimeError, match="pool"):
                call()
        assert all(torch.equal(x, y) for x, y in zip(before, cache._tensors))
        pool.release(batch, i32([0]))
        PagePool(5, 64).extend(batch, i32([3]), 3)
        cache.append(k, v, batch)
        assert torch.equal(cache.read(batch, 3)[0][0], k.transpose(0, 1))
        cache.attend(q, batch, scale=0.1)
