"""Argument checks of the page pool (no GPU)."""
import copy
import ctypes
import pickle

import pytest
import torch

FAKE = 0x10000  # 16-byte aligned, never dereferenced here


def test_arguments():
    from parrot import _abi
    lib, ref = _abi.load(), ctypes.byref

    def pool(**kw):
        return _abi.PagedPoolStruct(**{**dict(uses=FAKE, pages=100, page=64), **kw})

    def batch(**kw):
        fields = dict(table=FAKE, lengths=FAKE, starts=FAKE, batch=3, width=8)
        return _abi.PagedBatchStruct(**{**fields, **kw})

    def extend(p, b, new=None, rows=5, slots=FAKE, positions=FAKE, ws=None, wsb=0):
        return lib.parrot_paged_extend(ref(p), ref(b), new, rows, slots, positions, ws, wsb, None)

    def release(p, b, window=0, sinks=-1):
        return lib.parrot_paged_release(ref(p), ref(b), FAKE, window, sinks, None)
    for p, b, status in [(dict(uses=None), {}, -1), ({}, dict(table=None), -1),
                         ({}, dict(lengths=None), -1), ({}, dict(starts=None), -1),
                         (dict(pages=-1), {}, -2), (dict(pages=(1 << 30) + 1), {}, -2),
                         (dict(page=0), {}, -2), (dict(page=48), {}, -3), ({}, dict(batch=-1), -2),
                         ({}, dict(width=-1), -2), ({}, dict(width=1 << 26), -2),
                         ({}, dict(batch=70000), -3), (dict(uses=FAKE + 8), {}, -5)]:
        for call in (extend, release):
            assert call(pool(**p), batch(**b)) == status, (p, b, call.__name__)
    assert lib.parrot_paged_extend(None, ref(batch()), FAKE, 5, FAKE, FAKE, None, 0, None) == -1
    assert lib.parrot_paged_release(ref(pool()), None, FAKE, 0, 0, None) == -1
    assert extend(pool(), batch()) == -1  # no new rows
    assert extend(pool(), batch(), FAKE, slots=None) == -1
    assert extend(pool(), batch(), FAKE, positions=None) == -1
    assert extend(pool(), batch(), FAKE, rows=-1) == -2
    assert extend(pool(), batch(), FAKE, rows=(1 << 30) + 1) == -2
    assert release(pool(), batch()) == -2  # sinks below 0
    assert extend(pool(), batch(), FAKE, slots=FAKE + 8) == -5
    assert extend(pool(), batch(), FAKE, positions=FAKE + 4) == -5
    size = lib.parrot_paged_extend_workspace_bytes
    assert size(100, 0, 0) == 0 and size(100, -1, 5) == 0 and size(100, 70000, 5) == 0
    assert size(-1, 5, 50000) == 0 and size(100, 5, -1) == 0 and size(100, 5, 50000) > 0
    many, need = batch(batch=60000), size(100, 60000, 5)
    assert need > 0
    assert extend(pool(), many, FAKE, ws=None, wsb=need) == -4
    assert extend(pool(), many, FAKE, ws=FAKE, wsb=need - 1) == -4
    assert extend(pool(), many, FAKE, ws=FAKE + 8, wsb=need) == -5


def test_pool_checks():
    from parrot import PagedBatch, PagePool
    with pytest.raises(RuntimeError):
        PagePool(-1, 64, device="cpu")
    for page in (0, 48, -32):
        with pytest.raises(RuntimeError):
            PagePool(4, page, device="cpu")
    for bad in (torch.zeros(4), torch.zeros(4, 2, dtype=torch.int32),
                torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(8, dtype=torch.int32)[1:],
                torch.zeros(4, dtype=torch.int64)):
        with pytest.raises(RuntimeError):
            PagePool.from_uses(bad, 64)
    uses = torch.zeros(4, dtype=torch.int32)
    p = PagePool.from_uses(uses, 64)
    assert p.uses is uses and p.page_size == 64 and PagePool(3, 32, device="cpu").uses.tolist() == [0] * 3
    for q in (copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert torch.equal(q.uses, uses) and q.uses.data_ptr() != uses.data_ptr()
        assert q._struct.uses == q.uses.data_ptr() and q._struct.pages == 4 and q.page_size == 64
    b = PagedBatch.from_lists([[0], [1]], [5, 6], [1, 1], device="cpu")
    with pytest.raises(RuntimeError):  # not on a GPU
        p.extend(b, torch.ones(2, dtype=torch.int32), 2)
    with pytest.raises(RuntimeError):
        p.release(b)


def test_the_plain_form():
    """The plain form that the GPU tests compare with, at a few steps by hand."""
    from pool_cases import PlainPool
    p = PlainPool([0, 1, 0, 0, -1, 0], 32, [[1, -1, -1], [-1, -1, -1], [-1, -1, -1]], [31, 0, 0])
    assert p.extend([2, 33, 1], 40) == ([1 * 32 + 31, 0 * 32] + [2 * 32 + i for i in range(32)] + [96, 128]
                                        + [-1] * 4, [31, 32, *range(33), 0] + [-1] * 4)
    assert p.starts == [0, 2, 35, 36] and p.lengths == [33, 33, 1]
    assert p.table == [[1, 0, -1], [2, 3, -1], [4, -1, -1]] and p.uses == [1, 1, 1, 1, 1, 0]
    # the first has room on its pages, the second takes the last one, the third gets none
    assert p.extend([31, 63, 32], 200)[1][:95] == [*range(33, 64), *range(33, 96), -1]
    assert p.starts == [0, 31, 94, 94] and p.uses == [1] * 6
    # a table without room asks for nothing; what needs no page is not refused
    assert p.extend([33, 1, 31], 200)[1][:32] == [*range(1, 32), -1]
    p.release([64, 32, 0])
    assert p.table == [[1, 0, -1], [2, -1, -1], [-1, -1, -1]] and p.uses == [1, 1, 1, 0, 0, 0]
    p.release(window=33)
    assert p.table[0] == [-1, 0, -1] and p.uses == [1, 0, 1, 0, 0, 0] and p.lengths == [64, 32, 0]


def test_rows_of_a_step_are_bounded():
    """Numbers of rows that the library has no 32 bits for are refused before anything is
    allocated for them (the check comes before that for a GPU)."""
    from parrot import PagedBatch, PagePool
    p = PagePool(4, 64, device="cpu")
    b = PagedBatch.from_lists([[0]], [5], [1], device="cpu")
    for rows in (-1, 2 ** 30 + 1, 2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 64 + 1):
        with pytest.raises(RuntimeError, match="rows"):
            p.extend(b, torch.ones(1, dtype=torch.int32), rows)


def test_caches_know_their_pool():
    """A cache takes a batch that nobody or a fitting pool handed pages to, and no other; copies
    of a batch are nobody's."""
    from parrot import PagedBatch, PagedKVCache, PagePool
    cache = PagedKVCache(9, 64, 2, 96, device="cpu")
    b = PagedBatch.from_lists([[0]], [5], [1], device="cpu")
    assert cache._batch(b) == b._at
    for pages, page, fits in ((9, 64, True), (10, 64, False), (9, 32, False), (4, 128, False),
                              (3, 64, True)):
        object.__setattr__(b, "_pool", PagePool(pages, page, device="cpu"))
        if fits:
            assert cache._batch(b) == b._at
        else:
            with pytest.raises(RuntimeError, match=f"{pages} pages of {page}"):
                cache._batch(b)
            assert cache._batch(copy.copy(b))
