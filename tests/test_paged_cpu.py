"""Argument checks of the paged KV cache, of attention over it and of sampling
(no GPU)."""
import ctypes

import pytest
import torch

FAKE = 0x10000  # 16-byte aligned, never dereferenced here


def _cache(**kw):
    from parrot import _abi
    fields = dict(key=FAKE, value=FAKE, key_exponent=FAKE, value_exponent=FAKE, pages=10, page=64,
                  kv_heads=2, head_dim=96, type=1)
    return _abi.PagedCacheStruct(**{**fields, **kw})


def _batch(**kw):
    from parrot import _abi
    fields = dict(table=FAKE, lengths=FAKE, starts=FAKE, batch=3, width=8)
    return _abi.PagedBatchStruct(**{**fields, **kw})


BAD = [(dict(key=None), {}, -1), (dict(value_exponent=None), {}, -1), ({}, dict(table=None), -1),
       ({}, dict(lengths=None), -1), ({}, dict(starts=None), -1), (dict(page=0), {}, -2),
       (dict(pages=-1), {}, -2), (dict(pages=1 << 30), {}, -2), (dict(pages=1 << 62), {}, -2),
       (dict(kv_heads=0), {}, -2), ({}, dict(batch=-1), -2),
       ({}, dict(width=-1), -2), ({}, dict(width=1 << 26), -2), (dict(page=48), {}, -3),
       (dict(head_dim=80), {}, -3), (dict(type=3), {}, -3), (dict(type=-1), {}, -3),
       ({}, dict(batch=70000), -3), (dict(key=FAKE + 8), {}, -5), (dict(key_exponent=FAKE + 2), {}, -5)]


def test_paged_arguments():
    from parrot import _abi
    lib, ref = _abi.load(), ctypes.byref
    two, three = (192, 96), (19200, 9600, 96)

    def append(c, b, k=FAKE, ks=two, v=FAKE, vs=two, rows=4):
        return lib.parrot_paged_append_bf16(ref(c), ref(b), k, *ks, v, *vs, rows, None)

    def read(c, b, positions=100, k=FAKE, ks=three, v=FAKE, vs=three):
        return lib.parrot_paged_read_bf16(ref(c), ref(b), positions, k, *ks, v, *vs, None)

    def attend(c, b, q=FAKE, qs=two, rows=4, heads=8, window=0, sinks=0, scale=0.1, out=FAKE,
               ws=FAKE, wsb=1 << 40):
        return lib.parrot_paged_attention_bf16(ref(c), ref(b), q, *qs, rows, heads, window, sinks,
                                               scale, out, ws, wsb, None)
    for c, b, status in BAD:
        for call in (append, read, attend):
            assert call(_cache(**c), _batch(**b)) == status, (c, b, call.__name__)
    assert lib.parrot_paged_append_bf16(None, ref(_batch()), FAKE, *two, FAKE, *two, 4, None) == -1
    assert lib.parrot_paged_read_bf16(ref(_cache()), None, 9, FAKE, *three, FAKE, *three, None) == -1
    c, b = _cache(), _batch()
    odd2, odd3 = (192, 98), (19200, 9600, 97)
    assert append(c, b, k=None) == -1 and append(c, b, v=None) == -1
    assert append(c, b, rows=-1) == -2 and append(c, b, rows=0) == 0
    assert append(c, b, ks=odd2) == -5 and append(c, b, v=FAKE + 4) == -5
    assert read(c, b, v=None) == -1 and read(c, b, positions=-1) == -2
    assert read(c, b, positions=0) == 0 and read(c, _batch(batch=0)) == 0
    assert read(c, b, ks=odd3) == -5 and read(c, b, k=FAKE + 2) == -5
    assert attend(c, b, q=None) == -1 and attend(c, b, out=None) == -1
    assert attend(c, b, heads=7) == -2 and attend(c, b, heads=0) == -2
    assert attend(c, b, rows=-1) == -2 and attend(c, b, rows=1 << 28) == -2
    assert attend(c, b, sinks=-1) == -2
    for scale in (0.0, float("nan"), float("inf")):
        assert attend(c, b, scale=scale) == -2
    assert attend(c, b, rows=0) == 0 and attend(c, _batch(batch=0)) == 0
    assert attend(c, b, qs=(196, 96)) == -5
    assert attend(c, b, q=FAKE + 8) == -5 and attend(c, b, out=FAKE + 4) == -5
    size = lib.parrot_paged_attention_workspace_bytes
    need = size(ref(c), ref(_batch(width=60)), 4, 8, 0, 0)
    assert need > 0
    wide = _batch(width=60)
    assert attend(c, wide, wsb=need - 1) == -4 and attend(c, wide, ws=None) == -4
    assert attend(c, wide, ws=FAKE + 8) == -5
    assert size(ref(c), ref(b), 4, 7, 0, 0) == 0 and size(ref(_cache(page=33)), ref(b), 4, 8, 0, 0) == 0


def test_sample_arguments():
    from parrot import _abi
    lib = _abi.load()

    def sample(x=FAKE, type=0, rows=2, vocab=100, stride=100, u=FAKE, token=FAKE):
        return lib.parrot_sample(x, type, rows, vocab, stride, u, None, 1.0, None, 0, None, 1.0,
                                 None, 0.0, token, None, None)
    assert sample(x=None) == -1 and sample(u=None) == -1 and sample(token=None) == -1
    assert sample(rows=-1) == -2 and sample(vocab=0) == -2 and sample(stride=99) == -2
    assert sample(vocab=(1 << 20) + 1, stride=1 << 21) == -3 and sample(type=3) == -3
    assert sample(x=FAKE + 2) == -5 and sample(x=FAKE + 1, type=1) == -5
    assert sample(rows=0, x=None) == 0


def test_cache_checks():
    from parrot import PagedBatch, PagedKVCache
    for bad in ((4, 48, 2, 96), (4, 0, 2, 96), (-1, 64, 2, 96), (4, 64, 0, 96), (4, 64, 2, 80)):
        with pytest.raises(RuntimeError):
            PagedKVCache(*bad, device="cpu")
    with pytest.raises(RuntimeError):
        PagedKVCache(4, 64, 2, 96, torch.float16, device="cpu")
    c = PagedKVCache(4, 64, 2, 96, torch.int8, device="cpu")
    assert (c.page_size, c.kv_heads, c.head_dim) == (64, 2, 96)
    PagedKVCache.from_pages(c.key, c.value, c.key_exponent, c.value_exponent)
    for bad in ((c.key, c.value), (c.key, c.value[:3], c.key_exponent, c.value_exponent),
                (c.key, c.value, c.key_exponent, c.value_exponent[..., :32]),
                (c.key.transpose(0, 1), c.value.transpose(0, 1), c.key_exponent, c.value_exponent),
                (c.key[0], c.value[0], c.key_exponent, c.value_exponent),
                (c.key, c.value.view(torch.float8_e4m3fn), c.key_exponent, c.value_exponent)):
        with pytest.raises(RuntimeError):
            PagedKVCache.from_pages(*bad)
    for bad in (([[0]], [3], [1, 1]), ([[0]], [3], [4]), ([[0]], [3], [-1])):
        with pytest.raises(ValueError):
            PagedBatch.from_lists(*bad, device="cpu")
    i32 = dict(dtype=torch.int32)
    for bad in ((torch.zeros(2, 3, **i32), torch.zeros(3, **i32), torch.zeros(3, **i32)),
                (torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(2, **i32)),
                (torch.zeros(2, 3), torch.zeros(2, **i32), torch.zeros(3, **i32)),
                (torch.zeros(3, 2, **i32).t(), torch.zeros(2, **i32), torch.zeros(3, **i32))):
        with pytest.raises(RuntimeError):
            PagedBatch(*bad)
    b = PagedBatch.from_lists([[0, 2], [1]], [70, 3], [1, 2], device="cpu")
    assert b.table.tolist() == [[0, 2], [1, -1]] and b.starts.tolist() == [0, 1, 3]
    q = torch.zeros(3, 8, 96, dtype=torch.bfloat16)
    with torch.no_grad():
        with pytest.raises(RuntimeError):  # not on a GPU
            c.attend(q, b, scale=0.1)
        with pytest.raises(RuntimeError):
            c.append(q[:, :2], q[:, :2], b)


def test_stored_forms():
    """The plain form that the GPU tests compare with: e4m3 by torch's own
    conversion, powers of two that bring a row inside the type's range."""
    from paged_cases import LARGEST, stored
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(200, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (200, 1),
                                                                       generator=g))).bfloat16()
    for dtype in LARGEST:
        y = stored(x, dtype)
        assert torch.equal(y.bfloat16().double(), y)  # exact in bf16
        amax = x.double().abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(amax / LARGEST[dtype])))
        assert (amax / step <= LARGEST[dtype]).all() and (amax / step > LARGEST[dtype] / 2).all()
        q = (x.double() / step).float()
        q = q.to(dtype) if dtype == torch.float8_e4m3fn else q.round()
        assert torch.equal(q.double() * step, y)


def test_scales_that_attention_refuses():
    """A scale whose product with log2(e), and 4 for int8 pages, is no fp32 number."""
    from parrot import _abi
    lib, ref, c, b = _abi.load(), ctypes.byref, _cache(), _batch()
    for scale, status in ((2.0 ** 126, -2), (-3e38, -2), (float("-inf"), -2), (2.0 ** 125, -1),
                          (-(2.0 ** 125), -1), (1e-30, -1)):  # (-1: no query rows)
        for type in range(3):
            c.type = type
            assert lib.parrot_paged_attention_bf16(ref(c), ref(b), None, 192, 96, 4, 8, 0, 0, scale,
                                                   FAKE, FAKE, 1 << 40, None) == status, scale


def test_copies_and_pickles():
    """Of a cache and a batch: tensors of their own, whose addresses the calls get."""
    import copy
    import pickle
    from parrot import PagedBatch, PagedKVCache
    for dtype in (torch.bfloat16, torch.float8_e4m3fn, torch.int8):
        c = PagedKVCache(3, 64, 2, 64, dtype, device="cpu")
        c.key.view(torch.uint8).random_(0, 100)
        copies = [copy.deepcopy(c), copy.deepcopy({"cache": c})["cache"]]
        if dtype != torch.float8_e4m3fn:  # (torch itself does not unpickle such a tensor)
            copies.append(pickle.loads(pickle.dumps(c)))
        for d in copies:
            assert (d.page_size, d.kv_heads, d.head_dim, d.dtype) == (64, 2, 64, dtype)
            for x, y, at in zip(c._tensors, d._tensors, ("key", "value", "key_exponent",
                                                         "value_exponent")):
                if x is None:
                    assert y is None
                    continue
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
                assert getattr(d._struct, at) == y.data_ptr() != x.data_ptr()
            assert d._at == ctypes.addressof(d._struct) and d._struct.type == c._struct.type
        assert copy.copy(c).key is c.key
    b = PagedBatch.from_lists([[0, 2], [1]], [70, 3], [1, 2], device="cpu")
    for d in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert torch.equal(b.table, d.table) and torch.equal(b.lengths, d.lengths)
        assert d._struct.table == d.table.data_ptr() != b.table.data_ptr()
        assert d._at == ctypes.addressof(d._struct)
