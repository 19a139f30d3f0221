"""Checks of the paged KV cache in 4 bits that need no GPU: its arguments, its tensors,
and the plain form that the GPU tests compare with."""
import copy
import ctypes
import io
import pickle

import pytest
import torch

from test_paged_cpu import BAD, FAKE, _batch, _cache

E2M1 = torch.float4_e2m1fn_x2


def test_arguments():
    from parrot import _abi
    lib, ref = _abi.load(), ctypes.byref

    def append(c, b):
        return lib.parrot_paged_append_bf16(ref(c), ref(b), None, 192, 96, FAKE, 192, 96, 4, None)

    def read(c, b):
        return lib.parrot_paged_read_bf16(ref(c), ref(b), 9, None, 19200, 9600, 96, FAKE, 19200, 9600,
                                          96, None)

    def attend(c, b):
        return lib.parrot_paged_attention_bf16(ref(c), ref(b), None, 192, 96, 4, 8, 0, 0, 0.1, FAKE,
                                               FAKE, 1 << 40, None)
    for call in (append, read, attend):
        assert call(_cache(type=4), _batch()) == -1  # (no rows)
        for c, b, status in BAD:
            if "type" not in c:
                assert call(_cache(**{"type": 4, **c}), _batch(**b)) == status, (c, b)
        for name in ("key_exponent", "value_exponent"):
            assert call(_cache(**{"type": 4, name: FAKE + 4}), _batch()) == -5
            assert call(_cache(**{"type": 4, name: None}), _batch()) == -1
        assert call(_cache(type=5), _batch()) == -3
    for scale, status in ((2.0 ** 126, -2), (2.0 ** 125, -1), (0.0, -2)):
        c, b = _cache(type=4), _batch()
        assert lib.parrot_paged_attention_bf16(ref(c), ref(b), None, 192, 96, 4, 8, 0, 0, scale,
                                               FAKE, FAKE, 1 << 40, None) == status


@pytest.mark.parametrize("d", [64, 96, 128])
def test_cache_checks(d):
    from parrot import PagedKVCache
    c = PagedKVCache(4, 96, 3, d, E2M1, device="cpu")
    assert (c.page_size, c.kv_heads, c.head_dim, c.dtype) == (96, 3, d, E2M1)
    assert c.key.shape == c.value.shape == (4, 3, 3, 16 * d)
    assert c.key_exponent.shape == (4, 3, 3, d) and c.value_exponent.shape == (4, 3, 96)
    assert c._struct.type == 4 and c._struct.head_dim == d
    again = PagedKVCache.from_pages(c.key, c.value, c.key_exponent, c.value_exponent)
    assert again.key is c.key and again.head_dim == d
    rows = c.value_exponent
    for bad in ((c.key, c.value), (c.key, c.value, rows, rows),
                (c.key, c.value, c.key_exponent, c.key_exponent),
                (c.key, c.value[:3], c.key_exponent, rows),
                (c.key, c.value.view(torch.uint8), c.key_exponent, rows),
                (c.key[..., :8 * d], c.value[..., :8 * d], c.key_exponent, rows),
                (c.key, c.value, c.key_exponent.transpose(2, 3), rows),
                (c.key, c.value, c.key_exponent.float(), rows)):
        with pytest.raises(RuntimeError):
            PagedKVCache.from_pages(*bad)
    with pytest.raises(RuntimeError):
        PagedKVCache(4, 64, 2, 80, E2M1, device="cpu")
    c.key.view(torch.uint8).random_(0, 256)
    d = copy.deepcopy(c)
    for x, y in zip(c._tensors, d._tensors):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and x.data_ptr() != y.data_ptr()
    assert d._struct.key == d.key.data_ptr() and d._struct.key_exponent == d.key_exponent.data_ptr()


def test_stored_forms():
    """Powers that leave the largest magnitude above 3.5 and not above 7; every value the
    nearest of the eight magnitudes, of two as near the one whose last bit is 0."""
    from paged4_cases import stored
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(300, 96, generator=g) * torch.exp2(torch.randint(-20, 20, (300, 1),
                                                                       generator=g))).bfloat16()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    for group in (32, 96):
        y = stored(x, group)
        assert torch.equal(y.bfloat16().double(), y)  # exact in bf16
        z = x.double().unflatten(-1, (-1, group))
        amax = z.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(amax / 7)))
        assert (amax / step <= 7).all() and (amax / step > 3.5).all()
        q = (z / step).abs()
        off = (q[..., None] - grid).abs()
        best = off.argmin(-1)  # the lower of two
        tie = (off.gather(-1, best[..., None]) == off.gather(
            -1, (best + 1).clamp_max(7)[..., None]))[..., 0] & (best < 7) & (best % 2 == 1)
        want = grid[best + tie] * step * z.sign()
        assert torch.equal(want.flatten(-2), y)
        # what the documentation says of normal rows: their error is 11 % of the norm
        assert 0.108 < ((y - x.double()).norm(dim=-1) / x.double().norm(dim=-1)).mean() < 0.117


def test_pickles():
    """Caches of 4 bits are pickled and saved as those of the other types are; a copy is over
    the same memory."""
    from parrot import PagedKVCache
    c = PagedKVCache(4, 64, 2, 96, E2M1, device="cpu")
    for x in c._tensors:
        x.view(torch.uint8).random_(0, 256)
    saved = io.BytesIO()
    torch.save(c, saved)
    saved.seek(0)
    for d in (pickle.loads(pickle.dumps(c)), torch.load(saved, weights_only=False)):
        assert d.dtype == E2M1 and (d.page_size, d.kv_heads, d.head_dim) == (64, 2, 96)
        for x, y in zip(c._tensors, d._tensors):
            assert x.dtype == y.dtype and x.data_ptr() != y.data_ptr()
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        assert d._struct.key == d.key.data_ptr() and d._struct.type == 4
    for x, y in zip(c._tensors, copy.copy(c)._tensors):
        assert x.data_ptr() == y.data_ptr()
