"""GPU checks of paged attention over pages that were not written by append: rows whose byte
says that they are not finite (255) are NaN, whatever values stand under it."""
import math

import pytest
import torch

from paged_cases import Plain

pytestmark = pytest.mark.gpu

TYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8, "e2m1": torch.float4_e2m1fn_x2}
# bytes that make values of about 1
USUAL = {"e4m3": 119, "int8": 121, "e2m1": 125}


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def _cache(g, name, pages, page, kv_heads, d):
    """Pages of any values but zeros and NaN."""
    from parrot import PagedKVCache
    cache = PagedKVCache(pages, page, kv_heads, d, TYPES[name])
    for x in (cache.key, cache.value):
        x = x.view(torch.uint8)
        if name == "e2m1":
            code = torch.randint(0, 2, (2, *x.shape), generator=g) * 8 + \
                torch.randint(1, 8, (2, *x.shape), generator=g)
            x.copy_(code[0] + 16 * code[1])
        else:
            x.copy_(torch.randint(1, 127, x.shape, generator=g) +
                    128 * torch.randint(0, 2, x.shape, generator=g))
    for x in (cache.key_exponent, cache.value_exponent):
        x.copy_(USUAL[name] - torch.randint(0, 3, x.shape, generator=g))
    return cache


# tiles of 4, 8, 16, 32 and 128 rows; blocks that rows see whole and in part
@pytest.mark.parametrize("d", [64, 96])
@pytest.mark.parametrize("n,length,copies", [(1, 150, 1), (1, 1000, 1), (2, 150, 1), (2, 1000, 20),
                                             (6, 150, 1), (40, 300, 1), (73, 150, 128)])
@pytest.mark.parametrize("name", TYPES)
def test_rows_that_are_not_finite(name, n, length, copies, d):
    from parrot import PagedBatch, PagedKVCache
    g = torch.Generator().manual_seed(n + length)
    page = 64
    pages = (length + page - 1) // page
    table = torch.arange(pages, dtype=torch.int32).repeat(copies, 1).cuda()
    batch = PagedBatch(table, torch.full((copies,), length, dtype=torch.int32, device="cuda"),
                       torch.arange(0, n * copies + 1, n, dtype=torch.int32, device="cuda"))
    q = (torch.randn(n, 8, d, generator=g) * 1.5).bfloat16()
    for bad in (40, length - n // 2 - 1):
        cache = _cache(g, name, pages, page, 2, d)
        one = PagedBatch(table[:1], batch.lengths[:1], batch.starts[:2])
        k, v = (x[0].transpose(0, 1).double().cpu() for x in cache.read(one, length))
        assert torch.isfinite(k).all() and torch.isfinite(v).all()
        # a key of the first kv head, a value of the second
        at, p = bad // page, bad % page
        if name == "e2m1":
            byte = cache.key_exponent[at, 0, p // 32].view(16, 2, d // 32)
            byte[p % 16, p % 32 // 16, 1] = 255
        else:
            cache.key_exponent[at, 0, p] = 255
        cache.value_exponent[at, 1, p] = 255
        key, value = (x[0].cpu() for x in cache.read(one, length))
        dims = 32 if name == "e2m1" else d
        assert key[0, bad].isnan().sum() == key.isnan().sum() == dims
        assert value[1, bad].isnan().all() and value.isnan().sum() == d
        plain = Plain(torch.bfloat16, 2, d, 1)
        k[bad, 0] = v[bad, 1] = 0.0
        for window, sinks in ((None, 0), (100, 0), (100, 41)):
            print(f"{name}: {copies} x {n} after {length}, {bad}, window {window}", flush=True)
            got = cache.attend(q.cuda().repeat(copies, 1, 1), batch, scale=d ** -0.5, window=window,
                               sinks=sinks).view(copies, n, 2, -1)
            assert torch.equal(got.view(torch.int16), got[:1].view(torch.int16).expand_as(got))
            got = got[0].double().cpu()
            pos = torch.arange(length - n, length)
            sees = (pos >= bad) & ((bad > pos - (window or math.inf)) | (bad < sinks))
            assert got[sees].isnan().all()
            for head in (0, 1):  # the other kv head's row is gone for both
                plain.k, plain.v = [k], [v]
                ref, bound = plain.attend(q, [n], d ** -0.5, window, sinks)
                off = (got[:, head] - ref.view(n, 2, -1)[:, head]).abs()
                assert (off <= bound.view(n, 2, -1)[:, head])[~sees].all()
