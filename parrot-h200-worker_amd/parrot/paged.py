"""A paged KV cache of the MI355X backend, and attention over it.

``PagedKVCache`` holds one layer's keys and values for many sequences in pages,
in bf16 or in 8 bits (quantised as they are written); ``PagedBatch`` says which
pages, lengths and new rows belong to which sequence of a call.  A step of a
layer appends the new rows and attends from them::

    cache.append(k, v, batch)
    y = cache.attend(q, batch, scale=head_dim ** -0.5, window=2048, sinks=4)

New beside the contiguous caches of ``Parrot.prefill`` / ``decode_step``
(parrot/model.py:239-295), whose sequences all have one length.  As in
``parrot.hip_moe``, every call runs on PyTorch's current HIP stream, allocates
with torch, never synchronises with the host (so it can be captured in a HIP
graph) and raises on inputs that it does not take.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch import Tensor

from . import _abi
from .hip_moe import ATTENTION_HEAD_DIMS, _on, _require, _stream

PAGE_TYPES = {torch.bfloat16: 0, torch.float8_e4m3fn: 1, torch.int8: 2}
PAGE_BLOCK = 32  # a page is a whole number of blocks of so many positions


@dataclass(frozen=True, eq=False)
class PagedBatch:
    """Which part of a call belongs to which sequence; int32 device tensors.

    ``table`` [b, width]: the pages of each sequence, position p in page
    ``table[i, p // page_size]``.  An id outside the cache holds nothing: keys that
    fall there are not seen, writes to it are dropped (so pages that a window has
    left for good may be given back).  ``lengths`` [b]: positions of each
    sequence, the new ones included.  ``starts`` [b + 1]: sequence i's new rows
    are rows ``starts[i]`` to ``starts[i + 1] - 1`` of the call's operands, its last
    positions.  A sequence may have no new row.  Rows past ``starts[b]`` (a padded
    batch) belong to nobody: they are neither read nor written.

    The tensors are read when a call runs, so a captured step follows what a
    program writes into them (and needs them for as long as it is replayed);
    the kernels bound every number they read."""
    table: Tensor
    lengths: Tensor
    starts: Tensor

    def __post_init__(self):
        for name in ("table", "lengths", "starts"):
            x = getattr(self, name)
            if x.dtype != torch.int32 or x.device != self.table.device or not x.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous int32 tensor, all three on one "
                                   "device")
        if self.table.ndim != 2 or self.lengths.shape != (self.table.shape[0],) or \
                self.starts.shape != (self.table.shape[0] + 1,):
            raise RuntimeError("a batch is table [b, width], lengths [b] and starts [b + 1]")
        b, width = self.table.shape
        object.__setattr__(self, "_struct", _abi.PagedBatchStruct(
            self.table.data_ptr(), self.lengths.data_ptr(), self.starts.data_ptr(), b, width))
        object.__setattr__(self, "_at", ctypes.addressof(self._struct))

    # (copies and pickles are of the tensors, not of their addresses)
    def __reduce__(self):
        return type(self), (self.table, self.lengths, self.starts)

    @classmethod
    def from_lists(cls, pages: list[list[int]], lengths: list[int], new: list[int],
                   device="cuda") -> "PagedBatch":
        """The batch of sequences with these pages, whole lengths and numbers of
        new rows; checks them."""
        if not len(pages) == len(lengths) == len(new):
            raise ValueError("one list of pages, one length and one number of new rows "
                             "per sequence")
        if any(n < 0 or n > length for n, length in zip(new, lengths)):
            raise ValueError("a sequence's new rows are part of its length")
        width = max((len(p) for p in pages), default=0)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        table = torch.tensor([list(p) + [-1] * (width - len(p)) for p in pages],
                             dtype=torch.int32).view(len(pages), width)
        return cls(table.to(device), torch.tensor(lengths, dtype=torch.int32).to(device),
                   torch.tensor(starts, dtype=torch.int32).to(device))


class PagedKVCache:
    """Pages of keys and values of one layer.

    ``key`` / ``value`` [pages, kv_heads, page_size / 32, 32 head_dim] of ``dtype``
    (bf16, float8_e4m3fn or int8) hold blocks of 32 positions in the order in
    which the attention kernels read them (include/parrot_hip.h); ``read`` gives
    rows.  8-bit rows are scaled by a power of two of their own, one byte per
    position and head in ``key_exponent`` / ``value_exponent`` [pages, kv_heads,
    page_size], so that a stored value is exact in bf16.  What that costs, for
    normally distributed rows of 96: 2.7 % of the row's norm in e4m3 (whatever
    the row holds: its error goes with the value), 0.9 % in int8.  A row with a
    NaN or an infinity reads back as NaN."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        self._check(pages, page_size, kv_heads, head_dim, dtype)
        # (8 bits as bytes that are viewed: no tensor beside those that are kept)
        byte = torch.uint8 if dtype.itemsize == 1 else dtype
        shape = (pages, kv_heads, page_size // PAGE_BLOCK, PAGE_BLOCK * head_dim)
        rows = [torch.zeros(shape, dtype=byte, device=device).view(dtype) for _ in range(2)]
        exponents = [None, None] if dtype == torch.bfloat16 else \
            [torch.zeros((pages, kv_heads, page_size), dtype=torch.uint8, device=device)
             for _ in range(2)]
        self._describe(*rows, *exponents)

    @classmethod
    def from_pages(cls, key: Tensor, value: Tensor, key_exponent: Tensor | None = None,
                   value_exponent: Tensor | None = None) -> "PagedKVCache":
        """A cache over tensors that are there already, laid out as above."""
        if key.ndim != 4 or key.shape[3] % PAGE_BLOCK:
            raise RuntimeError("pages are [pages, kv_heads, page_size / 32, 32 head_dim]")
        pages, kv_heads, blocks, width = key.shape
        cls._check(pages, blocks * PAGE_BLOCK, kv_heads, width // PAGE_BLOCK, key.dtype)
        exponents = () if key.dtype == torch.bfloat16 else (key_exponent, value_exponent)
        if value.shape != key.shape or value.dtype != key.dtype or \
                not (key.is_contiguous() and value.is_contiguous()):
            raise RuntimeError("key and value pages must be contiguous, of one shape and type")
        for x in exponents:
            if x is None or x.dtype != torch.uint8 or not x.is_contiguous() or \
                    x.shape != (pages, kv_heads, blocks * PAGE_BLOCK):
                raise RuntimeError("8-bit pages need contiguous uint8 exponents "
                                   "[pages, kv_heads, page_size]")
        if any(x.device != key.device for x in (value, *exponents)):
            raise RuntimeError("a cache's tensors must be on one device")
        self = cls.__new__(cls)
        self._describe(key, value, *(exponents or (None, None)))
        return self

    # (as PagedBatch)
    def __reduce__(self):
        return type(self).from_pages, self._tensors

    @staticmethod
    def _check(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype) -> None:
        if dtype not in PAGE_TYPES:
            raise RuntimeError(f"pages hold {', '.join(map(str, PAGE_TYPES))}, got {dtype}")
        if head_dim not in ATTENTION_HEAD_DIMS:
            raise RuntimeError(f"HIP attention supports head widths {ATTENTION_HEAD_DIMS}")
        if pages < 0 or kv_heads < 1 or page_size < 1 or page_size % PAGE_BLOCK:
            raise RuntimeError(f"a page is a multiple of {PAGE_BLOCK} positions of one or more "
                               "kv heads")

    def _describe(self, *tensors: Tensor | None) -> None:
        self._tensors = tensors
        pages, kv_heads, blocks, width = self.key.shape
        self.page_size, self.kv_heads = blocks * PAGE_BLOCK, kv_heads
        self.head_dim, self.dtype, self.device = width // PAGE_BLOCK, self.key.dtype, self.key.device
        self._struct = _abi.PagedCacheStruct(
            self.key.data_ptr(), self.value.data_ptr(), _abi.ptr(self.key_exponent),
            _abi.ptr(self.value_exponent), pages, self.page_size, kv_heads, self.head_dim,
            PAGE_TYPES[self.dtype])
        self._at = ctypes.addressof(self._struct)
        self._sizes: dict[tuple, int] = {}

    # The calls hand the tensors' addresses over, so they stay what they were made with.
    key = property(lambda self: self._tensors[0])
    value = property(lambda self: self._tensors[1])
    key_exponent = property(lambda self: self._tensors[2])
    value_exponent = property(lambda self: self._tensors[3])

    def _workspace_bytes(self, *sizes: int) -> int:
        """The attention's workspace for (batch, width, rows, heads, window, sinks)."""
        nbytes = self._sizes.get(sizes)
        if nbytes is None:
            if len(self._sizes) >= 256:
                self._sizes.clear()
            b = _abi.PagedBatchStruct(self._at, self._at, self._at, *sizes[:2])  # (not read)
            nbytes = self._sizes[sizes] = _abi.load().parrot_paged_attention_workspace_bytes(
                self._at, ctypes.addressof(b), *sizes[2:])
        return nbytes

    def _batch(self, batch: PagedBatch) -> int:
        if batch.table.device != self.device:
            raise RuntimeError("the batch must be on the cache's device")
        return batch._at

    def _new_rows(self, x: Tensor, heads: int, what: str, step: int) -> Tensor:
        _require(x, what)
        if x.ndim != 3 or x.shape[1] != heads or x.shape[2] != self.head_dim or \
                x.device != self.device:
            raise RuntimeError(f"{what} takes rows [rows, {heads}, {self.head_dim}] on the "
                               "cache's device")
        sr, sh, sd = x.stride()
        if sd != 1 or sr % step or sh % step or x.data_ptr() % (2 * step):
            x = x.clone(memory_format=torch.contiguous_format)
        return x

    def append(self, key: Tensor, value: Tensor, batch: PagedBatch) -> None:
        """Writes the new rows key and value [rows, kv_heads, head_dim] (bf16, any
        row and head strides) into their sequences' pages.  Other positions stay
        as they are.  A page that is written must belong to one sequence, once."""
        key = self._new_rows(key, self.kv_heads, "HIP paged append", 4)
        value = self._new_rows(value, self.kv_heads, "HIP paged append", 4)
        if key.shape != value.shape:
            raise RuntimeError("as many rows of values as of keys")
        b, (kr, kh, _), (vr, vh, _) = self._batch(batch), key.stride(), value.stride()
        with _on(self.device):
            _abi.check(_abi.load().parrot_paged_append_bf16(
                self._at, b, key.data_ptr(), kr, kh, value.data_ptr(), vr, vh, key.shape[0],
                _stream(self.device)), "parrot_paged_append_bf16")

    def append_rope(self, q: Tensor, key: Tensor, value: Tensor, batch: PagedBatch, cos: Tensor,
                    sin: Tensor) -> Tensor:
        """``append`` of keys that RoPE rotates first by their positions (interleaved
        pairs; fp32 tables [positions, head_dim / 2], past them by the last row), in
        the same launch.  Returns the query rows q [rows, heads, head_dim] rotated in
        the same way, a new tensor.  Rows of no sequence hold anything in it."""
        key = self._new_rows(key, self.kv_heads, "HIP paged append", 4)
        value = self._new_rows(value, self.kv_heads, "HIP paged append", 4)
        heads = q.shape[1] if q.ndim == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise RuntimeError("HIP paged append takes query rows [rows, heads, head_dim] of a "
                               "multiple of the cache's kv heads")
        q = self._new_rows(q, heads, "HIP paged append", 4)
        if not key.shape[0] == value.shape[0] == q.shape[0]:
            raise RuntimeError("as many rows of queries and values as of keys")
        for x in (cos, sin):
            if x.dtype != torch.float32 or x.device != self.device or not x.is_contiguous() or \
                    x.ndim != 2 or x.shape != (cos.shape[0], self.head_dim // 2) or not len(x):
                raise RuntimeError("RoPE tables must be contiguous fp32 [positions, head_dim / 2] "
                                   "on the cache's device")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        b = self._batch(batch)
        (kr, kh, _), (vr, vh, _), (qr, qh, _) = key.stride(), value.stride(), q.stride()
        with _on(self.device):
            _abi.check(_abi.load().parrot_paged_append_rope_bf16(
                self._at, b, key.data_ptr(), kr, kh, value.data_ptr(), vr, vh, key.shape[0],
                cos.data_ptr(), sin.data_ptr(), cos.shape[0], q.data_ptr(), qr, qh, heads,
                out.data_ptr(), _stream(self.device)), "parrot_paged_append_rope_bf16")
        return out

    def read(self, batch: PagedBatch, positions: int,
             out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
        """Keys and values of positions 0 .. positions - 1 of every sequence, bf16
        [b, kv_heads, positions, head_dim], zero from a sequence's length on and
        where it has no page.  ``out``: the two tensors to write them into (such as
        ``LocalKVCache.key[:, :, :positions]``; strides that are multiples of 4)."""
        if torch.is_grad_enabled():
            raise RuntimeError("HIP paged read is inference-only; disable gradients")
        if self.device.type != "cuda":
            raise RuntimeError(f"HIP paged read requires a ROCm (cuda) cache, got {self.device}")
        b = self._batch(batch)
        shape = (batch.table.shape[0], self.kv_heads, positions, self.head_dim)
        if out is None:
            key = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
            value = torch.empty_like(key)
        else:
            key, value = out
            for x in out:
                if x.dtype != torch.bfloat16 or x.device != self.device or x.shape != shape or \
                        x.stride(3) != 1 or any(st % 4 for st in x.stride()[:3]) or \
                        any(st == 0 and n > 1 for st, n in zip(x.stride(), shape)) or \
                        x.data_ptr() % 8:
                    raise RuntimeError(f"out must be two bf16 tensors {list(shape)} on the cache's "
                                       "device, strides multiples of 4, no element in two places")
        with _on(self.device):
            _abi.check(_abi.load().parrot_paged_read_bf16(
                self._at, b, positions, key.data_ptr(), *key.stride()[:3], value.data_ptr(),
                *value.stride()[:3], _stream(self.device)), "parrot_paged_read_bf16")
        return key, value

    def attend(self, q: Tensor, batch: PagedBatch, *, scale: float, window: int | None = None,
               sinks: int = 0, out: Tensor | None = None) -> Tensor:
        """Attention of the new rows q [rows, heads, head_dim] (bf16, any row and
        head strides) over their sequences, their own keys and values appended
        before: softmax(q k^T * scale) v with key j visible to the row at position i
        iff j <= i and (j > i - window or j < sinks); scale not 0, up to 2^125 either
        way.  Query head h reads kv head
        h // (heads // kv_heads).  Returns [rows, heads * head_dim] bf16, the
        layout of the output projection's input.  A row that sees no key is 0;
        rows of no sequence are left as they are in ``out`` (a contiguous tensor
        of that shape) and hold anything otherwise."""
        heads = q.shape[1] if q.ndim == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise RuntimeError("HIP paged attention takes rows [rows, heads, head_dim] of a "
                               "multiple of the cache's kv heads")
        q = self._new_rows(q, heads, "HIP paged attention", 8)
        if window is not None and window < 1:
            raise RuntimeError("window must be positive, or None")
        if sinks < 0:
            raise RuntimeError("sinks must not be negative")
        rows, device = q.shape[0], self.device
        b = self._batch(batch)
        if out is None:
            out = q.new_empty((rows, heads * self.head_dim))
        elif out.dtype != torch.bfloat16 or out.device != device or not out.is_contiguous() or \
                out.shape != (rows, heads * self.head_dim) or out.data_ptr() % 8:
            raise RuntimeError(f"out must be a contiguous bf16 tensor [{rows}, "
                               f"{heads * self.head_dim}] on the cache's device")
        window = 0 if window is None else min(window, 2 ** 31 - 1)
        sinks = min(sinks, 2 ** 31 - 1)
        nbytes = self._workspace_bytes(*batch.table.shape, rows, heads, window, sinks)
        # a fresh one per call: calls on several streams share nothing
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        row, head, _ = q.stride()
        with _on(device):
            _abi.check(_abi.load().parrot_paged_attention_bf16(
                self._at, b, q.data_ptr(), row, head, rows, heads, window, sinks, scale,
                out.data_ptr(), _abi.ptr(ws), nbytes, _stream(device)),
                "parrot_paged_attention_bf16")
        return out
