"""A paged KV cache of the MI355X backend, and attention over it.

``PagedKVCache`` holds one layer's keys and values for many sequences in pages,
in bf16, or in 8 or 4 bits (quantised as they are written); ``PagedBatch`` says which
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

# (torch.cuda.current_device() and current_stream().cuda_stream without their checks; a
# PyTorch without GPU support has neither, and calls neither)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_grads = torch.is_grad_enabled

PAGE_TYPES = {torch.bfloat16: 0, torch.float8_e4m3fn: 1, torch.int8: 2}
# an element of such a tensor is two values (None: a PyTorch that does not know the type)
FOUR_BITS = getattr(torch, "float4_e2m1fn_x2", None)
if FOUR_BITS is not None:
    PAGE_TYPES[FOUR_BITS] = 4
PAGE_BLOCK = 32  # a page is a whole number of blocks of so many positions
MOST_ROWS = 2 ** 30  # of a step that a pool places


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
        object.__setattr__(self, "_device", self.table.device)
        object.__setattr__(self, "_sizes", (b, width))
        object.__setattr__(self, "_pool", None)  # the last PagePool that handed it pages

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


def _run(name: str, device: torch.device, *args) -> None:
    """A call of the library on the device's current stream."""
    call, index = getattr(_abi.load(), name), device.index
    if index == _current_device():
        status = call(*args, _raw_stream(index))
    else:
        with _on(device):
            status = call(*args, _raw_stream(index))
    if status:
        _abi.check(status, name)


class PagePool:
    """The pages of one or more caches, handed to sequences and taken back on the GPU.

    ``uses`` int32 [pages] says how many tables name each page; a page with 0 (or less) is
    free.  ``extend`` and ``release`` keep it, and the table, lengths and starts of a
    ``PagedBatch``, so a serving loop whose sequences grow needs no number from the GPU,
    and its step can be captured whole::

        slots, positions = pool.extend(batch, new, rows)
        cache.append(k, v, batch)                        # of every layer
        y = cache.attend(q, batch, ...)
        pool.release(batch, kept, window=2048, sinks=4)  # refused rows, and what the window
                                                         # of the others has left

    What a window has left is gone: a later call that takes positions back does not bring
    it, and then lacks keys that the shorter sequence sees.  So positions that may be taken
    back are, before their window is released or in the same call.

    The caches have pages of the pool's size, and as many at least: their calls refuse a
    batch that a pool of another size, or of pages that they lack, was called with last.

    Calls on one pool or batch belong on one stream, or in order.  A program that lets a
    sequence begin with pages of another adds one to their ``uses`` (and new rows must not
    fall into them, so whole pages are shared)."""

    def __init__(self, pages: int, page_size: int, device="cuda"):
        if pages < 0:
            raise RuntimeError("a pool has no negative number of pages")
        self._describe(torch.zeros(pages, dtype=torch.int32, device=device), page_size)

    @classmethod
    def from_uses(cls, uses: Tensor, page_size: int) -> "PagePool":
        """A pool over a tensor that is there already."""
        self = cls.__new__(cls)
        self._describe(uses, page_size)
        return self

    def _describe(self, uses: Tensor, page_size: int) -> None:
        if uses.dtype != torch.int32 or uses.ndim != 1 or not uses.is_contiguous() or \
                uses.data_ptr() % 16:
            raise RuntimeError("uses must be a contiguous int32 tensor [pages], 16-byte aligned")
        if page_size < 1 or page_size % PAGE_BLOCK:
            raise RuntimeError(f"a page is a multiple of {PAGE_BLOCK} positions")
        self._uses, self.page_size, self.device = uses, page_size, uses.device
        self._struct = _abi.PagedPoolStruct(uses.data_ptr(), uses.shape[0], page_size)
        self._at = ctypes.addressof(self._struct)
        self._cuda = self.device.type == "cuda"
        self._slot = torch.empty(0, dtype=torch.int64, device=self.device)
        self._sizes: dict[tuple, int] = {}

    # (as PagedBatch)
    def __reduce__(self):
        return type(self).from_uses, (self._uses, self.page_size)

    # The calls hand its address over.
    uses = property(lambda self: self._uses)

    def _numbers(self, x: Tensor, batch: PagedBatch, what: str) -> int:
        if x.dtype != torch.int32 or x.device != self.device or not x.is_contiguous() or \
                x.shape != batch._sizes[:1]:
            raise RuntimeError(f"{what} must be a contiguous int32 tensor [b] on the pool's device")
        return x.data_ptr()

    def _batch(self, batch: PagedBatch, what: str) -> int:
        if not self._cuda:
            raise RuntimeError(f"{what} requires a ROCm (cuda) pool, got {self.device}")
        if batch._device != self.device:
            raise RuntimeError("the batch must be on the pool's device")
        object.__setattr__(batch, "_pool", self)
        return batch._at

    def extend(self, batch: PagedBatch, new: Tensor, rows: int) -> tuple[Tensor, Tensor]:
        """Gives each sequence ``new`` [b] (int32, below 0: none) more positions and the
        pages for them, in place: ``batch.lengths`` grow, ``batch.starts`` are this step's
        rows, ``batch.table`` names the pages, of which ``uses`` become 1.

        The sequences are served in order, each with all of its rows or none: it gets them
        iff its table has room, the new rows up to it come to no more than ``rows`` (what
        the step's operands hold), and it needs no page or the pages needed up to it come
        to no more than are free (what does not fit its own table asks for nothing; what is
        refused otherwise still counts, so that nobody is overtaken).  A sequence that is
        refused stays as it is, without new rows.  The lowest free pages go first.

        Columns of the table past a sequence's length must name no page (-1): what stands
        there is overwritten, and a use that it had is never given back.

        Returns ``slots`` int64 [rows], each new row's place in the pool (page *
        page_size + position in it), and ``positions`` int32 [rows]; both -1 past the last
        row, and a slot -1 where the table names no page of the pool."""
        if not 0 <= rows <= MOST_ROWS:  # (before memory is taken for them)
            raise RuntimeError(f"a step of a page pool has 0 to {MOST_ROWS} rows, got {rows}")
        at = self._batch(batch, "HIP page pool")
        fresh = self._numbers(new, batch, "new")
        slots, positions = self._slot.new_empty(rows), new.new_empty(rows)
        b = batch._sizes[0]
        nbytes = self._sizes.get((b, rows))
        if nbytes is None:
            if len(self._sizes) >= 256:
                self._sizes.clear()
            nbytes = self._sizes[b, rows] = _abi.load().parrot_paged_extend_workspace_bytes(
                self._uses.shape[0], b, rows)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        _run("parrot_paged_extend", self.device, self._at, at, fresh, rows, slots.data_ptr(),
             positions.data_ptr(), ws.data_ptr() if nbytes else None, nbytes)
        return slots, positions

    def release(self, batch: PagedBatch, lengths: Tensor | None = None, *,
                window: int | None = None, sinks: int = 0) -> None:
        """Takes positions back, in place: each sequence keeps its first ``lengths`` [b]
        (int32; 0 ends it, more than it has changes nothing; None: all of each), and pages
        wholly past them lose a use and their entry in the table, which becomes -1.  With a
        ``window`` so do the pages that no later position sees, from the kept lengths on, all
        but those of the first ``sinks`` positions: lengths that no call may shorten again
        (rows that may still be refused are not to be counted; give ``lengths`` without them
        in the same call).  ``batch.starts`` stay as they are."""
        at = self._batch(batch, "HIP page pool")
        to = None if lengths is None else self._numbers(lengths, batch, "lengths")
        if window is not None and window < 1:
            raise RuntimeError("window must be positive, or None")
        if sinks < 0:
            raise RuntimeError("sinks must not be negative")
        window = 0 if window is None else min(window, 2 ** 31 - 1)
        _run("parrot_paged_release", self.device, self._at, at, to, window, min(sinks, 2 ** 31 - 1))


class PagedKVCache:
    """Pages of keys and values of one layer.

    ``key`` / ``value`` [pages, kv_heads, page_size / 32, 32 head_dim] of ``dtype``
    (bf16, float8_e4m3fn, int8, or float4_e2m1fn_x2, whose elements are two values, half
    as many) hold blocks of 32 positions in the order in which the attention kernels read
    them (include/parrot_hip.h); ``read`` gives
    rows.  8-bit rows are scaled by a power of two of their own, one byte per
    position and head in ``key_exponent`` / ``value_exponent`` [pages, kv_heads,
    page_size], so that a stored value is exact in bf16.  What that costs, for
    normally distributed rows of 96: 2.7 % of the row's norm in e4m3 (whatever
    the row holds: its error goes with the value), 0.9 % in int8.  A row with a
    NaN or an infinity reads back as NaN.

    4 bits (e2m1): a power of two for 32 dims of a key each, ``key_exponent`` [pages,
    kv_heads, page_size / 32, head_dim], and one for a value row as above; it leaves the
    largest magnitude above 3.5 and not above 7, which becomes 6.  11.2 % of a normal
    key's norm, 11.4 % of a value's, in 100 bytes for both of 96 (int8: 194).  32 dims with
    a NaN or an infinity read back as NaN."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        self._check(pages, page_size, kv_heads, head_dim, dtype)
        # (8 bits as bytes that are viewed: no tensor beside those that are kept)
        byte = torch.uint8 if dtype.itemsize == 1 else dtype
        shape = (pages, kv_heads, page_size // PAGE_BLOCK,
                 PAGE_BLOCK * head_dim // (2 if dtype == FOUR_BITS else 1))
        rows = [torch.zeros(shape, dtype=byte, device=device).view(dtype) for _ in range(2)]
        exponents = [None, None] if dtype == torch.bfloat16 else \
            [torch.zeros(x, dtype=torch.uint8, device=device)
             for x in self._exponent_shapes(*shape[:3], head_dim, dtype)]
        self._describe(*rows, *exponents)

    @staticmethod
    def _exponent_shapes(pages: int, kv_heads: int, blocks: int, head_dim: int, dtype):
        rows = (pages, kv_heads, blocks * PAGE_BLOCK)
        return ((pages, kv_heads, blocks, head_dim) if dtype == FOUR_BITS else rows), rows

    @classmethod
    def from_pages(cls, key: Tensor, value: Tensor, key_exponent: Tensor | None = None,
                   value_exponent: Tensor | None = None) -> "PagedKVCache":
        """A cache over tensors that are there already, laid out as above."""
        per_dim = PAGE_BLOCK // 2 if key.dtype == FOUR_BITS else PAGE_BLOCK
        if key.ndim != 4 or key.shape[3] % per_dim:
            raise RuntimeError("pages are [pages, kv_heads, page_size / 32, 32 head_dim] (4 bits: "
                               "16 head_dim)")
        pages, kv_heads, blocks, width = key.shape
        cls._check(pages, blocks * PAGE_BLOCK, kv_heads, width // per_dim, key.dtype)
        exponents = () if key.dtype == torch.bfloat16 else (key_exponent, value_exponent)
        if value.shape != key.shape or value.dtype != key.dtype or \
                not (key.is_contiguous() and value.is_contiguous()):
            raise RuntimeError("key and value pages must be contiguous, of one shape and type")
        for x, shape in zip(exponents, cls._exponent_shapes(pages, kv_heads, blocks,
                                                            width // per_dim, key.dtype)):
            if x is None or x.dtype != torch.uint8 or not x.is_contiguous() or x.shape != shape:
                raise RuntimeError("8-bit and 4-bit pages need contiguous uint8 exponents "
                                   f"{list(shape)}")
        if any(x.device != key.device for x in (value, *exponents)):
            raise RuntimeError("a cache's tensors must be on one device")
        self = cls.__new__(cls)
        self._describe(key, value, *(exponents or (None, None)))
        return self

    # (as PagedBatch; 4 bits as bytes, since pickle knows no tensors of that type)
    def __reduce__(self):
        if self.dtype != FOUR_BITS:
            return type(self).from_pages, self._tensors
        return type(self)._from_bytes, (*(x.view(torch.uint8) for x in self._tensors[:2]),
                                        *self._tensors[2:])

    @classmethod
    def _from_bytes(cls, key: Tensor, value: Tensor, *exponents: Tensor) -> "PagedKVCache":
        return cls.from_pages(key.view(FOUR_BITS), value.view(FOUR_BITS), *exponents)

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
        self.dtype, self.device = self.key.dtype, self.key.device
        self._cuda = self.device.type == "cuda"
        self._row = torch.empty(0, dtype=torch.bfloat16, device=self.device)
        self.head_dim = width * (2 if self.dtype == FOUR_BITS else 1) // PAGE_BLOCK
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
        if batch._device != self.device:
            raise RuntimeError("the batch must be on the cache's device")
        pool = batch._pool
        if pool is not None and (pool.page_size != self.page_size or
                                 pool._struct.pages > self._struct.pages):
            raise RuntimeError(f"the batch's pool has {pool._struct.pages} pages of {pool.page_size} "
                               f"positions, the cache {self._struct.pages} of {self.page_size}")
        return batch._at

    def _new_rows(self, x: Tensor, heads: int, what: str, step: int):
        """The rows as the kernels read them: their number, the tensor, its address, row and
        head strides."""
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or \
                x.dtype != torch.bfloat16 or x.device != self.device or not self._cuda or _grads():
            _require(x, what)
            raise RuntimeError(f"{what} takes rows [rows, {heads}, {self.head_dim}] on the "
                               "cache's device")
        row, head, one = x.stride()
        at = x.data_ptr()
        if one != 1 or row % step or head % step or at % (2 * step):
            x = x.clone(memory_format=torch.contiguous_format)
            (row, head, _), at = x.stride(), x.data_ptr()
        return shape[0], x, at, row, head

    def append(self, key: Tensor, value: Tensor, batch: PagedBatch) -> None:
        """Writes the new rows key and value [rows, kv_heads, head_dim] (bf16, any
        row and head strides) into their sequences' pages.  Other positions stay
        as they are.  A page that is written must belong to one sequence, once."""
        rows, key, k, kr, kh = self._new_rows(key, self.kv_heads, "HIP paged append", 4)
        values, value, v, vr, vh = self._new_rows(value, self.kv_heads, "HIP paged append", 4)
        if rows != values:
            raise RuntimeError("as many rows of values as of keys")
        _run("parrot_paged_append_bf16", self.device, self._at, self._batch(batch), k, kr, kh, v, vr,
             vh, rows)

    def append_rope(self, q: Tensor, key: Tensor, value: Tensor, batch: PagedBatch, cos: Tensor,
                    sin: Tensor) -> Tensor:
        """``append`` of keys that RoPE rotates first by their positions (interleaved
        pairs; fp32 tables [positions, head_dim / 2], past them by the last row), in
        the same launch.  Returns the query rows q [rows, heads, head_dim] rotated in
        the same way, a new tensor.  Rows of no sequence hold anything in it."""
        rows, key, *k = self._new_rows(key, self.kv_heads, "HIP paged append", 4)
        values, value, *v = self._new_rows(value, self.kv_heads, "HIP paged append", 4)
        heads = q.shape[1] if q.ndim == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise RuntimeError("HIP paged append takes query rows [rows, heads, head_dim] of a "
                               "multiple of the cache's kv heads")
        queries, q, *query = self._new_rows(q, heads, "HIP paged append", 4)
        if not rows == values == queries:
            raise RuntimeError("as many rows of queries and values as of keys")
        for x in (cos, sin):
            if x.dtype != torch.float32 or x.device != self.device or not x.is_contiguous() or \
                    x.ndim != 2 or x.shape != (cos.shape[0], self.head_dim // 2) or not len(x):
                raise RuntimeError("RoPE tables must be contiguous fp32 [positions, head_dim / 2] "
                                   "on the cache's device")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _run("parrot_paged_append_rope_bf16", self.device, self._at, self._batch(batch), *k, *v, rows,
             cos.data_ptr(), sin.data_ptr(), cos.shape[0], *query, heads, out.data_ptr())
        return out

    def read(self, batch: PagedBatch, positions: int,
             out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
        """Keys and values of positions 0 .. positions - 1 of every sequence, bf16
        [b, kv_heads, positions, head_dim], zero from a sequence's length on and
        where it has no page.  ``out``: the two tensors to write them into (such as
        ``LocalKVCache.key[:, :, :positions]``; strides that are multiples of 4)."""
        if _grads():
            raise RuntimeError("HIP paged read is inference-only; disable gradients")
        if not self._cuda:
            raise RuntimeError(f"HIP paged read requires a ROCm (cuda) cache, got {self.device}")
        b = self._batch(batch)
        heads, d = self.kv_heads, self.head_dim
        shape = (batch._sizes[0], heads, positions, d)
        if out is None:
            key = self._row.new_empty(shape)
            value = torch.empty_like(key)
            step = positions * d
            _run("parrot_paged_read_bf16", self.device, self._at, b, positions, key.data_ptr(),
                 heads * step, step, d, value.data_ptr(), heads * step, step, d)
        else:
            key, value = out
            for x in out:
                if x.dtype != torch.bfloat16 or x.device != self.device or x.shape != shape or \
                        x.stride(3) != 1 or any(st % 4 for st in x.stride()[:3]) or \
                        any(st == 0 and n > 1 for st, n in zip(x.stride(), shape)) or \
                        x.data_ptr() % 8:
                    raise RuntimeError(f"out must be two bf16 tensors {list(shape)} on the cache's "
                                       "device, strides multiples of 4, no element in two places")
            _run("parrot_paged_read_bf16", self.device, self._at, b, positions, key.data_ptr(),
                 *key.stride()[:3], value.data_ptr(), *value.stride()[:3])
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
        shape = q.shape
        heads = shape[1] if len(shape) == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise RuntimeError("HIP paged attention takes rows [rows, heads, head_dim] of a "
                               "multiple of the cache's kv heads")
        rows, q, query, row, head = self._new_rows(q, heads, "HIP paged attention", 8)
        if window is not None and window < 1:
            raise RuntimeError("window must be positive, or None")
        if sinks < 0:
            raise RuntimeError("sinks must not be negative")
        device = self.device
        b = self._batch(batch)
        if out is None:
            out = q.new_empty((rows, heads * self.head_dim))
        elif out.dtype != torch.bfloat16 or out.device != device or not out.is_contiguous() or \
                out.shape != (rows, heads * self.head_dim) or out.data_ptr() % 8:
            raise RuntimeError(f"out must be a contiguous bf16 tensor [{rows}, "
                               f"{heads * self.head_dim}] on the cache's device")
        window = 0 if window is None else min(window, 2 ** 31 - 1)
        sinks = min(sinks, 2 ** 31 - 1)
        nbytes = self._workspace_bytes(*batch._sizes, rows, heads, window, sinks)
        # a fresh one per call: calls on several streams share nothing
        # (of bf16: two bytes an element)
        ws = self._row.new_empty((nbytes + 1) // 2) if nbytes else None
        _run("parrot_paged_attention_bf16", device, self._at, b, query, row, head, rows, heads,
             window, sinks, scale, out.data_ptr(), ws.data_ptr() if nbytes else None, nbytes)
        return out
