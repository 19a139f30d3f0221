// Pages handed out and taken back on the GPU: the tables, starts, positions and slots of a
// step from its sequences' lengths.
//
//   need_i = ceil((length_i + new_i) / page) - ceil(length_i / page)
//   R_i, P_i = the running sums of new rows and of needed pages up to sequence i
// Sequence i gets its rows iff its table holds them, R_i <= rows and (need_i = 0 or P_i is
// not more than there are free pages); the pages it gets are the free ones of ranks
// P_i - need_i .. P_i - 1, the lowest first.  So what is handed out depends on the sums
// alone and not on the order in which anything runs.  Sums stop at kMost, past any number
// that is granted, which keeps them in 32 bits (and stays associative).
//
// What bounds it: one launch, and in it a chain of loads (lengths, then uses, then, for the
// rows, the table just written).
#include <algorithm>

#include "paged.h"

namespace parrot {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr uint32_t kMost = (1u << 30) + 1;  // rows and pages are 2^30 at most
constexpr int kLdsSequences = 4096;
constexpr int kPerThread = 4;  // pages

__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return min(a + b, kMost); }

// The sum of what the threads before this one give, and of all.
struct Sums {
  uint32_t before, all;
};

__device__ __forceinline__ Sums block_sums(uint32_t v, uint32_t (&s)[kWaves]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t upto = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t x = static_cast<uint32_t>(__shfl_up(static_cast<int>(upto), d));
    if (lane >= d) upto = add(upto, x);
  }
  __syncthreads();  // (s may be read still)
  if (lane == kWave - 1) s[wave] = upto;
  __syncthreads();
  uint32_t before = static_cast<uint32_t>(__shfl_up(static_cast<int>(upto), 1));
  if (lane == 0) before = 0;
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before = add(before, s[w]);
    all = add(all, s[w]);
  }
  return {before, all};
}

struct Asked {
  int length;
  uint32_t take, need;  // new rows; pages for them
};

__device__ __forceinline__ int pages_of(int length, int page) {
  return static_cast<int>((static_cast<uint32_t>(length) + page - 1) / page);
}

__device__ __forceinline__ Asked asked(const PagedPool& p, const PagedBatch& b,
                                       const int32_t* fresh, int i) {
  Asked a{0, 0, 0};
  if (i >= b.batch) return a;
  a.length = max(b.lengths[i], 0);
  const int n = max(fresh[i], 0), room = b.width * p.page;
  if (a.length > room || n > room - a.length) return a;
  a.take = min(static_cast<uint32_t>(n), kMost);
  a.need = pages_of(a.length + n, p.page) - pages_of(a.length, p.page);
  return a;
}

// Bits 0 .. 3: which of the pages at .. at + 3 are free.
__device__ __forceinline__ uint32_t free_pages(const PagedPool& p, int64_t at) {
  uint32_t free = 0;
  if (at + 3 < p.pages) {
    const int4 u = *reinterpret_cast<const int4*>(p.uses + at);
    free = (u.x <= 0 ? 1u : 0u) | (u.y <= 0 ? 2u : 0u) | (u.z <= 0 ? 4u : 0u) |
           (u.w <= 0 ? 8u : 0u);
  } else {
    for (int j = 0; j < kPerThread; ++j)
      if (at + j < p.pages && p.uses[at + j] <= 0) free |= 1u << j;
  }
  return free;
}

// The last i with sums[i] <= x (sums[0] = 0; n of them).
__device__ __forceinline__ int last_upto(const int32_t* sums, int n, int x) {
  int low = 0, high = n;
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (sums[mid] <= x) low = mid;
    else high = mid;
  }
  return low;
}

// Where new row r lies: starts and lengths are the step's.
__device__ __forceinline__ void place_row(const PagedPool& p, const PagedBatch& b,
                                          const int32_t* starts, int row, int64_t* slots,
                                          int32_t* positions) {
  int64_t slot = -1;
  int position = -1;
  if (row < starts[b.batch]) {
    const int i = last_upto(starts, b.batch, row);
    position = b.lengths[i] - starts[i + 1] + row;
    const int at = paged_page(b, PagedCache{nullptr, nullptr, nullptr, nullptr, p.pages, 0, 0}, i,
                              position / p.page);
    if (at >= 0) slot = static_cast<int64_t>(at) * p.page + position % p.page;
  }
  slots[row] = slot;
  positions[row] = position;
}

struct ExtendArgs {
  PagedPool pool;
  PagedBatch batch;
  const int32_t* fresh;  // new rows of each sequence
  int64_t* slots;
  int32_t* positions;
  int32_t* sums;  // [batch + 1], for more than kLdsSequences
};

template <bool LDS>
__global__ __launch_bounds__(kThreads) void extend_kernel(ExtendArgs a, bool place) {
  __shared__ uint32_t scan_s[kWaves];
  __shared__ int32_t pages_s[LDS ? kLdsSequences + 1 : 1], starts_s[LDS ? kLdsSequences + 1 : 1];
  const PagedPool& p = a.pool;
  const PagedBatch& b = a.batch;
  int32_t* const table = const_cast<int32_t*>(b.table);
  int32_t* const lengths = const_cast<int32_t*>(b.lengths);
  int32_t* const starts = const_cast<int32_t*>(b.starts);
  int32_t* const pages_upto = LDS ? pages_s : a.sums;
  int32_t* const rows_upto = LDS ? starts_s : starts;
  const int t = threadIdx.x;

  uint32_t wanted = 0;
  for (int c = 0; c < b.batch; c += kThreads)
    wanted = add(wanted, block_sums(asked(p, b, a.fresh, c + t).need, scan_s).all);
  // Free pages, as many as are wanted at the most.
  uint32_t there = 0;
  for (int64_t c = 0; c < p.pages && there < wanted; c += kThreads * kPerThread)
    there = add(there, block_sums(__popc(free_pages(p, c + t * kPerThread)), scan_s).all);

  uint32_t rows = 0, pages = 0, granted_rows = 0;
  for (int c = 0; c < b.batch; c += kThreads) {
    const Asked x = asked(p, b, a.fresh, c + t);
    const Sums r = block_sums(x.take, scan_s), n = block_sums(x.need, scan_s);
    const bool granted = add(add(rows, r.before), x.take) <= static_cast<uint32_t>(b.rows) &&
                         (x.need == 0 || add(add(pages, n.before), x.need) <= there);
    const Sums g = block_sums(granted ? x.take : 0, scan_s);
    if (c + t < b.batch) {
      pages_upto[c + t] = static_cast<int32_t>(add(pages, n.before));
      const int32_t first = static_cast<int32_t>(granted_rows + g.before);
      starts[c + t] = first;
      if (LDS) starts_s[c + t] = first;
      if (granted && x.take > 0) lengths[c + t] = x.length + static_cast<int>(x.take);
    }
    rows = add(rows, r.all);
    pages = add(pages, n.all);
    granted_rows += g.all;
  }
  if (t == 0) {
    starts[b.batch] = static_cast<int32_t>(granted_rows);
    if (LDS) starts_s[b.batch] = static_cast<int32_t>(granted_rows);
    pages_upto[b.batch] = static_cast<int32_t>(pages);
  }
  __syncthreads();
  // The free pages in order: rank k is sequence i's, sums[i] <= k < sums[i + 1].  Those that
  // were not granted any are the last.
  const uint32_t end = min(there, wanted);
  uint32_t rank = 0;
  for (int64_t c = 0; c < p.pages && rank < end; c += kThreads * kPerThread) {
    const int64_t at = c + t * kPerThread;
    uint32_t free = free_pages(p, at);
    const Sums n = block_sums(__popc(free), scan_s);
    uint32_t k = rank + n.before;
    rank += n.all;
    for (; free != 0 && k < end; ++k, free &= free - 1) {
      const int i = last_upto(pages_upto, b.batch, static_cast<int>(k));
      const int need = pages_upto[i + 1] - pages_upto[i];
      if (static_cast<uint32_t>(pages_upto[i + 1]) > there || rows_upto[i + 1] == rows_upto[i])
        continue;
      const int64_t page = at + __builtin_ctz(free);
      const int column = pages_of(lengths[i], p.page) - need + static_cast<int>(k) - pages_upto[i];
      table[static_cast<int64_t>(i) * b.width + column] = static_cast<int32_t>(page);
      p.uses[page] = 1;
    }
  }
  if (!place) return;
  __syncthreads();
  for (int row = t; row < b.rows; row += kThreads)
    place_row(p, b, rows_upto, row, a.slots, a.positions);
}

__global__ __launch_bounds__(256) void place_kernel(ExtendArgs a) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row < a.batch.rows) place_row(a.pool, a.batch, a.batch.starts, row, a.slots, a.positions);
}

// A sequence a workgroup: its pages past its new length, and those that a window has left.
__global__ __launch_bounds__(256) void release_kernel(PagedPool p, PagedBatch b,
                                                      const int32_t* to, int window, int sinks) {
  const int i = blockIdx.x;
  const int old = max(b.lengths[i], 0), length = to != nullptr ? min(max(to[i], 0), old) : old;
  const int all = min(pages_of(old, p.page), b.width), keep = min(pages_of(length, p.page), all);
  // (column w is left by the window: (w + 1) page <= length - window + 1, and w page >= sinks)
  const int left = length >= window ? (length - window + 1) / p.page : 0;
  const int first = static_cast<int>((static_cast<int64_t>(sinks) + p.page - 1) / p.page);
  int32_t* const row = const_cast<int32_t*>(b.table) + static_cast<int64_t>(i) * b.width;
  auto give = [&](int from, int upto) {
    for (int w = from + static_cast<int>(threadIdx.x); w < upto; w += blockDim.x) {
      const int page = row[w];
      if (page < 0 || page >= p.pages) continue;
      row[w] = -1;
      atomicSub(p.uses + page, 1);
    }
  };
  give(first, min(left, keep));
  give(keep, all);
  __syncthreads();  // (every thread has read the old length)
  if (threadIdx.x == 0 && to != nullptr && b.lengths[i] != length)
    const_cast<int32_t*>(b.lengths)[i] = length;
}

}  // namespace

size_t paged_extend_workspace_bytes(int batch) {
  return batch > kLdsSequences ? (static_cast<size_t>(batch) + 1) * sizeof(int32_t) : 0;
}

hipError_t launch_paged_extend(const PagedPool& pool, const PagedBatch& batch, const int32_t* fresh,
                               int64_t* slots, int32_t* positions, void* workspace,
                               hipStream_t s) {
  const ExtendArgs a{pool, batch, fresh, slots, positions, static_cast<int32_t*>(workspace)};
  const bool place = batch.rows <= 8 * kThreads;
  if (batch.batch <= kLdsSequences) extend_kernel<true><<<1, kThreads, 0, s>>>(a, place);
  else extend_kernel<false><<<1, kThreads, 0, s>>>(a, place);
  if (!place) place_kernel<<<(batch.rows + 255) / 256, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_release(const PagedPool& pool, const PagedBatch& batch, const int32_t* to,
                                int window, int sinks, hipStream_t s) {
  if (batch.batch == 0) return hipSuccess;
  release_kernel<<<batch.batch, batch.width <= 256 ? 64 : 256, 0, s>>>(pool, batch, to, window,
                                                                       sinks);
  return hipGetLastError();
}

}  // namespace parrot
