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
// One workgroup makes the plan: for each sequence where its rows begin and the rank of its
// first page, for each group of 64 pages which are free and the rank of the first of them.
// Rows are placed from that alone, by two searches, in the same launch up to kSmallRows rows
// and in a second one past that.
//
// What bounds it: a chain of loads (lengths and uses, then each sequence's last page) and four
// barriers of one workgroup; for many rows the bytes of their slots and positions, and, of each
// workgroup of the second launch, the plan's read and two searches before the first.  Measured: 8
// sequences' next token, 4096 pages, 5.0 us; 32 of 6 rows, 8192 pages, 6.0; 400 prompts of up to
// 4096, 40000 pages, 8.5 for the plan and 10.4 for 1.23 million rows (14.8 MB, 1.4 TB/s); release
// 2.6 to 3.0.  One workgroup that looks at each page twice took 43 us for that plan, and 6.4 and
// 9.5 for the others.  Not kept: 8 rows a thread in the second launch (12.5 us), 2 rows and 512
// threads (12.4), 1024 threads (12.2).
#include <algorithm>

#include "paged.h"

namespace parrot {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr uint32_t kMost = (1u << 30) + 1;  // rows and pages are 2^30 at most
constexpr int kSmallRows = 8192;
constexpr int kGroup = 64;                 // pages
constexpr int kRound = kThreads * kGroup;  // pages that the workgroup looks through at once

__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return min(a + b, kMost); }

// The sum up to and with this lane's value.
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
  auto step = [&](auto control, auto rows) {
    v = add(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                   0, static_cast<int>(v), decltype(control)::value, decltype(rows)::value, 0xf,
                   false)));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return v;
}

__device__ __forceinline__ uint32_t last_lane(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1));
}

// The sums of the waves before this one, and of all.
struct Sums {
  uint32_t before, all;
};

typedef uint32_t WaveSums[kWaves] __attribute__((aligned(16)));

__device__ __forceinline__ Sums over_waves(const WaveSums& s) {
  const int wave = threadIdx.x / kWave;
  Sums r{0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; w += 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(s + w);
    const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.before = add(r.before, w + i < wave ? v[i] : 0);
      r.all = add(r.all, v[i]);
    }
  }
  return r;
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
    for (int j = 0; j < 4; ++j)
      if (at + j < p.pages && p.uses[at + j] <= 0) free |= 1u << j;
  }
  return free;
}

// A round's pages, read four to a thread at a time, and then as groups of kGroup, one a
// thread: which are free.
struct Round {
  static constexpr int kQuads = kGroup / 4, kStep = 4 * kThreads;
  // (quads: a byte for each four pages of the round)
  static __device__ __forceinline__ void load(const PagedPool& p, int64_t from, uint8_t* quads) {
    const int t = threadIdx.x;
    uint32_t bits[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; ++j)  // (the loads of all quads at once)
      bits[j] = from + j * kStep < p.pages ? free_pages(p, from + j * kStep + 4 * t) : 0;
#pragma unroll
    for (int j = 0; j < kQuads; ++j) quads[j * kThreads + t] = static_cast<uint8_t>(bits[j]);
  }
  static __device__ __forceinline__ uint64_t group(const uint8_t* quads) {
    const uint4 w = *reinterpret_cast<const uint4*>(quads + kQuads * threadIdx.x);
    auto half = [](uint32_t x) {  // four bytes of four bits
      x = (x | (x >> 4)) & 0x00ff00ffu;
      return (x | (x >> 8)) & 0xffffu;
    };
    return static_cast<uint64_t>(half(w.x) | (half(w.y) << 16)) |
           (static_cast<uint64_t>(half(w.z) | (half(w.w) << 16)) << 32);
  }
};

// The r-th set bit.
__device__ __forceinline__ int nth_bit(uint64_t mask, int r) {
  uint32_t m = static_cast<uint32_t>(mask);
  int at = 0;
  if (const int n = __popc(m); r >= n) {
    r -= n;
    at = 32;
    m = static_cast<uint32_t>(mask >> 32);
  }
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) {
    const int n = __popc(m & ((1u << d) - 1));
    if (r >= n) {
      r -= n;
      at += d;
      m >>= d;
    }
  }
  return at;
}

// What a sequence's rows are placed by: the number of its first, its old length, the rank of
// the first page that it got, and its last page before that (-1: none).
struct __attribute__((aligned(16))) Placed {
  int32_t from, old, rank, last;
};

// (in LDS, or in the workspace for a second launch)
struct Plan {
  Placed* sequences;  // [batch + 1]: of the last only `from`, all rows
  uint64_t* free;     // [groups]
  int32_t* ranks;     // [groups]
  int32_t* groups;    // their number, as many as it took
};

struct ExtendArgs {
  PagedPool pool;
  PagedBatch batch;
  const int32_t* fresh;  // new rows of each sequence
  int64_t* slots;
  int32_t* positions;
  Plan plan;
};

// The last of n whose number is at most x, the first's being so.
template <typename F>
__device__ __forceinline__ int last_upto(int n, int x, F number) {
  int low = 0, high = n;
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (number(mid) <= x) low = mid;
    else high = mid;
  }
  return low;
}

// The page of the free ones' rank k.
__device__ __forceinline__ int page_of_rank(const Plan& plan, int groups, int k) {
  const int g = last_upto(groups, k, [&](int i) { return plan.ranks[i]; });
  return g * kGroup + nth_bit(plan.free[g], k - plan.ranks[g]);
}

// N rows from `row` on (rows: those that sequences have).  A page's first row enters it
// into the table: a new page has a new row as its first.
template <int N>
__device__ __forceinline__ void place(const ExtendArgs& a, const Plan& plan, int groups, int rows,
                                      int row, int64_t (&slot)[N], int32_t (&position)[N]) {
  const int size = a.pool.page;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    slot[j] = -1;
    position[j] = -1;
  }
  if (row >= rows) return;
  int i = last_upto(a.batch.batch, row, [&](int i) { return plan.sequences[i].from; });
  Placed x = plan.sequences[i];
  int end = plan.sequences[i + 1].from, column = -1, page = -1, in = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (row + j >= rows) return;
    if (row + j >= end) {
      do x = plan.sequences[++i], end = plan.sequences[i + 1].from;
      while (row + j >= end);
      column = -1;
    }
    const int p = x.old + row + j - x.from;
    if (column < 0 || ++in == size) {
      column = p / size;
      in = p - column * size;
      const int have = pages_of(x.old, size);
      page = column < have ? x.last : page_of_rank(plan, groups, x.rank + column - have);
    }
    position[j] = p;
    if (page >= 0 && page < a.pool.pages) slot[j] = static_cast<int64_t>(page) * size + in;
    if (in == 0) {
      const_cast<int32_t*>(a.batch.table)[static_cast<int64_t>(i) * a.batch.width + column] = page;
      a.pool.uses[page] = 1;
    }
  }
}

// The last page of a sequence before its new rows, -1 for none.
__device__ __forceinline__ int last_page(const PagedBatch& b, int page, int i, int length) {
  return length > 0 && length <= b.width * page
             ? b.table[static_cast<int64_t>(i) * b.width + (length - 1) / page]
             : -1;
}

// SMALL: at most kThreads sequences, kRound pages and kSmallRows rows, which are placed too.
template <bool SMALL>
__global__ __launch_bounds__(kThreads) void extend_kernel(ExtendArgs a) {
  __shared__ WaveSums take_s, need_s, free_s, grant_s;
  __shared__ __attribute__((aligned(16))) uint8_t quads_s[kRound / 4];
  __shared__ Placed sequences_s[SMALL ? kThreads + 1 : 1];
  __shared__ uint64_t groups_s[SMALL ? kThreads : 1];
  __shared__ int32_t ranks_s[SMALL ? kThreads : 1];
  const PagedPool& p = a.pool;
  const PagedBatch& b = a.batch;
  const Plan plan = SMALL ? Plan{sequences_s, groups_s, ranks_s, nullptr} : a.plan;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;

  Asked x = asked(p, b, a.fresh, t);
  Round::load(p, 0, quads_s);
  int last = t < b.batch ? last_page(b, p.page, t, x.length) : -1;
  uint32_t take = wave_upto(x.take), need = wave_upto(x.need);
  if (lane == kWave - 1) {
    take_s[wave] = take;
    need_s[wave] = need;
  }
  __syncthreads();
  uint32_t wanted = over_waves(need_s).all;  // of the first kThreads sequences; then of all
  if constexpr (!SMALL) {
    for (int c = kThreads; c < b.batch; c += kThreads) {
      const uint32_t all = last_lane(wave_upto(asked(p, b, a.fresh, c + t).need));
      __syncthreads();
      if (lane == 0) grant_s[wave] = all;
      __syncthreads();
      wanted = add(wanted, over_waves(grant_s).all);
    }
  }
  // Free pages, a round after the other while there are too few: no more than rows, since
  // each that is handed out has a new row.
  const uint32_t most = min(wanted, static_cast<uint32_t>(b.rows));
  uint32_t there = 0;
  int groups = 0;
  for (int64_t from = 0;;) {
    const uint64_t free = Round::group(quads_s);
    const uint32_t mine = __popcll(free), upto = wave_upto(mine);
    if (lane == kWave - 1) free_s[wave] = upto;
    __syncthreads();
    const Sums n = over_waves(free_s);
    if (from + t * kGroup < p.pages) {
      plan.free[groups + t] = free;
      plan.ranks[groups + t] = static_cast<int>(there + n.before + upto - mine);
    }
    there += n.all;
    groups += static_cast<int>(min(int64_t{kThreads}, (p.pages - from + kGroup - 1) / kGroup));
    from += kRound;
    if (SMALL || there >= most || from >= p.pages) break;
    Round::load(p, from, quads_s);  // (past the barrier: the bytes before are read)
    __syncthreads();
  }
  // Who gets what.  (sums of the sequences before these, all that asked and those granted)
  uint32_t rows_before = 0, pages_before = 0, granted = 0;
  for (int c = 0;;) {
    const Sums r = over_waves(take_s), n = over_waves(need_s);
    const uint32_t upto_rows = add(add(rows_before, r.before), take);
    const uint32_t upto_pages = add(add(pages_before, n.before), need);
    const bool yes = upto_rows <= static_cast<uint32_t>(b.rows) &&
                     (x.need == 0 || upto_pages <= there);
    const uint32_t mine = yes ? x.take : 0, upto = wave_upto(mine);
    if (!SMALL) __syncthreads();  // (the sums before are read)
    if (lane == kWave - 1) grant_s[wave] = upto;
    __syncthreads();
    const Sums g = over_waves(grant_s);
    if (c + t < b.batch) {
      const int first = static_cast<int>(granted + g.before + upto - mine);
      const_cast<int32_t*>(b.starts)[c + t] = first;
      if (mine > 0) const_cast<int32_t*>(b.lengths)[c + t] = x.length + static_cast<int>(mine);
      plan.sequences[c + t] = {first, x.length, static_cast<int>(upto_pages - x.need), last};
    }
    granted += g.all;
    rows_before = add(rows_before, r.all);
    pages_before = add(pages_before, n.all);
    c += kThreads;
    if (SMALL || c >= b.batch) break;
    x = asked(p, b, a.fresh, c + t);
    last = c + t < b.batch ? last_page(b, p.page, c + t, x.length) : -1;
    take = wave_upto(x.take), need = wave_upto(x.need);
    if (lane == kWave - 1) {
      take_s[wave] = take;
      need_s[wave] = need;
    }
    __syncthreads();
  }
  if (t == 0) {
    const_cast<int32_t*>(b.starts)[b.batch] = static_cast<int32_t>(granted);
    plan.sequences[b.batch] = {static_cast<int32_t>(granted), 0, 0, 0};
    if (!SMALL) *plan.groups = groups;
  }
  if constexpr (SMALL) {
    __syncthreads();
    for (int row = t; row < b.rows; row += kThreads) {
      int64_t slot[1];
      int32_t position[1];
      place(a, plan, groups, static_cast<int>(granted), row, slot, position);
      a.slots[row] = slot[0];
      a.positions[row] = position[0];
    }
  }
}

// The second launch: four rows a thread.  HELD: the plan is read into LDS first (kThreads
// sequences and groups at most).
template <bool HELD>
__global__ __launch_bounds__(256) void place_kernel(ExtendArgs a) {
  __shared__ Placed sequences_s[HELD ? kThreads + 1 : 1];
  __shared__ uint64_t groups_s[HELD ? kThreads : 1];
  __shared__ int32_t ranks_s[HELD ? kThreads : 1];
  Plan plan = a.plan;
  const int groups = *plan.groups, t = threadIdx.x;
  if constexpr (HELD) {
    for (int i = t; i <= a.batch.batch; i += 256) sequences_s[i] = plan.sequences[i];
    const int most = static_cast<int>((a.pool.pages + kGroup - 1) / kGroup);
    for (int i = t; i < most; i += 256) {  // (those past `groups` hold anything)
      groups_s[i] = plan.free[i];
      ranks_s[i] = plan.ranks[i];
    }
    __syncthreads();
    plan = Plan{sequences_s, groups_s, ranks_s, nullptr};
  }
  const int row = 4 * static_cast<int>(blockIdx.x * 256 + t), rows = plan.sequences[a.batch.batch].from;
  if (row >= a.batch.rows) return;
  int64_t slot[4];
  int32_t position[4];
  place(a, plan, groups, rows, row, slot, position);
  if (row + 3 < a.batch.rows) {
    *reinterpret_cast<int4*>(a.positions + row) =
        make_int4(position[0], position[1], position[2], position[3]);
    *reinterpret_cast<longlong2*>(a.slots + row) = make_longlong2(slot[0], slot[1]);
    *reinterpret_cast<longlong2*>(a.slots + row + 2) = make_longlong2(slot[2], slot[3]);
  } else {
    for (int j = 0; j < 4 && row + j < a.batch.rows; ++j) {
      a.slots[row + j] = slot[j];
      a.positions[row + j] = position[j];
    }
  }
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

namespace {

bool one_launch(int64_t pages, int batch, int rows) {
  return batch <= kThreads && pages <= kRound && rows <= kSmallRows;
}

int64_t groups_of(int64_t pages) { return (pages + kGroup - 1) / kGroup; }

}  // namespace

size_t paged_extend_workspace_bytes(int64_t pages, int batch, int rows) {
  if (one_launch(pages, batch, rows)) return 0;
  return (static_cast<size_t>(batch) + 2) * sizeof(Placed) +
         static_cast<size_t>(groups_of(pages)) * (sizeof(uint64_t) + sizeof(int32_t));
}

hipError_t launch_paged_extend(const PagedPool& pool, const PagedBatch& batch, const int32_t* fresh,
                               int64_t* slots, int32_t* positions, void* workspace,
                               hipStream_t s) {
  ExtendArgs a{pool, batch, fresh, slots, positions, {}};
  if (one_launch(pool.pages, batch.batch, batch.rows)) {
    extend_kernel<true><<<1, kThreads, 0, s>>>(a);
    return hipGetLastError();
  }
  const int64_t groups = groups_of(pool.pages);
  a.plan.groups = static_cast<int32_t*>(workspace);  // (16 bytes)
  a.plan.sequences = static_cast<Placed*>(workspace) + 1;
  a.plan.free = reinterpret_cast<uint64_t*>(a.plan.sequences + batch.batch + 1);
  a.plan.ranks = reinterpret_cast<int32_t*>(a.plan.free + groups);
  extend_kernel<false><<<1, kThreads, 0, s>>>(a);
  const int grid = (batch.rows + 1023) / 1024;
  if (grid > 0 && batch.batch <= kThreads && groups <= kThreads)
    place_kernel<true><<<grid, 256, 0, s>>>(a);
  else if (grid > 0)
    place_kernel<false><<<grid, 256, 0, s>>>(a);
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
