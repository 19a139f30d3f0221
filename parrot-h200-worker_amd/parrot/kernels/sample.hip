// Drawing a token per row of logits, with temperature, top-k, top-p and min-p,
// from one given uniform number u:
//   w_i = exp((x_i - max x) / T);
//   the top_k largest (equal ones by their index), of those the shortest
//   prefix that holds top_p of their mass, of those w_i >= min_p;
//   the first token, by index, at which the sum of w passes u times the whole.
//
// Weights are 64-bit whole numbers (w 2^shift, rounded; a row's sum fits): their
// sums do not depend on an order, so a row's token does not depend on how the work
// is split, and a border between two tokens lies where it does in 64-bit arithmetic
// up to the errors of single weights (1e-10 of a weight, and its rounding, 2^-47 of
// the largest at 32768 tokens).
//
// A workgroup per row, which keeps the row in LDS (32768 logits; longer rows are
// read again, from L2, in each pass).  Nothing is sorted: the border of top-k or
// top-p is found by one histogram over the distance from the largest logit (in
// whole numbers: counts or weights) and the order of the few logits in the
// border's bin by comparing each with each.  A bin with too many of them (equal
// logits) is split by its range of bit patterns, 2047 parts at a time.
//
// What bounds it: one CU's vector instructions, some 10 clocks per logit and pass
// of 20 instructions, and the 64-bit exponentials.  So with a top_k of up to 512
// the row is passed twice only: the k-th largest of the 1024 threads' maxima bounds
// the k-th largest logit from below, and what passes it, hardly more than k, is
// gathered in the order of indices, one logit a thread.  Without top_k each
// exponential is made once and its weight stays in registers.
//
// Measured (graph of launches): a row of 32768 fp32 logits with top_k 50 and top_p 11.2 us,
// the largest alone 8.4, top_p alone 23.7 (8.5 of 2000 logits), bf16 and fp16 within 1 us;
// 64 rows with parameters of their own as their slowest, 26; the bytes would take 0.1 and 1.7.
// 4 rows of 128000, which each pass reads and weighs again: 34 with top_k 50, 64 without any
// restriction, 101 with top_k 2000, 159 with top_p.
#include <math.h>

#include "common.h"

namespace parrot {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kStep = 4 * kWave;   // logits of a wavefront's step, four a lane
constexpr int kMost = 8;           // steps of a row that LDS holds (32768 logits)
constexpr int kBins = 2048;
constexpr int kList = 256;         // logits compared each with each
constexpr int kTableBits = 8, kTable = 1 << kTableBits;
constexpr int kPairs = 128;        // logits of a list that are ordered each with each
constexpr int kShort = 512;        // top_k for which a list is made

enum LogitType { kLogitF32 = 0, kLogitBf16 = 1, kLogitF16 = 2 };

// 2^(k / 256), by the exponential's series.
struct Powers {
  double at[kTable];
  constexpr Powers() : at() {
    for (int k = 0; k < kTable; ++k) {
      const long double x = 0.693147180559945309417232121458L * k / kTable;
      long double sum = 1.0L, term = 1.0L;
      for (int i = 1; i < 24; ++i) {
        term *= x / i;
        sum += term;
      }
      at[k] = static_cast<double>(sum);
    }
  }
};
__device__ const Powers kPowers;

struct SampleArgs {
  const void* logits;
  int64_t stride;  // elements between rows
  int vocab;
  const float* uniform;
  const float* temperature;  // per row; null: the number beside it for every row
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  double temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int shift;  // weights are w 2^shift
  int64_t* token;
  float* probability;  // optional
};

template <int TYPE>
__device__ __forceinline__ float logit(const void* row, int i) {
  float x;
  if constexpr (TYPE == kLogitF32) x = static_cast<const float*>(row)[i];
  else if constexpr (TYPE == kLogitBf16) x = bf16_to_f32(static_cast<const uint16_t*>(row)[i]);
  else x = static_cast<float>(static_cast<const _Float16*>(row)[i]);
  return x;
}

// Four logits from i on; a NaN is -infinity, what lies past the row a NaN (which is
// larger or smaller than nothing, so no pass over a held row counts it).
// aligned: the row is, and a whole number of fours: loads without a branch.
template <int TYPE>
__device__ __forceinline__ float4 logits4(const void* row, int at, int n, bool aligned) {
  float x[4];
  int i = at;
  if (aligned) {
    i = min(at, n - 4);
    if constexpr (TYPE == kLogitF32) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + i);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + i);
      if constexpr (TYPE == kLogitBf16) {
        x[0] = lo_bf16(v.x), x[1] = hi_bf16(v.x), x[2] = lo_bf16(v.y), x[3] = hi_bf16(v.y);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = static_cast<float>(__builtin_bit_cast(
              _Float16, static_cast<uint16_t>((j < 2 ? v.x : v.y) >> (16 * (j & 1)))));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? logit<TYPE>(row, i + j) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float past = at + j < n ? -INFINITY : __uint_as_float(0x7fc00000u);
    x[j] = x[j] == x[j] && at + j < n ? x[j] : past;
  }
  return make_float4(x[0], x[1], x[2], x[3]);
}

// A row whose largest logit is an infinity: only the infinities are drawn from, alike.
__device__ __forceinline__ float4 finite_of(float4 v) {
  auto f = [](float x) { return x == INFINITY ? 0.0f : x == x ? -INFINITY : x; };
  return make_float4(f(v.x), f(v.y), f(v.z), f(v.w));
}

struct Entry {
  uint64_t f;
  uint32_t key;
  int index;
};

struct Shared {
  double table[kTable];  // 2^(k / 256)
  union {
    uint64_t bins[kBins];
    Entry list[kList];
  };
  float few[kThreads];     // a list of logits and their indices, in order
  int few_index[kThreads];
  uint64_t wave[kWaves];
  uint64_t ahead[kList];  // of a list's logits: the mass before each
  int rank[kList];         // ... and their number
  uint64_t before;
  uint32_t low[kWaves], high[kWaves];
  int found;
  int count;
  float edge;
  int until;
};

// v of another lane by DPP, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The sum of the lanes up to this one: by 1, 2, 4, 8 lanes to the right inside rows
// of 16, then a row's last lane to the next row (rows 1, 3) and lane 31 to the upper
// half (VALU moves; a shuffle is an LDS trip).
__device__ __forceinline__ uint64_t wave_upto(uint64_t v) {
  v += dpp64<0x111, 0xf>(v);
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  v += dpp64<0x142, 0xa>(v);
  return v + dpp64<0x143, 0xc>(v);
}

__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), kWave - 1);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ uint64_t wave_total(uint64_t v) { return last_lane(wave_upto(v)); }

// A row: `steps` times 256 consecutive logits per wavefront, so that sums over
// wavefronts, steps, lanes and a lane's four are sums by index.
// STEPS > 0: the row is held in LDS.
template <int TYPE, int STEPS>
struct Row {
  const void* at;
  const float* held;
  int n, steps;
  bool aligned;
  bool infinite;  // infinities are 0 and everything else is left out (-infinity)
  __device__ __forceinline__ int first(int step) const {
    return (static_cast<int>(threadIdx.x >> 6) * steps + step) * kStep +
           4 * static_cast<int>(threadIdx.x & (kWave - 1));
  }
  __device__ __forceinline__ float4 get(int step) const {
    const int i = first(step);
    if constexpr (STEPS > 0) return *reinterpret_cast<const float4*>(held + i);
    float4 v = logits4<TYPE>(at, i, n, aligned);
    return infinite ? finite_of(v) : v;
  }
  // f(index, logit, weight if one is held) for this thread's logits
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int s = 0; s < steps; ++s) {
      const int i = first(s);
      if (i - 4 * static_cast<int>(threadIdx.x & (kWave - 1)) >= n) break;  // (the wavefront's)
      const float4 v = get(s);
      if (i < n) f(i, v.x, uint64_t{0});
      if (i + 1 < n) f(i + 1, v.y, uint64_t{0});
      if (i + 2 < n) f(i + 2, v.z, uint64_t{0});
      if (i + 3 < n) f(i + 3, v.w, uint64_t{0});
    }
  }
  // The first index at which the sum of f passes `target` (below the whole); f's
  // shares as total() left them.
  template <typename F>
  __device__ __forceinline__ int locate(F f, uint64_t target, Shared& sh) const {
    return locate_by(
        [&](int s, uint64_t(&w)[4]) {
          const int i = first(s);
          const float4 v = get(s);
          w[0] = i < n ? f(i, v.x, uint64_t{0}) : 0;
          w[1] = i + 1 < n ? f(i + 1, v.y, uint64_t{0}) : 0;
          w[2] = i + 2 < n ? f(i + 2, v.z, uint64_t{0}) : 0;
          w[3] = i + 3 < n ? f(i + 3, v.w, uint64_t{0}) : 0;
        },
        target, sh);
  }
  template <typename W>
  __device__ __forceinline__ int locate_by(W weights, uint64_t target, Shared& sh) const {
    const int wave = threadIdx.x >> 6;
    uint64_t before = 0;
    for (int w = 0; w < wave; ++w) before += sh.wave[w];
    if (before <= target && target < before + sh.wave[wave]) {  // one wavefront
      for (int s = 0; s < steps; ++s) {
        uint64_t w[4];
        weights(s, w);
        const uint64_t mine = w[0] + w[1] + w[2] + w[3];
        const uint64_t upto = wave_upto(mine);
        const uint64_t all = last_lane(upto);
        if (target < before + all) {
          uint64_t at = before + upto - mine;
          if (at <= target && target < at + mine) {
            int j = 0;
            while (target >= at + w[0]) {  // (at most three times)
              at += w[0];
              w[0] = w[1], w[1] = w[2], w[2] = w[3];
              ++j;
            }
            sh.found = first(s) + j;
          }
          break;
        }
        before += all;
      }
    }
    __syncthreads();
    return sh.found;
  }
};

// A held row and its weights, in registers (past its end 0).  Of a row of kMost steps the
// steps past its end are left out, which also leaves the compiler fewer registers to spill
// than passing all would (26.6 us for 31.4 at 32768); in keep it is the other way round.
template <typename R, int kSteps>
struct Weights {
  const R row;
  uint64_t w[kSteps][4];
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (kSteps == kMost && s >= row.steps) break;
      const int i = row.first(s);
      const float4 v = row.get(s);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i + j, x[j], w[s][j]);
      __builtin_amdgcn_sched_barrier(0);  // (a step at a time: the weights fill the registers)
    }
  }
  template <typename F>
  __device__ __forceinline__ int locate(F f, uint64_t target, Shared& sh) const {
    return row.locate_by(
        [&](int s, uint64_t(&y)[4]) {
          const int i = row.first(s);
          const float4 v = row.get(s);
          const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int q = 0; q < kSteps; ++q)
            if (q == s) {
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = f(i + j, x[j], w[q][j]);
            }
        },
        target, sh);
  }
  // Leaves out what f does not keep.
  template <typename F>
  __device__ __forceinline__ void keep(F f) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int i = row.first(s);
      const float4 v = row.get(s);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) w[s][j] = f(i + j, x[j], w[s][j]) ? w[s][j] : 0;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The sum of the weights; leaves each wavefront's share in sh.wave.
  __device__ __forceinline__ uint64_t sum(Shared& sh) const {
    uint64_t all = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) all += (w[s][0] + w[s][1]) + (w[s][2] + w[s][3]);
    all = wave_total(all);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh.wave[threadIdx.x >> 6] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all += sh.wave[i];
    return all;
  }
  // The first index at which the sum of the weights passes `target`.
  __device__ __forceinline__ int locate(uint64_t target, Shared& sh) const {
    const int wave = threadIdx.x >> 6;
    uint64_t before = 0;
    for (int i = 0; i < wave; ++i) before += sh.wave[i];
    if (before <= target && target < before + sh.wave[wave]) {  // one wavefront
      bool found = false;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (found) continue;
        const uint64_t mine = (w[s][0] + w[s][1]) + (w[s][2] + w[s][3]);
        const uint64_t upto = before + wave_upto(mine);
        before = last_lane(upto);
        found = target < before;  // one step
        uint64_t at = upto - mine;
        if (found && at <= target && target < at + mine) {
          int j = 0;
          if (target >= at + w[s][0]) at += w[s][0], j = 1;
          if (j == 1 && target >= at + w[s][1]) at += w[s][1], j = 2;
          if (j == 2 && target >= at + w[s][2]) j = 3;
          sh.found = row.first(s) + j;
        }
      }
    }
    __syncthreads();
    return sh.found;
  }
};

// A list of at most one logit a thread, in the order of indices.
struct Few {
  int n;
  float x;     // this thread's
  uint64_t w;  // and its weight
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (static_cast<int>(threadIdx.x) < n) f(static_cast<int>(threadIdx.x), x, w);
  }
  template <typename F>
  __device__ __forceinline__ int locate(F f, uint64_t target, Shared& sh) const {
    const int t = threadIdx.x;
    uint64_t before = 0;
    for (int w = 0; w < (t >> 6); ++w) before += sh.wave[w];
    const uint64_t mine = t < n ? f(t, x, w) : 0;
    before += wave_upto(mine) - mine;
    if (before <= target && target < before + mine) sh.found = t;
    __syncthreads();
    return sh.found;
  }
};

// The sum of f over the row; leaves each wavefront's share in sh.wave.
template <typename R, typename F>
__device__ __forceinline__ uint64_t total(const R& row, F f, Shared& sh) {
  uint64_t t = 0;
  row.each([&](int i, float x, uint64_t w) { t += f(i, x, w); });
  t = wave_total(t);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sh.wave[threadIdx.x >> 6] = t;
  __syncthreads();
  t = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) t += sh.wave[i];
  return t;
}

// The first bin at which the sum over bins reaches `need`, and the sum before it;
// the last bin (kBins - 1, never counted) where the others do not.
__device__ __forceinline__ int find_bin(uint64_t need, uint64_t& before, Shared& sh) {
  const int t = threadIdx.x;
  const uint64_t a = sh.bins[2 * t], b = sh.bins[2 * t + 1];
  uint64_t upto = wave_upto(a + b);
  if ((t & (kWave - 1)) == kWave - 1) sh.wave[t >> 6] = upto;
  if (t == 0) sh.found = kBins - 1;
  __syncthreads();
  uint64_t all = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < (t >> 6)) upto += sh.wave[w];
    all += sh.wave[w];
  }
  if (t == 0 && all < need) sh.before = all;
  if (upto >= need && upto - a - b < need) {
    const bool second = upto - b < need;
    sh.found = 2 * t + second;
    sh.before = second ? upto - b : upto - a - b;
  }
  __syncthreads();
  before = sh.before;
  return sh.found;
}

struct Edge {
  float x;
  int until;
  // (as by order_key: -0 and 0 are equal; there is no NaN)
  __device__ __forceinline__ bool keeps(int i, float y) const {
    return (y > x) | ((y == x) & (i <= until));
  }
};

// The bin of a logit: by its distance from the largest, the last one for all that
// lies further.
struct Bins {
  float top, per_unit;
  __device__ __forceinline__ float distance(float x) const { return (top - x) * per_unit; }
  __device__ __forceinline__ int operator()(float x) const {
    return static_cast<int>(fminf(distance(x), static_cast<float>(kBins - 1)));
  }
  // Whether the logit is in the bin.
  __device__ __forceinline__ bool in(float x, float bin) const {
    const float d = distance(x);
    return d >= bin && (d < bin + 1.0f || bin == static_cast<float>(kBins - 1));
  }
};

__device__ __forceinline__ void clear_bins(Shared& sh) {
  __syncthreads();
  sh.bins[threadIdx.x] = sh.bins[threadIdx.x + kThreads] = 0;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
}

__device__ __forceinline__ void add_to_bin(int bin, uint64_t v, Shared& sh) {
  if (v) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[bin]), v);
}

// Of the n <= kList logits in sh.list: how many of them come before each (in the order
// of size and index), and their sum, to sh.rank and sh.ahead.  Each is compared with
// each, by as many threads a logit as there are.
__device__ __forceinline__ void order_list(int n, Shared& sh) {
  const int t = threadIdx.x;
  const int width = n <= 64 ? 64 : n <= 128 ? 128 : kList;
  const int i = t & (width - 1), parts = kThreads / width, part = t / width;
  if (t < kList) {
    sh.ahead[t] = 0;
    sh.rank[t] = 0;
  }
  __syncthreads();
  if (i < n) {
    const Entry mine = sh.list[i];
    uint64_t sum = 0;
    int rank = 0;
#pragma unroll 4
    for (int j = part; j < n; j += parts) {
      const Entry e = sh.list[j];
      const bool before = (e.key > mine.key) | ((e.key == mine.key) & (e.index < mine.index));
      rank += before;
      sum += before ? e.f : 0;
    }
    if (rank) {
      atomicAdd(&sh.rank[i], rank);
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.ahead[i]), sum);
    }
  }
  __syncthreads();
}

// The last logit, in the order of size and index, that is needed for the sum of f
// to reach `need` (1 .. the whole): its key and index.  filled: the bins hold f's
// sums already.
template <typename R, typename F>
__device__ __forceinline__ Edge select(const R& row, F f, uint64_t need, Bins bin_of, bool filled, Shared& sh) {
  if (!filled) {
    clear_bins(sh);
    row.each([&](int i, float x, uint64_t w) {
      const int b = bin_of(x);
      if (b < kBins - 1) add_to_bin(b, f(i, x, w), sh);
    });
    __syncthreads();
  }
  uint64_t before;
  const int bin = find_bin(need, before, sh);
  // The logits of that bin (one counter: a wavefront's in one step) and their keys'
  // range.
  uint32_t low = 0xffffffffu, high = 0;
  row.each([&](int i, float x, uint64_t w) {
    if (!bin_of.in(x, static_cast<float>(bin))) return;
    const uint32_t key = order_key(x);
    low = min(low, key);
    high = max(high, key);
    const uint64_t who = __ballot(1);
    const int lane = threadIdx.x & (kWave - 1);
    int at = 0;
    if (lane == __builtin_ctzll(who)) at = atomicAdd(&sh.count, __popcll(who));
    at = __shfl(at, __builtin_ctzll(who)) + __popcll(who & ((uint64_t{1} << lane) - 1));
    if (at < kList) sh.list[at] = {f(i, x, w), key, i};
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= kList) {
    order_list(n, sh);
    if (static_cast<int>(threadIdx.x) < n) {
      const Entry mine = sh.list[threadIdx.x];
      const uint64_t at = before + sh.ahead[threadIdx.x];
      if (at < need && need <= at + mine.f) {
        sh.edge = key_value(static_cast<uint64_t>(mine.key) << 32);
        sh.until = mine.index;
      }
    }
    __syncthreads();
    return {sh.edge, sh.until};
  }
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    low = min(low, static_cast<uint32_t>(__shfl_xor(static_cast<int>(low), d)));
    high = max(high, static_cast<uint32_t>(__shfl_xor(static_cast<int>(high), d)));
  }
  if ((threadIdx.x & (kWave - 1)) == 0) {
    sh.low[threadIdx.x >> 6] = low;
    sh.high[threadIdx.x >> 6] = high;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    low = min(low, sh.low[w]);
    high = max(high, sh.high[w]);
  }
  while (low < high) {
    int bits = 0;  // (high - low) >> bits < kBins - 1
    while (((high - low) >> bits) >= kBins - 1) ++bits;
    clear_bins(sh);
    row.each([&](int i, float x, uint64_t w) {
      const uint32_t key = order_key(x);
      if (key >= low && key <= high) add_to_bin((high - key) >> bits, f(i, x, w), sh);
    });
    __syncthreads();
    uint64_t within;
    const uint32_t b = find_bin(need - before, within, sh);
    before += within;
    high -= b << bits;
    low = max(low, high - ((1u << bits) - 1));
  }
  auto equal = [&](int i, float x, uint64_t w) -> uint64_t {
    return order_key(x) == low ? f(i, x, w) : 0;
  };
  total(row, equal, sh);
  return {key_value(static_cast<uint64_t>(low) << 32), row.locate(equal, need - before - 1, sh)};
}

template <int TYPE, int STEPS>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  constexpr bool HELD = STEPS > 0;
  __shared__ __attribute__((aligned(16))) float held[HELD ? STEPS * kWaves * kStep : 4];
  __shared__ Shared sh;
  const int r = blockIdx.x, t = threadIdx.x;
  Row<TYPE, STEPS> row;
  constexpr int kBytes = TYPE == kLogitF32 ? 4 : 2;
  row.at = static_cast<const char*>(a.logits) + r * a.stride * kBytes;
  row.held = held;
  row.n = a.vocab;
  row.steps = HELD && STEPS < kMost ? STEPS : (a.vocab + kWaves * kStep - 1) / (kWaves * kStep);
  row.aligned = (reinterpret_cast<uintptr_t>(row.at) & (4 * kBytes - 1)) == 0 && row.n % 4 == 0;
  row.infinite = false;
  // (NaN: as 0; infinity: every logit but -infinity weighs 1)
  const double temperature = a.temperature ? a.temperature[r] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_all;
  const double top_p = a.top_p ? a.top_p[r] : a.top_p_all;  // (NaN: as 1)
  // (the largest always stays; NaN: as 0)
  const double min_p = fmin(fmax(a.min_p ? a.min_p[r] : a.min_p_all, 0.0), 1.0);
  if (t < kTable) sh.table[t] = kPowers.at[t];

  // This thread's and the row's largest logit.
  float mine = -INFINITY;
  {
    constexpr int kAhead = HELD ? STEPS : kMost;  // loads in flight
    for (int from = 0; from < row.steps; from += kAhead) {
      float4 v[kAhead];
      if (row.aligned) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
          v[s] = logits4<TYPE>(row.at, from + s < row.steps ? row.first(from + s) : row.n, row.n,
                               true);
      } else {
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
          v[s] = logits4<TYPE>(row.at, from + s < row.steps ? row.first(from + s) : row.n, row.n,
                               false);
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (HELD && s < row.steps) *reinterpret_cast<float4*>(&held[row.first(s)]) = v[s];
        mine = fmaxf(fmaxf(mine, fmaxf(v[s].x, v[s].y)), fmaxf(v[s].z, v[s].w));
      }
    }
  }
  float top = mine;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if ((t & (kWave - 1)) == 0) sh.low[t >> 6] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, __uint_as_float(sh.low[w]));
  auto answer = [&](int token, double share) {
    if (t == 0) {
      a.token[r] = token;
      if (a.probability) a.probability[r] = static_cast<float>(share);
    }
  };
  if (top == -INFINITY) return answer(-1, 0.0);  // nothing to draw from
  if (!(temperature > 0.0) || top_k == 1) {  // the first of the largest
    auto largest = [&](int, float x, uint64_t) -> uint64_t { return x == top; };
    total(row, largest, sh);
    return answer(row.locate(largest, 0, sh), 1.0);
  }

  if (top == INFINITY) {
    row.infinite = true;
    if constexpr (HELD) {
      __syncthreads();
      for (int s = 0; s < row.steps; ++s) {
        float4* const v = reinterpret_cast<float4*>(&held[row.first(s)]);
        *v = finite_of(*v);
      }
      __syncthreads();
    }
    mine = mine == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
  }

  // w 2^shift: w = 2^(k / 256) e^r with k = round(256 log2 w), |r| <= ln 2 / 512, and
  // e^r - 1 <= 0.00136 to the third power in 32 bits: w is right to 1e-10.
  // (below 2e-306 the quotient would be infinite and the largest's own weight, by 0 times
  // it, nothing; at 1e-300 the nearest two logits, 2^-149 apart, already differ by a weight
  // that rounds to 0)
  const double per_unit = kTable * 1.4426950408889634074 / fmax(temperature, 1e-300);
  const double origin = top;
  const double lowest = -kTable * (a.shift + 2);  // rounds to 0
  auto weight = [&](float x, int scale) -> double {  // w 2^scale
    const double z = fmax((static_cast<double>(x) - origin) * per_unit, lowest);
    const double whole = rint(z);
    const int k = static_cast<int>(whole);
    const float r = static_cast<float>(z - whole) * (0.693147180559945309f / kTable);
    const float more = __builtin_fmaf(__builtin_fmaf(r, 1.0f / 6.0f, 0.5f) * r, r, r);
    const double at = sh.table[k & (kTable - 1)];
    return ldexp(fma(at, static_cast<double>(more), at), (k >> kTableBits) + scale);
  };
  // (rounded to a whole number where 2^52 is added to it)
  auto mass = [&](float x) -> uint64_t {
    return __builtin_bit_cast(uint64_t, weight(x, a.shift) + 0x1p52) - (uint64_t{1075} << 52);
  };
  // The bins reach as far as weights do (2^-46 at 32 T), but no further than 32.
  const Bins bins{top, (kBins - 1) / static_cast<float>(
                                         fmax(fmin(32.0 * temperature, 32.0), 1e-30))};
  const uint64_t least_mass = static_cast<uint64_t>(ldexp(min_p, a.shift));
  auto needed = [&](uint64_t all) -> uint64_t {  // of the mass, for top_p
    const uint64_t x = static_cast<uint64_t>(ceil(fmax(top_p, 0.0) * static_cast<double>(all)));
    return x < 1 ? 1 : x > all ? all : x;
  };
  auto drawn = [&](uint64_t all) -> uint64_t {
    // (u below 1: the product is below the sum but for its rounding; NaN: as 0)
    const double u = fmax(static_cast<double>(a.uniform[r]), 0.0) * static_cast<double>(all);
    const uint64_t x = u < static_cast<double>(all) ? static_cast<uint64_t>(u) : all - 1;
    return x < all ? x : all - 1;
  };
  auto share = [&](float x, uint64_t all) -> double {
    return weight(x, a.shift) / static_cast<double>(all);
  };
  auto one = [](int, float, uint64_t) -> uint64_t { return 1; };
  auto held_weight = [](int, float, uint64_t w) -> uint64_t { return w; };
  const bool by_count = top_k > 0 && top_k < row.n;

  // A list that holds the top_k: what lies in the bins of the k largest of the
  // threads' maxima.  Or the whole of a short row.
  int few = row.n <= kThreads ? row.n : 0;
  if (few == 0 && by_count && top_k <= kShort) {
    clear_bins(sh);
    const int b = bins(mine);
    if (b < kBins - 1) add_to_bin(b, 1, sh);
    __syncthreads();
    uint64_t before;
    const int last = find_bin(top_k, before, sh);
    if (last < kBins - 1) {
      // One bin further down, so that no rounding here leaves one of them out (the
      // count says whether it did).
      const float from = top - static_cast<float>(last + 2) / bins.per_unit;
      const int wave = t >> 6, lane = t & (kWave - 1);
      int n = 0;
      for (int s = 0; s < row.steps; ++s) {
        const float4 v = row.get(s);
        n += (v.x >= from) + (v.y >= from) + (v.z >= from) + (v.w >= from);
      }
      n = static_cast<int>(wave_total(n));
      if (lane == 0) sh.low[wave] = n;
      __syncthreads();
      int at = 0;  // where this wavefront's begin
      n = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) at += sh.low[w];
        n += sh.low[w];
      }
      if (n >= top_k && n <= kThreads) {
        const uint64_t below = (uint64_t{1} << lane) - 1;
        for (int s = 0; s < row.steps; ++s) {
          const int i = row.first(s);
          const float4 v = row.get(s);
          const float x[4] = {v.x, v.y, v.z, v.w};
          // (of most steps none)
          if (__ballot(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= from) == 0) continue;
          uint64_t who[4];
          int to = at;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            who[j] = __ballot(x[j] >= from);
            to += __popcll(who[j] & below);
            at += __popcll(who[j]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (x[j] >= from) {
              sh.few[to] = x[j];
              sh.few_index[to++] = i + j;
            }
          }
        }
        few = n;
      }
    }
    __syncthreads();
  } else if (few > 0) {
    row.each([&](int i, float x, uint64_t) {
      sh.few[i] = x;
      sh.few_index[i] = i;
    });
    __syncthreads();
  }
  if (few > 0) {
    Few list{few, t < few ? sh.few[t] : -INFINITY, 0};
    if (t < few) list.w = mass(list.x);
    if (few <= kPairs) {
      // (all that come before a logit that top_k keeps are kept by it)
      if (t < few) sh.list[t] = {list.w, order_key(list.x), t};
      __syncthreads();
      order_list(few, sh);
      // The rest by one wavefront, two logits a lane, without a barrier.
      if (t >= kWave) return;
      static_assert(kPairs == 2 * kWave, "two a lane");
      uint64_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = t + kWave * h;
        w[h] = e < few && !(by_count && sh.rank[e] >= top_k) ? sh.list[e].f : 0;
      }
      if (top_p < 1.0) {
        const uint64_t need = needed(wave_total(w[0] + w[1]));
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = sh.ahead[t + kWave * h] >= need ? 0 : w[h];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) w[h] = w[h] < least_mass ? 0 : w[h];
      const uint64_t first = wave_upto(w[0]), second = last_lane(first) + wave_upto(w[1]);
      const uint64_t all = last_lane(second), target = drawn(all);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t upto = h ? second : first;
        if (upto - w[h] <= target && target < upto) {
          const int e = t + kWave * h;
          a.token[r] = sh.few_index[e];
          if (a.probability) a.probability[r] = static_cast<float>(share(sh.few[e], all));
        }
      }
      return;
    }
    auto cut = [&](Edge edge) {
      if (!edge.keeps(t, list.x)) list.w = 0;
    };
    if (by_count && top_k < few) cut(select(list, one, top_k, bins, false, sh));
    if (top_p < 1.0)
      cut(select(list, held_weight, needed(total(list, held_weight, sh)), bins, false, sh));
    if (list.w < least_mass) list.w = 0;
    const uint64_t all = total(list, held_weight, sh);
    const int at = list.locate(held_weight, drawn(all), sh);
    return answer(sh.few_index[at], share(sh.few[at], all));
  }

  Edge edge{-INFINITY, row.n};
  if (by_count) edge = select(row, one, top_k, bins, false, sh);
  auto f = [&](int i, float x, uint64_t) -> uint64_t {
    const uint64_t w = mass(x);
    return edge.keeps(i, x) ? w : 0;
  };
  if constexpr (HELD) {
    // Every weight once, in registers.
    Weights<Row<TYPE, STEPS>, STEPS> all_of{row, {}};
    if (top_p < 1.0) clear_bins(sh);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s < row.steps) {
        const int i = row.first(s);
        const float4 v = row.get(s);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t w = f(i + j, x[j], 0);
          all_of.w[s][j] = w;
          if (top_p < 1.0) {
            const float d = bins.distance(x[j]);
            if (d < static_cast<float>(kBins - 1)) add_to_bin(static_cast<int>(d), w, sh);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (top_p < 1.0) {
      const uint64_t need = needed(all_of.sum(sh));
      __syncthreads();
      edge = select(all_of, held_weight, need, bins, true, sh);
    }
    if (top_p < 1.0 || least_mass > 0)
      all_of.keep([&](int i, float x, uint64_t w) { return (w >= least_mass) & edge.keeps(i, x); });
    const uint64_t all = all_of.sum(sh);
    const int token = all_of.locate(drawn(all), sh);
    return answer(token, share(held[token], all));
  } else {
    if (top_p < 1.0) edge = select(row, f, needed(total(row, f, sh)), bins, false, sh);
    auto last = [&](int i, float x, uint64_t) -> uint64_t {
      const uint64_t w = f(i, x, 0);
      return w < least_mass ? 0 : w;
    };
    const uint64_t all = total(row, last, sh);
    const int token = row.locate(last, drawn(all), sh);
    const float x = logit<TYPE>(row.at, token);
    return answer(token, share(row.infinite ? 0.0f : x, all));
  }
}

// (a step's 4096 logits are passed whole, so the fewest that hold the row)
template <int TYPE>
void launch(const SampleArgs& a, int rows, hipStream_t s) {
  constexpr int kOne = kWaves * kStep;
  if (a.vocab <= kOne) sample_kernel<TYPE, 1><<<rows, kThreads, 0, s>>>(a);
  else if (a.vocab <= 2 * kOne) sample_kernel<TYPE, 2><<<rows, kThreads, 0, s>>>(a);
  else if (a.vocab <= 4 * kOne) sample_kernel<TYPE, 4><<<rows, kThreads, 0, s>>>(a);
  else if (a.vocab <= kMost * kOne) sample_kernel<TYPE, kMost><<<rows, kThreads, 0, s>>>(a);
  else sample_kernel<TYPE, 0><<<rows, kThreads, 0, s>>>(a);
}

}  // namespace

hipError_t launch_sample(const void* logits, int type, int rows, int vocab, int64_t stride,
                         const float* uniform, const float* temperature, double temperature_all,
                         const int32_t* top_k, int32_t top_k_all, const float* top_p,
                         double top_p_all, const float* min_p, double min_p_all, int64_t* token,
                         float* probability, hipStream_t s) {
  if (rows == 0) return hipSuccess;
  SampleArgs a{logits, stride, vocab, uniform, temperature, top_k, top_p, min_p,
               temperature_all, top_p_all, min_p_all, top_k_all, 0, token, probability};
  int bits = 0;
  while ((int64_t{1} << bits) < vocab) ++bits;
  a.shift = bits > 12 ? 62 - bits : 50;  // (a row's sum fits 63 bits, a weight 52)
  if (type == kLogitF32) launch<kLogitF32>(a, rows, s);
  else if (type == kLogitBf16) launch<kLogitBf16>(a, rows, s);
  else launch<kLogitF16>(a, rows, s);
  return hipGetLastError();
}

}  // namespace parrot
