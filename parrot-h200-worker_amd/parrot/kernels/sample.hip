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
// up to the rounding of single weights (2^-47 of the largest at 32768 tokens).
//
// A workgroup per row, which keeps the row in LDS (32768 logits; longer rows are
// read again, from L2, in each pass).  Nothing is sorted: the border of top-k or
// top-p is found by one histogram over the distance from the largest logit, its
// bins as wide as to spread the row, in whole numbers (counts or weights), and
// the order of the few logits in the border's bin by comparing each with each.
// A bin with too many of them (equal logits, tiny temperatures) is split by its
// range of bit patterns, 2048 parts at a time.
#include <math.h>

#include "common.h"

namespace parrot {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kStep = 4 * kWave;   // logits of a wavefront's step, four a lane
constexpr int kHeld = 32768;       // logits of a row that LDS holds
constexpr int kBins = 2048;
constexpr int kList = 256;         // logits compared each with each
constexpr int kTable = 256;

enum LogitType { kLogitF32 = 0, kLogitBf16 = 1, kLogitF16 = 2 };

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

// Four logits from i on; a NaN, and what lies past the row, is -infinity.
template <int TYPE>
__device__ __forceinline__ float4 logits4(const void* row, int i, int n, bool aligned) {
  float x[4];
  if (aligned && i + 3 < n) {
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
  for (int j = 0; j < 4; ++j) x[j] = x[j] == x[j] ? x[j] : -INFINITY;
  return make_float4(x[0], x[1], x[2], x[3]);
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
  uint64_t wave[kWaves];
  uint64_t before;
  uint32_t low[kWaves], high[kWaves];
  int found;
  int count;
  uint32_t edge;
  int until;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return __shfl_up(static_cast<unsigned long long>(v), d);
}

__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(static_cast<unsigned long long>(v), d);
  return v;
}

__device__ __forceinline__ uint64_t wave_upto(uint64_t v) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint64_t x = shfl_up64(v, d);
    if (lane >= d) v += x;
  }
  return v;
}

// A row: `steps` times 256 consecutive logits per wavefront, so that sums over
// wavefronts, steps, lanes and a lane's four are sums by index.
template <int TYPE, bool HELD>
struct Row {
  const void* at;
  const float* held;
  int n, steps;
  bool aligned;
  __device__ __forceinline__ int first(int step) const {
    return (static_cast<int>(threadIdx.x >> 6) * steps + step) * kStep +
           4 * static_cast<int>(threadIdx.x & (kWave - 1));
  }
  __device__ __forceinline__ float4 get(int step) const {
    const int i = first(step);
    if constexpr (HELD) return *reinterpret_cast<const float4*>(held + i);
    return logits4<TYPE>(at, i, n, aligned);
  }
  // f(index, logit) for this thread's logits
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int s = 0; s < steps; ++s) {
      const int i = first(s);
      if (i >= n) break;
      const float4 v = get(s);
      f(i, v.x);
      if (i + 1 < n) f(i + 1, v.y);
      if (i + 2 < n) f(i + 2, v.z);
      if (i + 3 < n) f(i + 3, v.w);
    }
  }
};

// The sum of f over the row; leaves each wavefront's share in sh.wave.
template <typename R, typename F>
__device__ uint64_t total(const R& row, F f, Shared& sh) {
  uint64_t t = 0;
  row.each([&](int i, float x) { t += f(i, x); });
  t = wave_total(t);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sh.wave[threadIdx.x >> 6] = t;
  __syncthreads();
  t = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) t += sh.wave[i];
  return t;
}

// The first index at which the sum of f passes `target` (below the whole); f's
// shares as total() left them.
template <typename R, typename F>
__device__ int locate(const R& row, F f, uint64_t target, Shared& sh) {
  const int wave = threadIdx.x >> 6;
  uint64_t before = 0;
  for (int w = 0; w < wave; ++w) before += sh.wave[w];
  if (before <= target && target < before + sh.wave[wave]) {  // one wavefront
    for (int s = 0; s < row.steps; ++s) {
      const int i = row.first(s);
      const float4 v = row.get(s);
      const uint64_t f0 = i < row.n ? f(i, v.x) : 0, f1 = i + 1 < row.n ? f(i + 1, v.y) : 0;
      const uint64_t f2 = i + 2 < row.n ? f(i + 2, v.z) : 0;
      const uint64_t f3 = i + 3 < row.n ? f(i + 3, v.w) : 0;
      const uint64_t mine = f0 + f1 + f2 + f3;
      const uint64_t upto = wave_upto(mine);
      const uint64_t all = __shfl(static_cast<unsigned long long>(upto), kWave - 1);
      if (target < before + all) {
        uint64_t at = before + upto - mine;
        if (at <= target && target < at + mine) {
          int j = i;
          if (target >= at + f0) ++j, at += f0;
          if (j == i + 1 && target >= at + f1) ++j, at += f1;
          if (j == i + 2 && target >= at + f2) ++j;
          sh.found = j;
        }
        break;
      }
      before += all;
    }
  }
  __syncthreads();
  return sh.found;
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
  uint32_t key;
  int until;
};

// The last logit, in the order of size and index, that is needed for the sum of f
// to reach `need` (1 .. the whole): its key and index.  per: bins per unit of
// distance from `top`, the largest logit.
template <typename R, typename F>
__device__ Edge select(const R& row, F f, uint64_t need, float top, float per, Shared& sh) {
  auto bin_of = [&](float x) {
    const float d = x == top ? 0.0f : (top - x) * per;
    return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
  };
  auto clear = [&] {
    __syncthreads();
    sh.bins[threadIdx.x] = sh.bins[threadIdx.x + kThreads] = 0;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
  };
  auto add = [&](int bin, uint64_t v) {
    if (v) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[bin]), v);
  };
  clear();
  row.each([&](int i, float x) {
    const int b = bin_of(x);
    if (b < kBins - 1) add(b, f(i, x));
  });
  __syncthreads();
  uint64_t before;
  const int bin = find_bin(need, before, sh);
  // The logits of that bin (one counter: a wavefront's in one step) and their keys'
  // range.
  uint32_t low = 0xffffffffu, high = 0;
  row.each([&](int i, float x) {
    if (bin_of(x) != bin) return;
    const uint32_t key = order_key(x);
    low = min(low, key);
    high = max(high, key);
    const uint64_t who = __ballot(1);
    const int lane = threadIdx.x & (kWave - 1);
    int at = 0;
    if (lane == __builtin_ctzll(who)) at = atomicAdd(&sh.count, __popcll(who));
    at = __shfl(at, __builtin_ctzll(who)) + __popcll(who & ((uint64_t{1} << lane) - 1));
    if (at < kList) sh.list[at] = {f(i, x), key, i};
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= kList) {
    if (static_cast<int>(threadIdx.x) < n) {
      const Entry mine = sh.list[threadIdx.x];
      uint64_t at = before;
      for (int j = 0; j < n; ++j) {
        const Entry e = sh.list[j];
        if (e.key > mine.key || (e.key == mine.key && e.index < mine.index)) at += e.f;
      }
      if (at < need && need <= at + mine.f) {
        sh.edge = mine.key;
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
    clear();
    row.each([&](int i, float x) {
      const uint32_t key = order_key(x);
      if (key >= low && key <= high) add((high - key) >> bits, f(i, x));
    });
    __syncthreads();
    uint64_t within;
    const uint32_t b = find_bin(need - before, within, sh);
    before += within;
    high -= b << bits;
    low = max(low, high - ((1u << bits) - 1));
  }
  auto equal = [&](int i, float x) -> uint64_t { return order_key(x) == low ? f(i, x) : 0; };
  total(row, equal, sh);
  return {low, locate(row, equal, need - before - 1, sh)};
}

template <int TYPE, bool HELD>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) float held[HELD ? kHeld : 4];
  __shared__ Shared sh;
  const int r = blockIdx.x, t = threadIdx.x;
  Row<TYPE, HELD> row;
  constexpr int kBytes = TYPE == kLogitF32 ? 4 : 2;
  row.at = static_cast<const char*>(a.logits) + r * a.stride * kBytes;
  row.held = held;
  row.n = a.vocab;
  row.steps = (a.vocab + kWaves * kStep - 1) / (kWaves * kStep);
  row.aligned = (reinterpret_cast<uintptr_t>(row.at) & (4 * kBytes - 1)) == 0;
  const double temperature = a.temperature ? a.temperature[r] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_all;
  const double top_p = a.top_p ? a.top_p[r] : a.top_p_all;
  // (the largest always stays)
  const double min_p = fmin(a.min_p ? a.min_p[r] : a.min_p_all, 1.0);
  if (t < kTable) sh.table[t] = exp2(t * (1.0 / kTable));

  // The largest logit (the lowest index among equal ones), the smallest finite one.
  uint64_t best = 0;
  float least = INFINITY;
  for (int s = 0; s < row.steps; ++s) {
    const int i = row.first(s);
    if (i >= row.n && !HELD) break;
    const float4 v = logits4<TYPE>(row.at, i, row.n, row.aligned);
    if constexpr (HELD) *reinterpret_cast<float4*>(&held[i]) = v;
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t key = expert_key(x[j], i + j);
      best = key > best ? key : best;
      least = x[j] > -INFINITY ? fminf(least, x[j]) : least;
    }
  }
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint64_t key = __shfl_xor(static_cast<unsigned long long>(best), d);
    best = key > best ? key : best;
    least = fminf(least, __shfl_xor(least, d));
  }
  if ((t & (kWave - 1)) == 0) {
    sh.wave[t >> 6] = best;
    sh.low[t >> 6] = __float_as_uint(least);
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    best = sh.wave[w] > best ? sh.wave[w] : best;
    least = fminf(least, __uint_as_float(sh.low[w]));
  }
  const float top = key_value(best);
  const bool greedy = !(temperature > 0.0) || top_k == 1;
  if (top == -INFINITY || greedy) {  // nothing to draw from; nothing to choose
    if (t == 0) {
      a.token[r] = top == -INFINITY ? -1 : key_expert(best);
      if (a.probability) a.probability[r] = top == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }

  // log2 w, and w 2^shift: 2^y = 2^(k / 256) e^r with k = round(256 y), r = (256 y -
  // k) ln 2 / 256, |r| <= 0.00136, whose series to the third power is right to 2e-13.
  const double per_unit = 1.4426950408889634074 / temperature;
  auto power = [&](float x) -> double {
    return x == top ? 0.0 : x == -INFINITY ? -INFINITY : (static_cast<double>(x) - top) * per_unit;
  };
  auto scaled = [&](double y, int& k) -> double {  // 2^(y - floor(k / 256))
    const double z = y * kTable, whole = rint(z);
    k = static_cast<int>(whole);
    const double e = (z - whole) * (0.69314718055994530942 / kTable);
    return sh.table[k & (kTable - 1)] * fma(fma(fma(e, 1.0 / 6.0, 0.5), e, 1.0), e, 1.0);
  };
  auto mass = [&](double y) -> uint64_t {
    if (!(y > -(a.shift + 2))) return 0;
    int k;
    const uint64_t u = __builtin_bit_cast(uint64_t, scaled(y, k));
    const int down = 52 - a.shift - (static_cast<int>(u >> 52) - 1023 + (k >> 8));  // 2 .. 56
    return (((u & ((uint64_t{1} << 52) - 1)) | (uint64_t{1} << 52)) + (uint64_t{1} << (down - 1))) >>
           down;
  };
  // Bins: over the whole row, or the distance from which on weights round to 0 (32
  // T: the last ones are not counted but known to be there).
  const float range = fminf(static_cast<float>(fmin(32.0 * temperature, 1e30)), top - least);
  const float per = range > 0.0f && top < INFINITY ? (kBins - 1.5f) / range : 0.0f;

  Edge edge{0, a.vocab};
  auto kept = [&](int i, float x) {
    const uint32_t k = order_key(x);
    return k > edge.key || (k == edge.key && i <= edge.until);
  };
  if (top_k > 0 && top_k < a.vocab)
    edge = select(row, [&](int, float) { return uint64_t{1}; }, top_k, top, per, sh);
  if (top_p < 1.0) {
    auto f = [&](int i, float x) -> uint64_t { return kept(i, x) ? mass(power(x)) : 0; };
    const uint64_t all = total(row, f, sh);
    uint64_t need = static_cast<uint64_t>(ceil(fmax(top_p, 0.0) * static_cast<double>(all)));
    need = need < 1 ? 1 : need > all ? all : need;
    edge = select(row, f, need, top, per, sh);
  }
  const double floor_p = min_p > 0.0 ? log2(min_p) : -INFINITY;
  auto f = [&](int i, float x) -> uint64_t {
    if (!kept(i, x)) return 0;
    const double y = power(x);
    return y >= floor_p ? mass(y) : 0;
  };
  const uint64_t all = total(row, f, sh);
  // (u below 1: the product is below the sum but for its rounding)
  const double u = fmax(static_cast<double>(a.uniform[r]), 0.0) * static_cast<double>(all);
  const uint64_t target = u < static_cast<double>(all) ? static_cast<uint64_t>(u) : all - 1;
  const int token = locate(row, f, target < all ? target : all - 1, sh);
  if (t == 0) {
    a.token[r] = token;
    if (a.probability) {
      float x = logit<TYPE>(row.at, token);
      int k;
      const double w = scaled(power(x), k);
      a.probability[r] =
          static_cast<float>(ldexp(w, (k >> 8) + a.shift) / static_cast<double>(all));
    }
  }
}

template <int TYPE>
void launch(const SampleArgs& a, int rows, hipStream_t s) {
  if (a.vocab <= kHeld) sample_kernel<TYPE, true><<<rows, kThreads, 0, s>>>(a);
  else sample_kernel<TYPE, false><<<rows, kThreads, 0, s>>>(a);
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
  a.shift = bits > 12 ? 62 - bits : 50;  // (a row's sum fits 63 bits)
  if (type == kLogitF32) launch<kLogitF32>(a, rows, s);
  else if (type == kLogitBf16) launch<kLogitBf16>(a, rows, s);
  else launch<kLogitF16>(a, rows, s);
  return hipGetLastError();
}

}  // namespace parrot
