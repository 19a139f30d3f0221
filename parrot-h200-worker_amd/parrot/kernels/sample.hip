// Drawing a token per row of logits, with temperature, top-k, top-p and min-p,
// from one given uniform number u:
//   w_i = exp((x_i - max x) / T);
//   the top_k largest (equal ones by their index), of those the shortest
//   prefix that holds top_p of their mass, of those w_i >= min_p;
//   the first token, by index, at which the sum of w passes u times the whole.
//
// Weights are 64-bit whole numbers (w 2^s, rounded; s so that a row's sum fits):
// their sums do not depend on an order, so a row's token does not depend on how
// the work is split, and a border between two tokens lies where it does in 64-bit
// arithmetic up to the rounding of single weights (2^-47 at 32768 tokens).
#include <math.h>

#include "common.h"

namespace parrot {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;

enum LogitType { kLogitF32 = 0, kLogitBf16 = 1, kLogitF16 = 2 };

// exp(x) for x <= 0: 2^(k / 32) e^r with k = round(32 x / ln 2), r = x - k ln 2 /
// 32, |r| <= 0.0109, whose series to the fifth power is right to 2e-15.
__device__ __forceinline__ double exp_neg(double x) {
  if (!(x > -700.0)) return 0.0;
  const double k = rint(x * (32.0 / 0.69314718055994530942));
  double r = fma(k, -(0.69314718055994530942 / 32.0), x);
  r = fma(k, -(2.3190468138462996e-17 / 32.0), r);
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int n = static_cast<int>(k);
  return ldexp(p * exp2((n & 31) * (1.0 / 32.0)), n >> 5);
}

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
  return x == x ? x : -INFINITY;  // a NaN is never drawn
}

struct Block {
  uint64_t wave[kWaves];
  uint64_t found[2];
};

__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(static_cast<unsigned long long>(v), d);
  return v;
}

__device__ __forceinline__ uint64_t block_total(uint64_t v, Block& b) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) b.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) t += b.wave[i];
  return t;
}

// The sum of f(i) over the row.
template <typename F>
__device__ uint64_t total(int n, F f, Block& b) {
  uint64_t t = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) t += f(i);
  return block_total(t, b);
}

// The first index at which the sum of f up to it passes `target`, and the last
// index where none does.
template <typename F>
__device__ int locate(int n, F f, uint64_t target, Block& b) {
  uint64_t before = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + threadIdx.x;
    const uint64_t mine = i < n ? f(i) : 0;
    const uint64_t all = block_total(mine, b);
    if (before + all > target) {
      uint64_t upto = mine;
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) {
        const uint64_t x = __shfl_up(static_cast<unsigned long long>(upto), d);
        if (static_cast<int>(threadIdx.x & (kWave - 1)) >= d) upto += x;
      }
      for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) upto += b.wave[w];
      upto += before;
      if (upto > target && upto - mine <= target) b.found[0] = i;
      __syncthreads();
      return static_cast<int>(b.found[0]);
    }
    before += all;
  }
  return n - 1;
}

// The largest key t with sum of f over keys >= t of at least `need` (> 0, and at
// most the whole).
template <typename K, typename F>
__device__ uint32_t select(int n, K key, F f, uint64_t need, Block& b) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t next = t | (1u << bit);
    if (total(n, [&](int i) { return key(i) >= next ? f(i) : 0; }, b) >= need) t = next;
  }
  return t;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Block b;
  const int row = blockIdx.x, n = a.vocab;
  const void* const x = static_cast<const char*>(a.logits) +
                        row * a.stride * (TYPE == kLogitF32 ? 4 : 2);
  const double t = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const double top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const double min_p = fmin(a.min_p ? a.min_p[row] : a.min_p_all, 1.0);  // the first stays
  auto key = [&](int i) { return order_key(logit<TYPE>(x, i)); };
  const uint64_t one = 1;

  const uint32_t best = select(n, key, [&](int) { return one; }, 1, b);
  const float largest = key_value(static_cast<uint64_t>(best) << 32);
  if (largest == -INFINITY) {  // nothing to draw from
    if (threadIdx.x == 0) {
      a.token[row] = -1;
      if (a.probability) a.probability[row] = 0.0f;
    }
    return;
  }
  auto weight = [&](int i) -> double {
    const float v = logit<TYPE>(x, i);
    return v == largest ? 1.0 : exp_neg((static_cast<double>(v) - largest) / t);
  };
  auto mass = [&](int i) -> uint64_t {
    return static_cast<uint64_t>(rint(ldexp(weight(i), a.shift)));
  };
  // Kept: keys above `least`, and those equal to it up to index `until`.
  uint32_t least = 0;
  int until = n - 1;
  auto kept = [&](int i) {
    const uint32_t k = key(i);
    return k > least || (k == least && i <= until);
  };
  const bool greedy = !(t > 0.0);
  const int k = greedy ? 1 : top_k;
  if (k > 0 && k < n) {
    least = select(n, key, [&](int) { return one; }, k, b);
    const uint64_t above = total(n, [&](int i) -> uint64_t { return key(i) > least; }, b);
    until = locate(n, [&](int i) -> uint64_t { return key(i) == least; }, k - above - 1, b);
  }
  if (!greedy && top_p < 1.0) {
    auto f = [&](int i) -> uint64_t { return kept(i) ? mass(i) : 0; };
    const uint64_t all = total(n, f, b);
    uint64_t need = static_cast<uint64_t>(ceil(fmax(top_p, 0.0) * static_cast<double>(all)));
    need = need < 1 ? 1 : need > all ? all : need;
    const uint32_t edge = select(n, key, f, need, b);
    uint64_t above = total(n, [&](int i) -> uint64_t { return key(i) > edge ? f(i) : 0; }, b);
    const int last = locate(n, [&](int i) -> uint64_t { return key(i) == edge ? f(i) : 0; },
                            need - above - 1, b);
    least = edge;
    until = last;
  }
  auto f = [&](int i) -> uint64_t { return kept(i) && weight(i) >= min_p ? mass(i) : 0; };
  const uint64_t all = greedy ? 1 : total(n, f, b);
  int token;
  if (greedy) {
    token = until;
  } else {
    double u = static_cast<double>(a.uniform[row]) * static_cast<double>(all);
    u = u > 0.0 ? u : 0.0;
    uint64_t target = u < static_cast<double>(all) ? static_cast<uint64_t>(u) : all - 1;
    target = target < all ? target : all - 1;
    token = locate(n, f, target, b);
  }
  if (threadIdx.x == 0) {
    a.token[row] = token;
    if (a.probability)
      a.probability[row] = greedy ? 1.0f
                                  : static_cast<float>(ldexp(weight(token), a.shift) /
                                                       static_cast<double>(all));
  }
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
  a.shift = 62 - bits;
  if (type == kLogitF32) sample_kernel<kLogitF32><<<rows, kThreads, 0, s>>>(a);
  else if (type == kLogitBf16) sample_kernel<kLogitBf16><<<rows, kThreads, 0, s>>>(a);
  else sample_kernel<kLogitF16><<<rows, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace parrot
