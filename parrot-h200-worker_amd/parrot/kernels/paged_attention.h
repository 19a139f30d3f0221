// Attention of a chunk of new tokens (one, or thousands) over the pages of a
// KV cache: key j is visible to the query at position i iff j <= i and
// (j > i - window or j < sinks).
//
// The rows of a tile are (token, query head) pairs of one kv head, token-major:
// a decode step's query heads that share a kv head are rows of one tile, so its
// keys and values are read once for all of them.
//
//   S^T = K Q^T     A = 32 keys, B = 32 rows: lane l holds 16 of the block's
//                   keys for row l % 32 (v_mfma_f32_32x32x16_bf16).
//   O^T += V^T P^T  P^T comes straight from those registers as the B operand:
//                   operand row i of K is key 16 j + 4 (2 s + h) + r of the block
//                   (i = 16 s + 8 j + 4 h + r), so that the 8 scores a lane holds
//                   per 16-key step are the keys {4 g .. + 3, 16 + 4 g .. + 3},
//                   g = 2 s + l / 32, of one piece of V.
//
// (and the same on v_mfma_f32_16x16x32_bf16 for tiles of 16 rows).
//
// 8-bit rows enter the products unrounded: K as q 2^x (exact in bf16; int8: 2^(x - 2)), V as q
// with its power of two on the probability instead (one power per key, and a
// piece of V holds eight keys).  P is rounded to bf16 once, which the matrix
// instructions ask for: half a step of 2^-8 on each probability, 1.9 to 2.3e-3 of the output
// beside its own rounding's 1.6e-3 (in two parts, with twice the products: 1.6e-3, decode
// steps 2 to 3 % slower).  Everything else is summed in 32 bits.
#pragma once

#include <type_traits>

#include "paged.h"

namespace parrot {
namespace paged {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

static_assert(kMaxSplits == kWave, "a share a lane");

struct AttendArgs {
  PagedCache cache;
  PagedBatch batch;
  const uint16_t* q;
  int64_t qs[2];  // element strides: row, head
  int heads, rep;
  int window;  // INT_MAX: none
  int sinks;
  float scale_log2;  // |scale| log2(e), times kUnit
  uint32_t q_sign;   // 0x80008000 for a negative scale (q is negated), else 0
  int splits, whole;
  float* part;       // [rows * heads][splits][D], unnormalised
  float2* part_ml;   // [rows * heads][splits]
  uint16_t* out;     // [rows][heads][D]
};

// Which block of the cache (whose number fits 32 bits) a sequence's is, -1 where the table
// names no page.
__device__ __forceinline__ int cache_block(const AttendArgs& a, int sequence, int kvh, int block) {
  const int per_page = a.cache.page / kPagedBlock, at = block / per_page;
  const int page = paged_page(a.batch, a.cache, sequence, at);
  return page < 0 ? -1 : (page * a.cache.kv_heads + kvh) * per_page + block - at * per_page;
}

// Where a wavefront's key blocks (every fourth of its workgroup's share) lie among the
// cache's: lane j holds the j-th of the last 64.
struct WaveBlocks {
  const AttendArgs& a;
  const int sequence, kvh;
  const Blocks& blocks;
  const int begin, end;
  int held = -1;
  __device__ __forceinline__ WaveBlocks(const AttendArgs& args, int sequence, int kvh,
                                        const Blocks& blocks, int begin, int end)
      : a(args), sequence(sequence), kvh(kvh), blocks(blocks), begin(begin), end(end) {}
  // Of the share's block i, for every i of the wavefront in order.
  __device__ __forceinline__ int find(int i) {
    const int j = (i - begin) / kWaves % kWave;
    if (j == 0) {
      const int mine = i + kWaves * static_cast<int>(threadIdx.x & (kWave - 1));
      held = mine < end ? cache_block(a, sequence, kvh, blocks.at(mine)) : -1;
    }
    return __builtin_amdgcn_readlane(held, j);
  }
};

// The keys that a row sees: those of its window, and the first `sinks` up to itself.
struct Visible {
  int first;       // of the window
  uint32_t count;  // in the window
  int sinks;       // keys below this are seen too
  __device__ __forceinline__ bool window(int key) const {
    return static_cast<uint32_t>(key - first) < count;
  }
  __device__ __forceinline__ bool operator()(int key) const {
    return window(key) | (key < sinks);
  }
};

__device__ __forceinline__ Visible visible_to(int query, int stored, int window, int sinks) {
  const int last = min(query, stored - 1);
  const int first = query >= window ? query - window + 1 : 0;
  return {first, static_cast<uint32_t>(max(last - first + 1, 0)), min(sinks, last + 1)};
}

// int8 rows are multiplied by a quarter of their power of two, because the bias that their
// conversion takes off, 128 times the power, is no number for the two largest powers
// (rows past 2^127); the scale of scores, or the end of a sum, has the 4.
template <int TYPE>
constexpr float kUnit = TYPE == kPagedInt8 ? 4.0f : 1.0f;

// 2^(byte - 127) / kUnit; infinite for a row that is not finite, which makes it NaN.
template <int TYPE>
__device__ __forceinline__ float piece_power(uint32_t byte) {
  return __uint_as_float(byte << 23) * (1.0f / kUnit<TYPE>);
}

// A piece (8 values) of a page as bf16: K's values are times `power`, V's are
// q itself.
template <int TYPE>
struct Piece {
  using raw = uint2;
};
template <>
struct Piece<kPagedBf16> {
  using raw = uint4;
};

__device__ __forceinline__ uint32_t bits(bf16x2_t v) { return __builtin_bit_cast(uint32_t, v); }

// 128 + the eight int8 values, each by one instruction (an unsigned byte to float).
__device__ __forceinline__ void int8_values(uint2 w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = (i ? w.y : w.x) ^ 0x80808080u;
    x[4 * i] = static_cast<float>(u & 0xffu);
    x[4 * i + 1] = static_cast<float>((u >> 8) & 0xffu);
    x[4 * i + 2] = static_cast<float>((u >> 16) & 0xffu);
    x[4 * i + 3] = static_cast<float>(u >> 24);
  }
}

template <int TYPE>
__device__ __forceinline__ bf16x8 piece_bf16(typename Piece<TYPE>::raw w, float power) {
  if constexpr (TYPE == kPagedBf16) {
    return __builtin_bit_cast(bf16x8, w);
  } else if constexpr (TYPE == kPagedE4m3) {
    uint4 y;
    y.x = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, power, false));
    y.y = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, power, true));
    y.z = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, power, false));
    y.w = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, power, true));
    return __builtin_bit_cast(bf16x8, y);
  } else {
    // (known to be 1, the compiler subtracts in whole numbers first: twice the work)
    asm("" : "+v"(power));
    const float shift = -128.0f * power;
    float x[8];
    int8_values(w, x);
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (eight significant bits: the upper halves are the values)
      y[i] = __builtin_amdgcn_perm(__float_as_uint(__builtin_fmaf(x[2 * i + 1], power, shift)),
                                   __float_as_uint(__builtin_fmaf(x[2 * i], power, shift)),
                                   0x07060302u);
    return __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
  }
}

// Whether any value is an infinity or a NaN: by the largest of their magnitudes' bits.
template <int N>
__device__ __forceinline__ bool has_nonfinite(const bf16x8 (&v)[N]) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint4 w = __builtin_bit_cast(uint4, v[i]);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[j] & 0x7fff7fffu));
  }
  return (most[0] >= 0x7f80) | (most[1] >= 0x7f80);
}

// Values that are not finite become 0.
template <int N>
__device__ __forceinline__ void clear_nonfinite(bf16x8 (&vf)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint4 v = __builtin_bit_cast(uint4, vf[i]);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((w[j] & 0x7f80u) == 0x7f80u) w[j] &= 0xffff0000u;
      if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] &= 0x0000ffffu;
    }
    vf[i] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// One wavefront's running softmax state over its 32 rows: m in log2 units,
// shared by a row's two lanes and raised only when a score passes it by more
// than 2^8; each lane sums its own probabilities.
template <int D>
struct State {
  static constexpr int DT = D / 32;
  float m = -INFINITY, l = 0.0f;
  f32x16 o[DT];
};

template <int D>
__device__ __forceinline__ void clear(State<D>& st) {
#pragma unroll
  for (int i = 0; i < State<D>::DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[i][e] = 0.0f;
}

// A row of a tile: its token's position, operand and output rows.
struct TileRow {
  int position;
  int token;  // row of q and of the output
  int head;
};

__device__ __forceinline__ TileRow tile_row(const PagedSequence& s, int row, int rows, int rep,
                                            int kv_head) {
  const int r = min(row, rows - 1);
  const int token = r / rep;
  return {s.length - s.count + token, s.first + token, kv_head * rep + (r - token * rep)};
}

// The four wavefronts' shares of a tile of R rows, each in the units of its own
// maximum, joined: to the output, or to the split's partial sums.
template <int D, int R>
__device__ __forceinline__ void merge_tile(const AttendArgs& a, const float (&o_s)[kWaves][R][D + 4],
                                           const float (&ml_s)[kWaves][2][R],
                                           const PagedSequence& s, int row0, int rows, int kvh,
                                           int split, const Share& share) {
  constexpr int kThreads = kWaves * kWave, kPieces = R * (D / 4);
#pragma unroll
  for (int k = 0; k < (kPieces + kThreads - 1) / kThreads; ++k) {
    const int i = threadIdx.x + k * kThreads;
    const int r = min(i / (D / 4), R - 1), d = 4 * (i % (D / 4));
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ml_s[w][0][r]);
    float sum = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = ml_s[w][0][r], lw = ml_s[w][1][r];
      // A wavefront that saw nothing adds nothing (its maximum is -inf, its sum
      // 0; a NaN sum has to come through).
      const bool nothing = (mw == -INFINITY) & (lw == 0.0f);
      const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
      const float4 x = *reinterpret_cast<const float4*>(&o_s[w][r][d]);
      sum += nothing ? 0.0f : lw * f;
      y.x += nothing ? 0.0f : x.x * f;
      y.y += nothing ? 0.0f : x.y * f;
      y.z += nothing ? 0.0f : x.z * f;
      y.w += nothing ? 0.0f : x.w * f;
    }
    if (i >= kPieces || row0 + r >= rows) continue;
    const TileRow row = tile_row(s, row0 + r, rows, a.rep, kvh);
    const int64_t to = static_cast<int64_t>(row.token) * a.heads + row.head;
    if (share.whole) {
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      *reinterpret_cast<uint2*>(a.out + to * D + d) =
          make_uint2(pack_bf16x2(y.x * f, y.y * f), pack_bf16x2(y.z * f, y.w * f));
      if (a.splits > 1 && d == 0) a.part_ml[to * a.splits] = make_float2(0.0f, kWhole);
    } else {
      const int64_t at = to * a.splits + split;
      if (d == 0) a.part_ml[at] = make_float2(m, sum);
      if (share.begin < share.end) *reinterpret_cast<float4*>(a.part + at * D + d) = y;
    }
  }
}

// The key of score e of a block of 32 from k0, in a 32-row tile.
__device__ __forceinline__ int tile_key(int k0, int e) {
  return k0 + 16 * ((e >> 2) & 1) +
         4 * (2 * (e >> 3) + (static_cast<int>(threadIdx.x & (kWave - 1)) >> 5)) + (e & 3);
}

// Scores that the lane's row does not see become -infinity.  True where the block
// holds a value that is not finite.
template <int D>
__device__ __forceinline__ bool mask_block(f32x16& sc, const bf16x8 (&vf)[D / 16], int k0,
                                           int query, int stored, const AttendArgs& a) {
  const Visible sees = visible_to(query, stored, a.window, a.sinks);
  if (k0 < a.sinks) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = sees(tile_key(k0, e)) ? sc[e] : -INFINITY;
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = sees.window(tile_key(k0, e)) ? sc[e] : -INFINITY;
  }
  return __ballot(has_nonfinite(vf)) != 0;
}

// Adds a block's values that are not finite (in the order of pages, in LDS) to the
// rows that see their keys, as they are: any probability above 0 leaves them so.
template <int D>
__device__ __forceinline__ void add_nonfinite(State<D>& st, const uint16_t* v, int k0, int query,
                                              int stored, const AttendArgs& a) {
  const int half = static_cast<int>(threadIdx.x & (kWave - 1)) >> 5;
  const Visible sees = visible_to(query, stored, a.window, a.sinks);
#pragma unroll 1
  for (int i = 0; i < kPagedBlock; ++i) {
    if (!sees(k0 + i)) continue;
    const uint16_t* const from = v + ((i >> 2) & 3) * 128 + 4 * (i >> 4) + (i & 3);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int dim = 32 * t + 8 * (e >> 2) + 4 * half + (e & 3);
        const uint16_t x = from[(dim >> 4) * 512 + (dim & 15) * 8];
        if ((x & 0x7f80u) == 0x7f80u) st.o[t][e] += bf16_to_f32(x);
      }
  }
}

// P of 16 scores as two B operands, each times power(e), rounded to bf16 once; l takes
// the sums before both.
template <int D, typename F>
__device__ __forceinline__ void probabilities(State<D>& st, const f32x16& sc, float scale_log2,
                                              bf16x8 (&pf)[2], F power) {
  // A row that has seen no key yet has m = -inf and only -inf scores:
  // exp2(-inf - 0) = 0.
  const float neg = st.m == -INFINITY ? 0.0f : -st.m;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + e], scale_log2, neg));
      sum[e & 3] += p;
      pf[s][e] = static_cast<__bf16>(power(p, 8 * s + e));
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ float largest(const f32x16& sc) {
  float t[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) t[i] = fmaxf(fmaxf(sc[3 * i], sc[3 * i + 1]), sc[3 * i + 2]);
  return fmaxf(fmaxf(fmaxf(t[0], t[1]), t[2]), fmaxf(fmaxf(t[3], t[4]), sc[15]));
}

// Raises the running maximum to this lane's largest score where one passes it by
// more than 2^8.
template <int D>
__device__ __forceinline__ void raise(State<D>& st, float mx, float scale_log2) {
  mx *= scale_log2;
  if (__ballot(mx > st.m + 8.0f) != 0) {
    const float mn = fmaxf(st.m, fmaxf(mx, __shfl_xor(mx, 32)));
    const float alpha = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
    st.l *= alpha;
#pragma unroll
    for (int i = 0; i < State<D>::DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[i][e] *= alpha;
    st.m = mn;
  }
}

hipError_t launch_step(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s);
hipError_t launch_rows(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s);
hipError_t launch_tiles(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s);

// f(type, head width) as compile-time constants.
template <typename F>
hipError_t by_type_and_width(int type, int head_dim, F f) {
  auto by_width = [&](auto t) {
    if (head_dim == 64) f(t, std::integral_constant<int, 64>{});
    else if (head_dim == 96) f(t, std::integral_constant<int, 96>{});
    else f(t, std::integral_constant<int, 128>{});
    return hipGetLastError();
  };
  if (type == kPagedBf16) return by_width(std::integral_constant<int, kPagedBf16>{});
  if (type == kPagedE4m3) return by_width(std::integral_constant<int, kPagedE4m3>{});
  return by_width(std::integral_constant<int, kPagedInt8>{});
}

}  // namespace paged
}  // namespace parrot
