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
// 8-bit rows enter the products unrounded: K as q 2^x (exact in bf16), V as q
// with its power of two on the probability instead (one power per key, and a
// piece of V holds eight keys).  P is rounded to bf16 once.
#include <algorithm>
#include <type_traits>

#include "attention_lds.h"
#include "paged.h"

namespace parrot {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kRows = 32;  // rows of a wavefront's tile
constexpr int kMaxSplits = kWave;

struct AttendArgs {
  PagedCache cache;
  PagedBatch batch;
  const uint16_t* q;
  int64_t qs[2];  // element strides: row, head
  int heads, rep;
  int window;  // INT_MAX: none
  int sinks;
  float scale_log2;  // |scale| log2(e)
  uint32_t q_sign;   // 0x80008000 for a negative scale (q is negated), else 0
  int splits, whole;
  float* part;       // [rows * heads][splits][D], unnormalised
  float2* part_ml;   // [rows * heads][splits]
  uint16_t* out;     // [rows][heads][D]
};

// The key blocks that a tile's rows see, in order: the first `sinks` blocks,
// then those from `lo` on.
struct Blocks {
  int sinks, lo, count;
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : lo + i - sinks; }
};

__device__ __forceinline__ Blocks tile_blocks(int first, int last, int stored, int window,
                                              int sinks) {
  Blocks r{0, 0, 0};
  last = min(last, stored - 1);
  if (last < 0) return r;
  // (a window past the first position reaches every key; first - window + 1 fits)
  r.lo = first >= window ? min((first - window + 1) / kPagedBlock, last / kPagedBlock + 1) : 0;
  // sinks > 0 only count where the window has left them
  r.sinks = min(static_cast<int>((static_cast<int64_t>(sinks) + kPagedBlock - 1) / kPagedBlock),
                r.lo);
  r.count = r.sinks + last / kPagedBlock - r.lo + 1;
  return r;
}

// The key blocks of a split: at least kMinShare, and as many as the sequence's last
// rows (which see the most) need for `splits` of them; all, where those see no more
// than `whole`.  A tile that one share covers writes its output itself; its partial
// sums say so (kWhole).
constexpr int kMinShare = 8;
constexpr float kWhole = -1.0f;  // in place of a sum

struct Share {
  int begin, end;
  bool whole;
};

__device__ __forceinline__ Share split_share(const PagedSequence& s, int rows, int tile, int rep,
                                             const Blocks& blocks, int split, int splits,
                                             int whole, int window, int sinks) {
  if (splits == 1) return {0, blocks.count, true};
  const int row0 = (rows - 1) / tile * tile;
  const Blocks most = tile_blocks(s.length - s.count + row0 / rep, s.length - 1, s.stored, window,
                                  sinks);
  const int share = most.count <= whole ? most.count : max((most.count + splits - 1) / splits, kMinShare);
  const int begin = min(split * share, blocks.count);
  return {begin, min(begin + share, blocks.count), blocks.count <= share};
}

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

// One block of 32 keys: scores, softmax and values.
//   kf: K operands; load_v(i, s): V operand of 32-dim tile i, 16-key step s;
//   vpower: 2^x of the lane's 16 keys (8-bit types); k0: the block's first
//   position; query: the lane's row's; the tile's rows are at positions first ..
//   last, and keys < stored.
template <int TYPE, int D, typename LoadV>
__device__ __forceinline__ void attend_block(State<D>& st, const bf16x8 (&kf)[D / 16],
                                             const bf16x8 (&qf)[D / 16], LoadV load_v,
                                             const uint32_t (&vbytes)[4], int k0, int query,
                                             int first, int last, int stored,
                                             const AttendArgs& a) {
  constexpr int DT = D / 32;
  const int lane = threadIdx.x & (kWave - 1);
  const int half = lane >> 5, col = lane & 31;
  constexpr float kLazy = 8.0f;
  f32x16 sc;
#pragma unroll
  for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
  for (int u = 0; u < D / 16; ++u)
    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u], qf[u], sc, 0, 0, 0);

  auto key_of = [&](int e) { return k0 + 16 * ((e >> 2) & 1) + 4 * (2 * (e >> 3) + half) + (e & 3); };
  // A block that every row of the tile sees whole needs no mask.
  const bool whole = k0 + 31 <= min(first, stored - 1) &&
                     (last - k0 < a.window || k0 + 31 < a.sinks);
  if (!whole) {
    const Visible sees = visible_to(query, stored, a.window, a.sinks);
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = sees(key_of(e)) ? sc[e] : -INFINITY;
  }
  float t[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) t[i] = fmaxf(fmaxf(sc[3 * i], sc[3 * i + 1]), sc[3 * i + 2]);
  float mx = fmaxf(fmaxf(fmaxf(t[0], t[1]), t[2]), fmaxf(fmaxf(t[3], t[4]), sc[15]));
  mx *= a.scale_log2;
  if (__ballot(mx > st.m + kLazy) != 0) {
    const float mn = fmaxf(st.m, fmaxf(mx, __shfl_xor(mx, 32)));
    const float alpha = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
    st.l *= alpha;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[i][e] *= alpha;
    st.m = mn;
  }
  // A row that has seen no key yet has m = -inf and only -inf scores:
  // exp2(-inf - 0) = 0.
  const float neg = st.m == -INFINITY ? 0.0f : -st.m;
  float p[16], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], a.scale_log2, neg));
    sum[e & 3] += p[e];
  }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);

  bf16x8 vf[2 * DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) vf[2 * i + s] = load_v(i, s);

  // Values that some row must not see: times a probability of 0 an infinity or
  // a NaN is not 0.  Such a block takes the values row by row, those of keys
  // that the row does not see cleared.
  bool odd = false;
  if (!whole) {
    bool mine = has_nonfinite(vf);
    if constexpr (TYPE != kPagedBf16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mine |= ((vbytes[i] >> (8 * r)) & 0xffu) == kPagedNotFinite;
    }
    odd = __ballot(mine) != 0;
  }
  if constexpr (TYPE != kPagedBf16) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t byte = (vbytes[e >> 2] >> (8 * (e & 3))) & 0xffu;
      const float y = p[e] * __uint_as_float(byte << 23);
      p[e] = odd && sc[e] == -INFINITY ? 0.0f : y;
    }
  }
  bf16x8 pf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) pf[s][e] = static_cast<__bf16>(p[8 * s + e]);

  if (odd) {
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      f32x16 sums = st.o[i];
#pragma unroll 1
      for (int row = 0; row < kRows; ++row) {
        const Visible sees = visible_to(__builtin_amdgcn_readlane(query, row), stored, a.window,
                                        a.sinks);
        f32x16 y = st.o[i];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          bf16x8 v = vf[2 * i + s];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!sees(key_of(8 * s + e))) v[e] = static_cast<__bf16>(0.0f);
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pf[s], y, 0, 0, 0);
        }
        if (col == row) sums = y;
      }
      st.o[i] = sums;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s)
      st.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * i + s], pf[s], st.o[i], 0, 0, 0);
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
  for (int i = threadIdx.x; i < R * (D / 4); i += kWaves * kWave) {
    const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
    if (row0 + r >= rows) break;
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
      if (mw == -INFINITY && lw == 0.0f) continue;
      const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
      sum += lw * f;
      const float4 x = *reinterpret_cast<const float4*>(&o_s[w][r][d]);
      y.x += x.x * f;
      y.y += x.y * f;
      y.z += x.z * f;
      y.w += x.w * f;
    }
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

// Every wavefront takes every fourth key block of the workgroup's share, its
// operands straight from the pages; the four are merged in LDS.
template <int TYPE, int D>
__global__ __launch_bounds__(kWaves * kWave, 2) void paged_attend_kernel(AttendArgs a) {
  constexpr int KU = D / 16, DT = D / 32;
  using raw = typename Piece<TYPE>::raw;
  __shared__ float o_s[kWaves][kRows][D + 4];
  __shared__ float ml_s[kWaves][2][kRows];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int kvh = blockIdx.y, split = blockIdx.z;

  auto units_of = [&](const PagedSequence& s) { return (s.count * a.rep + kRows - 1) / kRows; };
  int sequence, tile;
  PagedSequence s;
  if (!paged_find(a.batch, a.cache.page, blockIdx.x, units_of, sequence, tile, s)) return;
  const int rows = s.count * a.rep;
  const int row0 = tile * kRows;
  const TileRow mine = tile_row(s, row0 + col, rows, a.rep, kvh);
  const int first = s.length - s.count + row0 / a.rep;
  const int last = s.length - s.count + (min(row0 + kRows, rows) - 1) / a.rep;
  const Blocks blocks = tile_blocks(first, last, s.stored, a.window, a.sinks);
  const Share share = split_share(s, rows, kRows, a.rep, blocks, split, a.splits, a.whole,
                                  a.window, a.sinks);
  if (share.whole && split > 0) return;
  const int begin = share.begin, end = share.end;

  State<D> st;
  clear(st);
  if (begin < end) {
    bf16x8 qf[KU];
    {
      const uint16_t* row = a.q + mine.token * a.qs[0] + mine.head * a.qs[1] + 8 * half;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        uint4 v = *reinterpret_cast<const uint4*>(row + 16 * u);
        v.x ^= a.q_sign;
        v.y ^= a.q_sign;
        v.z ^= a.q_sign;
        v.w ^= a.q_sign;
        qf[u] = __builtin_bit_cast(bf16x8, v);
      }
    }
    const int per_page = a.cache.page / kPagedBlock;
    const int kn = (col >> 3) & 1;
    const int kc = 4 * (2 * (col >> 4) + ((col >> 2) & 1)) + (col & 3);
    const int k_off = (kn * (D / 32) * 512 + half * 128 + kc * 8) / 8;  // in pieces
    const int v_off = ((col >> 4) * 512 + half * 128 + (col & 15) * 8) / 8;
    for (int i = begin + wave; i < end; i += kWaves) {
      const int blk = blocks.at(i);
      const int page = __builtin_amdgcn_readfirstlane(
          paged_page(a.batch, a.cache, sequence, blk / per_page));
      if (page < 0) continue;
      const int64_t at = static_cast<int64_t>(page) * a.cache.kv_heads + kvh;
      const int64_t off = (at * per_page + blk % per_page) * (kPagedBlock * D / 8);
      const raw* kp = static_cast<const raw*>(a.cache.key) + off + k_off;
      const raw* vp = static_cast<const raw*>(a.cache.value) + off + v_off;
      raw kw[KU], vw[2 * DT];
#pragma unroll
      for (int u = 0; u < KU; ++u) kw[u] = kp[32 * u];
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) vw[2 * t + h] = vp[128 * t + 32 * h];
      float kpower = 1.0f;
      uint32_t vbytes[4] = {0, 0, 0, 0};
      if constexpr (TYPE != kPagedBf16) {
        const int64_t e = at * a.cache.page + (blk % per_page) * kPagedBlock;
        kpower = __uint_as_float(static_cast<uint32_t>(a.cache.key_exponent[e + 16 * kn + kc]) << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vbytes[j] = *reinterpret_cast<const uint32_t*>(a.cache.value_exponent + e + 16 * (j & 1) +
                                                         8 * (j >> 1) + 4 * half);
      }
      const int k0 = blk * kPagedBlock;
      bf16x8 kf[KU];
#pragma unroll
      for (int u = 0; u < KU; ++u) kf[u] = piece_bf16<TYPE>(kw[u], kpower);
      attend_block<TYPE, D>(
          st, kf, qf, [&](int t, int h) { return piece_bf16<TYPE>(vw[2 * t + h], 1.0f); }, vbytes,
          k0, mine.position, first, last, s.stored, a);
    }
  }
  const float l = st.l + __shfl_xor(st.l, 32);
  if (half == 0) {
    ml_s[wave][0][col] = st.m;
    ml_s[wave][1][col] = l;
  }
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4*>(&o_s[wave][col][32 * t + 8 * (e >> 2) + 4 * half]) =
          make_float4(st.o[t][e], st.o[t][e + 1], st.o[t][e + 2], st.o[t][e + 3]);
  __syncthreads();
  merge_tile<D, kRows>(a, o_s, ml_s, s, row0, rows, kvh, split, share);
}

// ---------------------------------------------------------------------------
// Few rows per sequence (decode steps, short chunks): tiles of 16 rows.
//
// What bounds it: the pages' bytes, and below some MB the chain of dependent loads
// (starts, lengths and table, then keys).  Each wavefront takes every fourth block of
// its workgroup's share, straight from the pages into operand registers: the next
// block's keys once its scores are made, the next values once these are added, so that
// a block's registers are never empty and there are few of them.
//
//   S^T = K Q^T     v_mfma_f32_16x16x32_bf16, A = 16 keys (two per block), B = 16
//                   rows: lane 16 g + c holds keys 4 g .. + 3 and 16 + 4 g .. + 3 of
//                   row c, which is the order in which
//   O^T += V^T P^T  takes P^T as its B operand (32 keys).
// ---------------------------------------------------------------------------

constexpr int kStepRows = 16;

template <int TYPE, int D>
struct StepBlock {
  using raw = typename Piece<TYPE>::raw;
  static constexpr int N = D / 16;  // pieces of K, and of V, per lane
  raw k[N], v[N];
  uint32_t kbytes[2], vbytes[2];  // exponents of the lane's key rows; of its 8 scores
  int page;                       // -1: none
};

template <int TYPE, int D>
struct StepState {
  float m = -INFINITY, l = 0.0f;
  f32x4 o[D / 16];
};

// One block: scores, softmax and values.  then(): called where the block's keys are no
// longer needed.
template <int TYPE, int D, typename F>
__device__ __forceinline__ void step_block(StepState<TYPE, D>& st, const StepBlock<TYPE, D>& b,
                                           const bf16x8 (&qf)[D / 32], int k0, int query,
                                           int first, int last, int stored,
                                           const AttendArgs& a, uint16_t* v_s, F then) {
  constexpr int S = D / 32, T = D / 16;
  const int lane = threadIdx.x & (kWave - 1);
  const int g = lane >> 4;
  constexpr float kLazy = 8.0f;
  f32x4 sc[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    sc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float power = TYPE == kPagedBf16 ? 1.0f : __uint_as_float(b.kbytes[n] << 23);
#pragma unroll
    for (int s = 0; s < S; ++s)
      sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(piece_bf16<TYPE>(b.k[n * S + s], power), qf[s],
                                                      sc[n], 0, 0, 0);
  }
  then();
  auto key_of = [&](int e) { return k0 + 16 * (e >> 2) + 4 * g + (e & 3); };
  const bool whole = k0 + 31 <= min(first, stored - 1) &&
                     (last - k0 < a.window || k0 + 31 < a.sinks);
  if (!whole) {
    const Visible sees = visible_to(query, stored, a.window, a.sinks);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sc[e >> 2][e & 3] = sees(key_of(e)) ? sc[e >> 2][e & 3] : -INFINITY;
  }
  float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                   fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
  mx *= a.scale_log2;
  if (__ballot(mx > st.m + kLazy) != 0) {
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(st.m, mx);
    const float alpha = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
    st.l *= alpha;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[t][e] *= alpha;
    st.m = mn;
  }
  const float neg = st.m == -INFINITY ? 0.0f : -st.m;
  float p[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e >> 2][e & 3], a.scale_log2, neg));
  st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));

  bf16x8 vf[T];
#pragma unroll
  for (int t = 0; t < T; ++t) vf[t] = piece_bf16<TYPE>(b.v[t], 1.0f);
  uint32_t bytes[2] = {b.vbytes[0], b.vbytes[1]};
  auto byte_of = [&](int e) { return (bytes[e >> 2] >> (8 * (e & 3))) & 0xffu; };
  // Values that some row must not see: times a probability of 0 an infinity or a NaN
  // is not 0.  They are left out and added to the rows that see them.
  bool odd = false;
  if (!whole) {
    bool mine = has_nonfinite(vf);
    if constexpr (TYPE != kPagedBf16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) mine |= byte_of(e) == kPagedNotFinite;
    }
    odd = __ballot(mine) != 0;
    if (odd) {
      if constexpr (TYPE != kPagedBf16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (byte_of(e) == kPagedNotFinite) {  // (such an int8 row holds zeros)
            bytes[e >> 2] &= ~(0xffu << (8 * (e & 3)));
#pragma unroll
            for (int t = 0; t < T; ++t) vf[t][e] = __builtin_bit_cast(__bf16, uint16_t{0x7fc0});
          }
        }
      }
#pragma unroll
      for (int t = 0; t < T; ++t) *reinterpret_cast<bf16x8*>(v_s + (kWave * t + lane) * 8) = vf[t];
      clear_nonfinite(vf);
    }
  }
  bf16x8 pf;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = TYPE == kPagedBf16 ? p[e] : p[e] * __uint_as_float(byte_of(e) << 23);
    pf[e] = static_cast<__bf16>(y);
  }
#pragma unroll
  for (int t = 0; t < T; ++t)
    st.o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[t], pf, st.o[t], 0, 0, 0);
  if (odd) {
    const Visible sees = visible_to(query, stored, a.window, a.sinks);
#pragma unroll 1
    for (int i = 0; i < kPagedBlock; ++i) {
      if (!sees(k0 + i)) continue;
      const uint16_t* const from = v_s + ((i >> 2) & 3) * 128 + 4 * (i >> 4) + (i & 3);
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t x = from[t * 512 + (4 * g + e) * 8];
          if ((x & 0x7f80u) == 0x7f80u) st.o[t][e] += bf16_to_f32(x);
        }
    }
  }
}

template <int TYPE, int D>
__global__ __launch_bounds__(kWaves * kWave, D < 128 ? 3 : 2) void paged_step_kernel(AttendArgs a) {
  constexpr int S = D / 32, T = D / 16;
  using raw = typename Piece<TYPE>::raw;
  // (a wavefront's part takes a block's values before the merge, if any is not finite)
  __shared__ __attribute__((aligned(16))) float o_s[kWaves][kStepRows][D + 4];
  static_assert(kStepRows * (D + 4) * 4 >= kPagedBlock * D * 2, "a block's values fit");
  __shared__ float ml_s[kWaves][2][kStepRows];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int kvh = blockIdx.y, split = blockIdx.z;

  auto units_of = [&](const PagedSequence& s) {
    return (s.count * a.rep + kStepRows - 1) / kStepRows;
  };
  int sequence, tile;
  PagedSequence s;
  if (!paged_find(a.batch, a.cache.page, blockIdx.x, units_of, sequence, tile, s)) return;
  const int rows = s.count * a.rep;
  const int row0 = tile * kStepRows;
  const TileRow mine = tile_row(s, row0 + col, rows, a.rep, kvh);
  const int first = s.length - s.count + row0 / a.rep;
  const int last = s.length - s.count + (min(row0 + kStepRows, rows) - 1) / a.rep;
  const Blocks blocks = tile_blocks(first, last, s.stored, a.window, a.sinks);
  const Share share = split_share(s, rows, kStepRows, a.rep, blocks, split, a.splits, a.whole,
                                  a.window, a.sinks);
  if (share.whole && split > 0) return;
  const int begin = share.begin, end = share.end;

  StepState<TYPE, D> st;
#pragma unroll
  for (int t = 0; t < T; ++t) st.o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (begin + wave < end) {
    const int per_page = a.cache.page / kPagedBlock;
    // Lane j: the page of this wavefront's j-th block (of the last 64), and which of
    // its blocks that is.
    int ids = -1, ins = 0;
    StepBlock<TYPE, D> b = {};
    int64_t at = 0;  // the page and head that are loaded, and the block
    int in = 0;
    auto find = [&](int i) {
      const int j = (i - begin) / kWaves;
      if (j % kWave == 0) {
        const int blk = blocks.at(i + kWaves * lane), at = blk / per_page;
        ids = i + kWaves * lane < end ? paged_page(a.batch, a.cache, sequence, at) : -1;
        ins = blk - at * per_page;
      }
      b.page = __builtin_amdgcn_readlane(ids, j % kWave);
      in = __builtin_amdgcn_readlane(ins, j % kWave);
      at = static_cast<int64_t>(max(b.page, 0)) * a.cache.kv_heads + kvh;
    };
    auto load = [&](const void* pages, const uint8_t* exponents, raw(&to)[T], uint32_t(&bytes)[2],
                    auto key) {
      if (b.page < 0) return;
      const raw* from = static_cast<const raw*>(pages) + (at * per_page + in) * (kPagedBlock * D / 8);
#pragma unroll
      for (int u = 0; u < T; ++u) to[u] = from[kWave * u + lane];
      if constexpr (TYPE != kPagedBf16) {
        const uint8_t* e = exponents + at * a.cache.page + in * kPagedBlock;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if constexpr (decltype(key)::value) bytes[n] = e[16 * n + col];
          else bytes[n] = *reinterpret_cast<const uint32_t*>(e + 16 * n + 4 * g);
        }
      }
    };
    auto load_keys = [&] {
      load(a.cache.key, a.cache.key_exponent, b.k, b.kbytes, std::true_type{});
    };
    auto load_values = [&] {
      load(a.cache.value, a.cache.value_exponent, b.v, b.vbytes, std::false_type{});
    };
    find(begin + wave);
    load_keys();
    load_values();
    bf16x8 qf[S];
    {
      const uint16_t* row = a.q + mine.token * a.qs[0] + mine.head * a.qs[1] + 8 * g;
#pragma unroll
      for (int u = 0; u < S; ++u) {
        uint4 v = *reinterpret_cast<const uint4*>(row + 32 * u);
        v.x ^= a.q_sign;
        v.y ^= a.q_sign;
        v.z ^= a.q_sign;
        v.w ^= a.q_sign;
        qf[u] = __builtin_bit_cast(bf16x8, v);
      }
    }
    for (int i = begin + wave; i < end; i += kWaves) {
      const bool more = i + kWaves < end;
      // (of a block without a page no row sees a key)
      step_block<TYPE, D>(st, b, qf, blocks.at(i) * kPagedBlock, mine.position, first, last,
                          b.page >= 0 ? s.stored : 0, a,
                          reinterpret_cast<uint16_t*>(&o_s[wave][0][0]), [&] {
                            if (!more) return;
                            find(i + kWaves);
                            load_keys();
                          });
      if (more) load_values();
    }
  }
  float l = st.l + __shfl_xor(st.l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) {
    ml_s[wave][0][col] = st.m;
    ml_s[wave][1][col] = l;
  }
#pragma unroll
  for (int t = 0; t < T; ++t)
    *reinterpret_cast<float4*>(&o_s[wave][col][16 * t + 4 * g]) =
        make_float4(st.o[t][0], st.o[t][1], st.o[t][2], st.o[t][3]);
  __syncthreads();
  merge_tile<D, kStepRows>(a, o_s, ml_s, s, row0, rows, kvh, split, share);
}

// ---------------------------------------------------------------------------
// Many rows per sequence (prompts and their chunks): a wavefront has 32 rows, the
// four of a workgroup share key blocks through LDS.
//
// Each wavefront brings one of a stage's four matrices (K and V of two blocks) from
// the pages into registers while the stage before is computed, and writes it to LDS
// as bf16: an 8-bit page is converted once for 128 rows.  K's second half lies 128
// bytes further, so that the 16 lanes of a read's phase, which take eight keys of
// each half, fall into different banks.
// ---------------------------------------------------------------------------

constexpr int kTileRows = kWaves * kRows;

// A V piece with its positions' powers of two (int8: shift = -128 times the power).
template <int TYPE>
__device__ __forceinline__ bf16x8 value_piece(uint2 w, const float (&power)[8],
                                              const float (&shift)[8]) {
  float x[8];
  if constexpr (TYPE == kPagedE4m3) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = static_cast<int>(i ? w.y : w.x);
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(u, false);
      const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(u, true);
      x[4 * i] = lo[0] * power[4 * i], x[4 * i + 1] = lo[1] * power[4 * i + 1];
      x[4 * i + 2] = hi[0] * power[4 * i + 2], x[4 * i + 3] = hi[1] * power[4 * i + 3];
    }
  } else {
    int8_values(w, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(x[e], power[e], shift[e]);
  }
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)  // (eight significant bits at most: the upper halves)
    y[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]),
                                 0x07060302u);
  return __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
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

// P of 16 scores as two B operands, rounded to bf16 once; l takes the sums before
// the rounding.
template <int D>
__device__ __forceinline__ void probabilities(State<D>& st, const f32x16& sc, float scale_log2,
                                              bf16x8 (&pf)[2]) {
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
      pf[s][e] = static_cast<__bf16>(p);
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Raises the running maximum to this lane's largest score where one passes it by
// more than 2^8.
template <int D>
__device__ __forceinline__ void raise(State<D>& st, const f32x16& sc, float scale_log2) {
  float t[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) t[i] = fmaxf(fmaxf(sc[3 * i], sc[3 * i + 1]), sc[3 * i + 2]);
  float mx = fmaxf(fmaxf(fmaxf(t[0], t[1]), t[2]), fmaxf(fmaxf(t[3], t[4]), sc[15]));
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

template <int TYPE, int D>
__global__ __launch_bounds__(kWaves * kWave, 2) void paged_tile_kernel(AttendArgs a) {
  constexpr int KU = D / 16, DT = D / 32, S = D / 32;
  constexpr int kHalf = 64;                                  // elements between K's halves
  constexpr int kK = kPagedBlock * D + kHalf;                // elements of K, then of V
  constexpr int kBlock = kK + kPagedBlock * D;
  constexpr int kBytes = TYPE == kPagedBf16 ? 2 : 1;
  constexpr int kLoads = kPagedBlock * D * kBytes / (16 * kWave);  // 1 KB pieces of a matrix
  __shared__ __attribute__((aligned(16))) uint16_t stage[2][2][kBlock];  // [buffer][block]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int unit = blockIdx.x / a.cache.kv_heads, kvh = blockIdx.x - unit * a.cache.kv_heads;
  const int split = blockIdx.z;

  auto units_of = [&](const PagedSequence& s) {
    return (s.count * a.rep + kTileRows - 1) / kTileRows;
  };
  int sequence, tile;
  PagedSequence s;
  if (!paged_find_last(a.batch, a.cache.page, unit, units_of, sequence, tile, s)) return;
  const int rows = s.count * a.rep;
  const int tile0 = tile * kTileRows, row0 = tile0 + wave * kRows;
  const TileRow mine = tile_row(s, row0 + col, rows, a.rep, kvh);
  const int before = s.length - s.count;
  const Blocks blocks = tile_blocks(before + tile0 / a.rep,
                                    before + (min(tile0 + kTileRows, rows) - 1) / a.rep, s.stored,
                                    a.window, a.sinks);
  const Share share = split_share(s, rows, kTileRows, a.rep, blocks, split, a.splits, a.whole,
                                  a.window, a.sinks);
  if (share.whole && split > 0) return;
  const int begin = share.begin, end = share.end;
  // This wavefront's own rows (none: it only brings blocks).
  const bool has = row0 < rows;
  const int first = before + row0 / a.rep;
  const int last = before + (min(row0 + kRows, rows) - 1) / a.rep;

  State<D> st;
  clear(st);
  if (begin < end) {
    bf16x8 qf[KU];
    {
      const uint16_t* row = a.q + mine.token * a.qs[0] + mine.head * a.qs[1] + 8 * half;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        uint4 v = *reinterpret_cast<const uint4*>(row + 16 * u);
        v.x ^= a.q_sign;
        v.y ^= a.q_sign;
        v.z ^= a.q_sign;
        v.w ^= a.q_sign;
        qf[u] = __builtin_bit_cast(bf16x8, v);
      }
    }
    const int per_page = a.cache.page / kPagedBlock;
    const int which = wave >> 1;       // block of a stage, and matrix, that this wavefront brings
    const bool brings_v = wave & 1;
    // Lane j: the page of the share's j-th block (of the last 64), and which of its
    // blocks that is.
    int ids = -1, ins = 0;
    int page0 = -1, page1 = -1;        // of the stage that is brought
    uint4 got[kLoads];                 // 8-bit types
    uint32_t bytes[2] = {0, 0};
    auto bring = [&](int i, int buf) {  // blocks i and i + 1
      const int j = (i - begin) % kWave;
      if (j == 0) {
        const int blk = blocks.at(i + lane), at = blk / per_page;
        ids = i + lane < end ? paged_page(a.batch, a.cache, sequence, at) : -1;
        ins = blk - at * per_page;
      }
      page0 = __builtin_amdgcn_readlane(ids, j);
      page1 = __builtin_amdgcn_readlane(ids, j + 1);
      const int page = which ? page1 : page0;
      if (page < 0) return;
      const int in = __builtin_amdgcn_readlane(ins, j + which);
      const int64_t at = static_cast<int64_t>(page) * a.cache.kv_heads + kvh;
      const char* from = static_cast<const char*>(brings_v ? a.cache.value : a.cache.key) +
                         (at * per_page + in) * (kPagedBlock * D * kBytes);
      if constexpr (TYPE == kPagedBf16) {
        const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(from, kPagedBlock * D * kBytes);
        uint16_t* to = &stage[buf][which][brings_v ? kK : 0];
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
          buffer_to_lds16(rsrc, to + 512 * u + (!brings_v && u >= S ? kHalf : 0), lane * 16u,
                          1024u * u);
      } else {
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
          got[u] = reinterpret_cast<const uint4*>(from)[kWave * u + lane];
        const int64_t e = at * a.cache.page + in * kPagedBlock;
        if (brings_v) {  // positions 4 g .. + 3 and 16 + 4 g .. + 3 of the lane's pieces
          const uint8_t* x = a.cache.value_exponent + e + 4 * ((lane >> 3) & 3);
          bytes[0] = *reinterpret_cast<const uint32_t*>(x);
          bytes[1] = *reinterpret_cast<const uint32_t*>(x + 16);
        } else {  // keys c, c + 1 of either half
          const uint8_t* x = a.cache.key_exponent + e + ((2 * lane) & 15);
          bytes[0] = *reinterpret_cast<const uint16_t*>(x);
          bytes[1] = *reinterpret_cast<const uint16_t*>(x + 16);
        }
      }
    };
    auto put = [&](int buf) {  // 8-bit types: what was brought, as bf16
      if constexpr (TYPE != kPagedBf16) {
        if ((which ? page1 : page0) < 0) return;
        uint16_t* const to = &stage[buf][which][brings_v ? kK : 0];
        if (brings_v) {
          float power[8], shift[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            power[e] = __uint_as_float(((bytes[e >> 2] >> (8 * (e & 3))) & 0xffu) << 23);
            shift[e] = -128.0f * power[e];
          }
#pragma unroll
          for (int u = 0; u < kLoads; ++u) {
            bf16x8* const p = reinterpret_cast<bf16x8*>(to + (kWave * u + lane) * 16);
            p[0] = value_piece<TYPE>(make_uint2(got[u].x, got[u].y), power, shift);
            p[1] = value_piece<TYPE>(make_uint2(got[u].z, got[u].w), power, shift);
          }
        } else {
#pragma unroll
          for (int u = 0; u < kLoads; ++u) {
            const int at = (kWave * u + lane) * 16;
            const uint32_t b = at >= 16 * D ? bytes[1] : bytes[0];
            bf16x8* const p = reinterpret_cast<bf16x8*>(to + at + (at >= 16 * D ? kHalf : 0));
            p[0] = piece_bf16<TYPE>(make_uint2(got[u].x, got[u].y), __uint_as_float((b & 0xffu) << 23));
            p[1] = piece_bf16<TYPE>(make_uint2(got[u].z, got[u].w), __uint_as_float((b >> 8) << 23));
          }
        }
      }
    };

    const int kn = (col >> 3) & 1;
    const int kc = 4 * (2 * (col >> 4) + ((col >> 2) & 1)) + (col & 3);
    const uint32_t k_off = static_cast<uint32_t>(kn * (S * 1024 + 2 * kHalf) + half * 256 + kc * 16);
    const uint32_t v_off =
        static_cast<uint32_t>(2 * kK + (col >> 4) * 1024 + half * 256 + (col & 15) * 16);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) const uint16_t*)&stage[0][0][0]));
    // True where values that are not finite were left out.
    auto block = [&](uint32_t lds, int k0) -> bool {
      bf16x8 kf[KU], vf[2 * DT], pf[2];
      lds_frags<0, 512>(lds + k_off, kf);
      f32x16 sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
      for (int u = 0; u < KU; ++u)
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u], qf[u], sc, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      read_values<0>(lds + v_off, vf);
      // A block that every row of the tile sees whole needs no mask.
      const bool whole = k0 + 31 <= min(first, s.stored - 1) &&
                         (last - k0 < a.window || k0 + 31 < a.sinks);
      // Values that some row must not see: times a probability of 0 an infinity or a
      // NaN is not 0.
      bool odd = false;
      if (!whole) {
        odd = mask_block<D>(sc, vf, k0, mine.position, s.stored, a);
        if (odd) clear_nonfinite(vf);
      }
      raise(st, sc, a.scale_log2);
      probabilities(st, sc, a.scale_log2, pf);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < DT; ++t)
          st.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * t + h], pf[h], st.o[t], 0, 0, 0);
      return odd;
    };
    bring(begin, 0);
    for (int i = begin, buf = 0; i < end; i += 2, buf ^= 1) {
      const int now0 = page0, now1 = page1;
      if constexpr (TYPE == kPagedBf16) {
        // This wavefront's copies have landed; past the barrier everybody's have, and
        // nobody reads the other buffer any more.
        wait_vm_barrier<0>();
      } else {
        put(buf);
        __syncthreads();
      }
      if (i + 2 < end) bring(i + 2, buf ^ 1);
      if (!has) continue;
      // Blocks without a page, and those that none of this wavefront's rows sees, are
      // left out.
      auto seen = [&](int k0) {
        return k0 <= last && (first - (k0 + 31) < a.window || k0 < a.sinks);
      };
      const uint32_t lds = lds0 + buf * (4 * kBlock);
      const int k0 = blocks.at(i) * kPagedBlock, k1 = blocks.at(i + 1) * kPagedBlock;
      uint32_t odd = 0;
      if (now0 >= 0 && seen(k0)) odd = block(lds, k0);
      if (now1 >= 0 && seen(k1)) odd |= 2 * block(lds + 2 * kBlock, k1);
#pragma unroll 1
      for (int b = 0; odd != 0; ++b, odd >>= 1)
        if (odd & 1)
          add_nonfinite<D>(st, &stage[buf][b][kK], b ? k1 : k0, mine.position, s.stored, a);
    }
  }
  const float l = st.l + __shfl_xor(st.l, 32);
  if (row0 + col >= rows) return;
  const int64_t to = static_cast<int64_t>(mine.token) * a.heads + mine.head;
  if (share.whole) {
    if (a.splits > 1 && half == 0) a.part_ml[to * a.splits] = make_float2(0.0f, kWhole);
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<uint2*>(a.out + to * D + 32 * t + 8 * (e >> 2) + 4 * half) =
            make_uint2(pack_bf16x2(st.o[t][e] * f, st.o[t][e + 1] * f),
                       pack_bf16x2(st.o[t][e + 2] * f, st.o[t][e + 3] * f));
  } else {
    const int64_t at = to * a.splits + split;
    if (half == 0) a.part_ml[at] = make_float2(st.m, l);
    if (begin < end) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<float4*>(a.part + at * D + 32 * t + 8 * (e >> 2) + 4 * half) =
              make_float4(st.o[t][e], st.o[t][e + 1], st.o[t][e + 2], st.o[t][e + 3]);
    }
  }
}

// A share's part in the joined row: in units of the largest maximum; -1 where it saw
// nothing (a NaN sum has to come through).
__device__ __forceinline__ float share_weight(float2 ml, float m) {
  if (ml.x == -INFINITY) return ml.y == 0.0f ? -1.0f : 1.0f;
  return __builtin_amdgcn_exp2f(ml.x - m);
}

// Rows of no sequence, and those that one share wrote whole, stay as they are.
__device__ __forceinline__ bool joined_already(const AttendArgs& a, int64_t to) {
  const int64_t token = to / a.heads;
  return token >= a.batch.rows || token < a.batch.starts[0] ||
         token >= a.batch.starts[a.batch.batch] || a.part_ml[to * a.splits].y == kWhole;
}

// Joins the shares of split tiles where there are many rows: D / 4 threads a row, one
// share after the other.
template <int D>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(AttendArgs a) {
  constexpr int kPer = 256 / (D / 4);
  const int slot = threadIdx.x / (D / 4), at = threadIdx.x - slot * (D / 4);
  const int64_t to = static_cast<int64_t>(blockIdx.x) * kPer + slot;
  if (slot >= kPer || joined_already(a, to)) return;
  const float2* const ml = a.part_ml + to * a.splits;
  const float4* const part = reinterpret_cast<const float4*>(a.part) + to * a.splits * (D / 4) + at;
  float m = -INFINITY, sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) m = fmaxf(m, ml[i].x);
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    const float f = share_weight(ml[i], m);
    if (f < 0.0f) continue;
    sum += ml[i].y * f;
    const float4 x = part[i * (D / 4)];
    y.x += x.x * f;
    y.y += x.y * f;
    y.z += x.z * f;
    y.w += x.w * f;
  }
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(a.out + to * D + 4 * at) =
      make_uint2(pack_bf16x2(y.x * f, y.y * f), pack_bf16x2(y.z * f, y.w * f));
}

// ... and where there are few: a workgroup a row, one share a lane for their weights,
// then D / 4 threads for every tenth share (D = 96).
template <int D>
__global__ __launch_bounds__(256) void paged_join_shares_kernel(AttendArgs a) {
  constexpr int kGroups = 256 / (D / 4);
  __shared__ float w_s[kMaxSplits];
  __shared__ float4 y_s[kGroups][D / 4];
  const int64_t to = blockIdx.x;
  if (joined_already(a, to)) return;
  if (threadIdx.x < kWave) {
    const int i = threadIdx.x;
    const float2 ml = i < a.splits ? a.part_ml[to * a.splits + i] : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float f = share_weight(ml, m);
    const float sum = wave_sum(f < 0.0f ? 0.0f : ml.y * f);
    w_s[i] = f < 0.0f ? -1.0f : sum == 0.0f ? 0.0f : f / sum;
  }
  __syncthreads();
  const int group = threadIdx.x / (D / 4), at = threadIdx.x - group * (D / 4);
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (group < kGroups) {
    for (int i = group; i < a.splits; i += kGroups) {
      const float f = w_s[i];
      if (f < 0.0f) continue;
      const float4 x = *reinterpret_cast<const float4*>(a.part + (to * a.splits + i) * D + 4 * at);
      y.x += x.x * f;
      y.y += x.y * f;
      y.z += x.z * f;
      y.w += x.w * f;
    }
    y_s[group][at] = y;
  }
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) {
    const float4 x = y_s[i][at];
    y.x += x.x;
    y.y += x.y;
    y.z += x.z;
    y.w += x.w;
  }
  *reinterpret_cast<uint2*>(a.out + to * D + 4 * at) =
      make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

}  // namespace

namespace {

// Rows of a workgroup's tile: 16 where a sequence has no more than 32 on average
// (most of a larger tile would be empty), 128 from 96 on.
int tile_rows(int batch, int rows, int rep) {
  const int64_t all = static_cast<int64_t>(rows) * rep, n = std::min(batch, rows);
  return all <= 32 * n ? kStepRows : all < 96 * n ? kRows : kTileRows;
}

}  // namespace

namespace {

struct Plan {
  int tile, splits, whole;
};

// Splits: enough workgroups for the chip, each with 256 keys at least, where a tile may
// see more keys than are faster without the join's launch: 768 for 16 and 32 rows
// (one sequence, 8 heads on 2 of 96, one launch / split, us: 512 keys 6.0 / 8.4, 768
// 7.1 / 8.1, 1024 8.2 / 8.3, 1536 10.4 / 8.4; 64 sequences of 8 kv heads of 64 in int8
// 768 17.3 / 18.1, 1024 21.3 / 21.1), and for 128 rows the more the more workgroups
// there are without (16: 384 12.8 / 14.2, 512 15.6 / 14.2; 104: 768 21.4 / 23.0, 1024
// 27.0 / 26.4).
Plan plan(int batch, int rows, int heads, int kv_heads, int page, int width, int window,
          int sinks) {
  const int rep = heads / kv_heads;
  const int tile = tile_rows(batch, rows, rep);
  const int64_t tiles = (static_cast<int64_t>(rows) * rep + tile - 1) / tile;
  const int64_t units = std::max<int64_t>({tiles, std::min(batch, rows), 1}) * kv_heads;
  // The most keys a tile can see: its table's, or the window, the sinks and
  // the tile's own span.
  int64_t keys = static_cast<int64_t>(width) * page;
  if (window < INT32_MAX) keys = std::min<int64_t>(keys, int64_t{window} + sinks + tile + 64);
  const int64_t line = tile == kTileRows ? std::min<int64_t>(384 + 4 * units, 1024) : 768;
  const int64_t want = (1024 + units - 1) / units;
  const int64_t splits =
      keys <= line ? 1 : std::min<int64_t>({want, (keys + 255) / 256, kMaxSplits});
  return {tile, static_cast<int>(splits), static_cast<int>(line / kPagedBlock)};
}

}  // namespace

int paged_attention_splits(int batch, int rows, int heads, int kv_heads, int page, int width,
                           int window, int sinks) {
  return plan(batch, rows, heads, kv_heads, page, width, window, sinks).splits;
}

size_t paged_attention_workspace_bytes(int splits, int rows, int heads, int head_dim) {
  if (splits <= 1) return 0;
  return static_cast<size_t>(splits) * rows * heads * (head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedCache& cache, int type, int head_dim,
                                  const PagedBatch& batch, const uint16_t* q,
                                  const int64_t* q_strides, int heads, int window, int sinks,
                                  float scale, void* workspace, uint16_t* out, hipStream_t s) {
  if (batch.rows == 0 || batch.batch == 0) return hipSuccess;
  AttendArgs a;
  a.cache = cache;
  a.batch = batch;
  a.q = q;
  a.qs[0] = q_strides[0];
  a.qs[1] = q_strides[1];
  a.heads = heads;
  a.rep = heads / cache.kv_heads;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.out = out;
  const Plan p = plan(batch.batch, batch.rows, heads, cache.kv_heads, cache.page, batch.width,
                      window, sinks);
  const int tile = p.tile, splits = p.splits;
  a.splits = splits;
  a.whole = p.whole;
  a.part = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part +
                                        static_cast<size_t>(splits) * batch.rows * heads * head_dim);
  // ceil(n rep / tile) tiles a sequence
  const int64_t tiles = static_cast<int64_t>(batch.rows) * a.rep / tile +
                        std::min(batch.batch, batch.rows);
  const dim3 grid(static_cast<uint32_t>(tiles), cache.kv_heads, splits);
  const dim3 tile_grid(static_cast<uint32_t>(tiles * cache.kv_heads), 1, splits);
  auto run = [&](auto t, auto d) {
    constexpr int TYPE = decltype(t)::value, D = decltype(d)::value;
    if (tile == kStepRows) paged_step_kernel<TYPE, D><<<grid, kWaves * kWave, 0, s>>>(a);
    else if (tile == kRows) paged_attend_kernel<TYPE, D><<<grid, kWaves * kWave, 0, s>>>(a);
    else paged_tile_kernel<TYPE, D><<<tile_grid, kWaves * kWave, 0, s>>>(a);
    if (splits > 1) {
      constexpr int kPer = 256 / (D / 4);
      const uint32_t rows = static_cast<uint32_t>(batch.rows * heads);
      if (rows < 2048) paged_join_shares_kernel<D><<<rows, 256, 0, s>>>(a);
      else paged_join_rows_kernel<D><<<(rows + kPer - 1) / kPer, 256, 0, s>>>(a);
    }
    return hipGetLastError();
  };
  auto by_width = [&](auto t) {
    if (head_dim == 64) return run(t, std::integral_constant<int, 64>{});
    if (head_dim == 96) return run(t, std::integral_constant<int, 96>{});
    return run(t, std::integral_constant<int, 128>{});
  };
  if (type == kPagedBf16) return by_width(std::integral_constant<int, kPagedBf16>{});
  if (type == kPagedE4m3) return by_width(std::integral_constant<int, kPagedE4m3>{});
  return by_width(std::integral_constant<int, kPagedInt8>{});
}

}  // namespace parrot
