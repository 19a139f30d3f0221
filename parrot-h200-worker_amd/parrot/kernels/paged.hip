// Writing new keys and values into the pages of a KV cache, quantised to 8 or 4
// bits on the way where the cache holds so few, and reading sequences back.
//
// A workgroup takes one block of 32 positions of one kv head: eight threads a
// row, each with D / 8 of its values, so that a row's largest magnitude is a
// maximum over eight lanes and K leaves in pieces of four consecutive dims.  V
// turns in LDS, because its pieces hold eight positions of one dim; a piece of
// which only some positions are new (a chunk's ends, a single token) is written
// value by value, the others are left as they are.
//
// What bounds it: bytes for many rows, the chain starts - table - page for few.
// Measured, 2 heads of 96: 16384 rows into e4m3 pages 6.1 us (19 MB, 3.1 TB/s), read back
// 6.2 us (3.0 TB/s), bf16 6.1 and 5.7 (25 MB, 4.1 and 4.4 TB/s); with RoPE and 8 query heads 16.9
// and 16.6 (71 and 77 MB, 4.2 and 4.6 TB/s); one row of one sequence 4.0 us, in bf16 3.3 and
// 2.9, with RoPE 6.3 and 5.6, of which 2.5 to 3 are a launch's.  Into 4-bit pages (a trace's
// times) 6.7 us (15.8 MB, 2.4 TB/s) and back 5.8 (2.7 TB/s), one row 3.9 and, of 501, 3.3.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace parrot {

namespace {

constexpr int kThreads = 256;

typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <int TYPE>
struct Stored {
  using type = uint8_t;
};
template <>
struct Stored<kPagedBf16> {
  using type = uint16_t;
};

// The byte of a row whose largest magnitude has the bf16 bits `amax`
// ((1 + m / 128) 2^(e - 127), m the low 7 bits): the type's largest value is
// 1.75 2^8 (448) or 127 / 64 2^6 (127), so the power is e - 127 less 8 or 6,
// one more where 1 + m / 128 is larger than that first factor.
template <int TYPE>
__device__ __forceinline__ uint32_t exponent_byte(uint32_t amax) {
  const int e = static_cast<int>(amax >> 7), m = static_cast<int>(amax & 0x7f);
  if (e == 255) return kPagedNotFinite;
  // (6 2^125 is the largest that e2m1 holds below 2^128)
  if (TYPE == kPagedE2m1)
    return static_cast<uint32_t>(min(max(e - 129 + (m > 96), kPagedMinExponent), 125) + 127);
  const int power = TYPE == kPagedE4m3 ? e - 135 + (m > 96) : e - 133 + (m > 126);
  return static_cast<uint32_t>(max(power, kPagedMinExponent) + 127);
}

// Four values over 2^(byte - 127), rounded to nearest even (a product by a
// power of two is exact; byte <= 249, so its inverse is a normal number).  At the
// largest power a magnitude may round up to 2^128: it stays at the value below
// that (240 2^120, 63 2^122), so that a finite row reads back finite.
template <int TYPE>
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], uint32_t byte) {
  if (byte == kPagedNotFinite) return TYPE == kPagedE4m3 ? 0x7f7f7f7fu : 0u;
  const float inverse = __uint_as_float((254u - byte) << 23);
  constexpr uint32_t kTop = TYPE == kPagedE4m3 ? 247 : 249;
  const float most = byte != kTop ? 448.0f : TYPE == kPagedE4m3 ? 240.0f : 63.0f;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(x[i] * inverse, -most), most);
  if constexpr (TYPE == kPagedE4m3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    return static_cast<uint32_t>(w);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w |= (static_cast<uint32_t>(static_cast<int>(rintf(y[i]))) & 0xffu) << (8 * i);
    return w;
  }
}

template <int TYPE>
__device__ __forceinline__ void value4(uint32_t w, uint32_t byte, float (&x)[4]) {
  if (byte == kPagedNotFinite) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(0x7fc00000u);
    return;
  }
  const float power = __uint_as_float(byte << 23);
  if constexpr (TYPE == kPagedE4m3) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = a[0] * power;
    x[1] = a[1] * power;
    x[2] = b[0] * power;
    x[3] = b[1] * power;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * power;
  }
}

// The largest magnitude (bf16 bits; a NaN's are the largest) of the eight
// lanes that share a row.
__device__ __forceinline__ uint32_t row_amax(uint32_t a) {
#pragma unroll
  for (int d = 1; d < 8; d *= 2) a = max(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), d)));
  return a;
}

// Four bf16 values over 2^(byte - 127) as 4 bits each, nearest even (one conversion, which
// keeps what is above 6 at 6); zeros for a byte of kPagedNotFinite.
__device__ __forceinline__ uint32_t quantise4_e2m1(uint2 x, uint32_t byte) {
  if (byte == kPagedNotFinite) return 0;
  const float power = __uint_as_float(byte << 23);
  const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      0, __builtin_bit_cast(bf16x2_t, x.x), power, 0);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x.y), power, 1);
}

// Where a block of 4-bit values lies, and what this thread has of it.  Rows: eight threads
// a row, thread `part` of row p with dims 32 j + 4 part .. of each group j.  V, which the
// records hold by positions, by quads: words (o, u) of records (g, c0 .. c0 + 3), D threads
// in all; in LDS the rows' four-value pieces, piece 8 u + 4 o + c0 / 4 of eight rows.
template <int D>
struct BlockE2m1 {
  static constexpr int S = D / 32, kLd = D / 4 + 2;
  uint8_t* k;             // 16-bit pieces of the thread's row: k + 4 j
  uint32_t* v;            // words of the thread's quad: v + 2 S i
  uint8_t* key_bytes;     // of the row's groups
  uint8_t* value_byte;
  int g, piece;           // of the quad; -1: none
  __device__ __forceinline__ BlockE2m1(const PagedCache& c, int64_t block) {
    const int p = threadIdx.x >> 3, part = threadIdx.x & 7, n = p >> 4, row = p & 15;
    k = static_cast<uint8_t*>(c.key) + block * (16 * D) +
        (((part >> 1) * 16 + row) * 2 * S + n * S) * 4 + 2 * (part & 1);
    key_bytes = c.key_exponent + block * D + (2 * row + n) * S;
    value_byte = c.value_exponent + block * kPagedBlock + p;
    const int quad = threadIdx.x / (2 * S), w = threadIdx.x - quad * 2 * S;
    const int o = w >= S, u = w - o * S;
    g = quad >> 2;
    piece = threadIdx.x < D ? 8 * u + 4 * o + (quad & 3) : -1;
    v = static_cast<uint32_t*>(c.value) + block * (4 * D) + quad * 4 * 2 * S + w;
  }
  // The position of the e-th value of the quad's words.
  __device__ __forceinline__ int position(int e) const { return (e >> 2) * 16 + 4 * g + (e & 3); }
};

// Rows lo .. hi - 1 of a block written (kw, vw: the thread's row); the others stay.
template <int D>
__device__ __forceinline__ void append_e2m1(const PagedCache& c, int64_t block,
                                            const uint2 (&kw)[D / 32], const uint2 (&vw)[D / 32],
                                            int lo, int hi, uint16_t (*v_s)[BlockE2m1<D>::kLd]) {
  constexpr int S = D / 32;
  const int p = threadIdx.x >> 3, part = threadIdx.x & 7;
  const bool fresh = p >= lo && p < hi;
  const BlockE2m1<D> at(c, block);
  // Words that hold other positions too are read before they are written.
  uint32_t keep = 0, old[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (at.position(e) < lo || at.position(e) >= hi) keep |= 0xfu << (4 * e);
  const bool writes = at.piece >= 0 && keep != ~0u;
  if (writes && keep != 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = at.v[2 * S * i];
  }
  auto largest = [](uint2 w) {
    return max(max(w.x & 0x7fffu, (w.x >> 16) & 0x7fffu), max(w.y & 0x7fffu, (w.y >> 16) & 0x7fffu));
  };
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const uint32_t byte = exponent_byte<kPagedE2m1>(row_amax(largest(kw[j])));
    if (fresh) {
      *reinterpret_cast<uint16_t*>(at.k + 4 * j) =
          static_cast<uint16_t>(quantise4_e2m1(kw[j], byte));
      if (part == 0) at.key_bytes[j] = static_cast<uint8_t>(byte);
    }
    most = max(most, largest(vw[j]));
  }
  const uint32_t byte = exponent_byte<kPagedE2m1>(row_amax(most));
  if (fresh && part == 0) *at.value_byte = static_cast<uint8_t>(byte);
#pragma unroll
  for (int j = 0; j < S; ++j)
    v_s[p][8 * j + part] = static_cast<uint16_t>(quantise4_e2m1(vw[j], byte));
  __syncthreads();
  if (!writes) return;
  uint32_t y[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t x = v_s[at.position(e)][at.piece];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] |= ((x >> (4 * i)) & 0xfu) << (4 * e);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) at.v[2 * S * i] = (y[i] & ~keep) | (old[i] & keep);
}

// The thread's row of a block.
template <int D>
__device__ __forceinline__ void read_e2m1(const PagedCache& c, int64_t block, uint2 (&kw)[D / 32],
                                          uint2 (&vw)[D / 32],
                                          uint16_t (*v_s)[BlockE2m1<D>::kLd]) {
  constexpr int S = D / 32;
  const int p = threadIdx.x >> 3, part = threadIdx.x & 7;
  const BlockE2m1<D> at(c, block);
  if (at.piece >= 0) {
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = at.v[2 * S * i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t x = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) x |= ((y[i] >> (4 * e)) & 0xfu) << (4 * i);
      v_s[at.position(e)][at.piece] = static_cast<uint16_t>(x);
    }
  }
  // (a byte of kPagedNotFinite makes the conversion's results NaN)
  const uint32_t byte = *at.value_byte;
#pragma unroll
  for (int j = 0; j < S; ++j)
    kw[j] = e2m1_bf16x4<0>(*reinterpret_cast<const uint16_t*>(at.k + 4 * j),
                           __uint_as_float(static_cast<uint32_t>(at.key_bytes[j]) << 23));
  __syncthreads();
#pragma unroll
  for (int j = 0; j < S; ++j)
    vw[j] = e2m1_bf16x4<0>(v_s[p][8 * j + part], __uint_as_float(byte << 23));
}

struct Rows {
  const uint16_t* k;
  const uint16_t* v;
  int64_t ks[2], vs[2];  // element strides: row, head
  PagedRope rope;        // (ROPE)
};

// Four values of a row from dimension `dim` on, rotated by the angles of its position.
__device__ __forceinline__ uint2 rotated(uint2 w, const PagedRope& r, int64_t angles, int dim) {
  const float2 c = *reinterpret_cast<const float2*>(r.cos + angles + dim / 2);
  const float2 s = *reinterpret_cast<const float2*>(r.sin + angles + dim / 2);
  const float e0 = lo_bf16(w.x), o0 = hi_bf16(w.x), e1 = lo_bf16(w.y), o1 = hi_bf16(w.y);
  return make_uint2(pack_bf16x2(rope_even(e0, o0, c.x, s.x), rope_odd(e0, o0, c.x, s.x)),
                    pack_bf16x2(rope_even(e1, o1, c.y, s.y), rope_odd(e1, o1, c.y, s.y)));
}

// ROPE: keys, and the query heads that share the kv head, are rotated first.
template <int TYPE, int D, bool ROPE>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedCache c, PagedBatch b,
                                                                Rows rows) {
  using E = typename Stored<TYPE>::type;
  constexpr int S = D / 32;
  constexpr int kLd = D + 16 / sizeof(E);
  __shared__ __attribute__((aligned(16))) E v_s[kPagedBlock][kLd];
  static_assert(2 * BlockE2m1<D>::kLd <= sizeof(E) * kLd, "a block's 4-bit values fit");

  // Blocks that new rows fall into.
  auto units_of = [&](const PagedSequence& s) {
    const int from = max(s.length - s.count, 0), to = ROPE ? s.length : s.stored;
    return to > from ? (to - 1) / kPagedBlock - from / kPagedBlock + 1 : 0;
  };
  int sequence, index;
  PagedSequence s;
  if (!paged_find(b, c.page, blockIdx.x, units_of, sequence, index, s)) return;
  const int from = max(s.length - s.count, 0);
  const int blk = from / kPagedBlock + index;
  const int per_page = c.page / kPagedBlock;
  const int page = blk / per_page < b.width ? paged_page(b, c, sequence, blk / per_page) : -1;
  if (!ROPE && page < 0) return;
  const int head = blockIdx.y;
  const int p = threadIdx.x >> 3, part = threadIdx.x & 7;
  const int position = blk * kPagedBlock + p;
  const int64_t row = s.first + (position - (s.length - s.count));
  int64_t angles = 0;
  if constexpr (ROPE) {
    const PagedRope& r = rows.rope;
    angles = static_cast<int64_t>(min(position, r.positions - 1)) * (D / 2);
    if (position >= from && position < s.length && r.q != nullptr) {
      const int rep = r.heads / c.kv_heads;
      for (int h = head * rep; h < (head + 1) * rep; ++h) {
        const uint16_t* const qr = r.q + row * r.qs[0] + h * r.qs[1] + 4 * part;
        uint16_t* const to = r.out + (row * r.heads + h) * D + 4 * part;
#pragma unroll
        for (int j = 0; j < S; ++j)
          *reinterpret_cast<uint2*>(to + 32 * j) = rotated(
              *reinterpret_cast<const uint2*>(qr + 32 * j), r, angles, 32 * j + 4 * part);
      }
    }
    if (page < 0) return;
  }
  const int64_t at = static_cast<int64_t>(page) * c.kv_heads + head;
  E* const kp = static_cast<E*>(c.key) + (at * per_page + blk % per_page) * (kPagedBlock * D);
  E* const vp = static_cast<E*>(c.value) + (at * per_page + blk % per_page) * (kPagedBlock * D);

  // Rows lo .. hi of the block are new.
  const int lo = max(from - blk * kPagedBlock, 0);
  const int hi = min(s.stored - blk * kPagedBlock, kPagedBlock);
  const bool fresh = p >= lo && p < hi;
  uint2 kw[S], vw[S];
#pragma unroll
  for (int j = 0; j < S; ++j) kw[j] = vw[j] = make_uint2(0, 0);
  if (fresh) {
    const uint16_t* const kr = rows.k + row * rows.ks[0] + head * rows.ks[1] + 4 * part;
    const uint16_t* const vr = rows.v + row * rows.vs[0] + head * rows.vs[1] + 4 * part;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      kw[j] = *reinterpret_cast<const uint2*>(kr + 32 * j);
      vw[j] = *reinterpret_cast<const uint2*>(vr + 32 * j);
    }
    if constexpr (ROPE) {
#pragma unroll
      for (int j = 0; j < S; ++j) kw[j] = rotated(kw[j], rows.rope, angles, 32 * j + 4 * part);
    }
  }
  if constexpr (TYPE == kPagedE2m1) {
    append_e2m1<D>(c, at * per_page + blk % per_page, kw, vw, lo, hi,
                   reinterpret_cast<uint16_t(*)[BlockE2m1<D>::kLd]>(&v_s[0][0]));
    return;
  }
  uint32_t kb = 0, vb = 0;
  if constexpr (TYPE != kPagedBf16) {
    auto largest = [&](const uint2(&w)[S]) {
      uint32_t a = 0;
#pragma unroll
      for (int j = 0; j < S; ++j)
        a = max(max(a, max(w[j].x & 0x7fffu, (w[j].x >> 16) & 0x7fffu)),
                max(w[j].y & 0x7fffu, (w[j].y >> 16) & 0x7fffu));
      return row_amax(a);
    };
    kb = exponent_byte<TYPE>(largest(kw));
    vb = exponent_byte<TYPE>(largest(vw));
    if (fresh && part == 0) {
      const int64_t e = at * c.page + position % c.page;
      c.key_exponent[e] = static_cast<uint8_t>(kb);
      c.value_exponent[e] = static_cast<uint8_t>(vb);
    }
  }
  auto packed = [&](uint2 w, uint32_t byte) {
    const float x[4] = {lo_bf16(w.x), hi_bf16(w.x), lo_bf16(w.y), hi_bf16(w.y)};
    return quantise4<TYPE>(x, byte);
  };
#pragma unroll
  for (int j = 0; j < S; ++j) {
    E* const to = kp + (((p >> 4) * S + j) * 4 + (part >> 1)) * 128 + (p & 15) * 8 + 4 * (part & 1);
    E* const turn = &v_s[p][32 * j + 4 * part];
    if constexpr (TYPE == kPagedBf16) {
      if (fresh) *reinterpret_cast<uint2*>(to) = kw[j];
      *reinterpret_cast<uint2*>(turn) = vw[j];
    } else {
      if (fresh) *reinterpret_cast<uint32_t*>(to) = packed(kw[j], kb);
      *reinterpret_cast<uint32_t*>(turn) = packed(vw[j], vb);
    }
  }
  __syncthreads();
  // Pieces of V: dim w, positions {4 g .. + 3, 16 + 4 g .. + 3}.
  for (int i = threadIdx.x; i < 4 * D; i += kThreads) {
    const int cc = i & 15, g = (i >> 4) & 3, w = (i >> 6) * 16 + cc;
    E* const to = vp + i * 8;
    const int first = 4 * g;
    if (lo <= first && hi >= first + 20) {
      E x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = v_s[(e >> 2) * 16 + first + (e & 3)][w];
      if constexpr (TYPE == kPagedBf16) {
        uint4 y;
        y.x = x[0] | (static_cast<uint32_t>(x[1]) << 16);
        y.y = x[2] | (static_cast<uint32_t>(x[3]) << 16);
        y.z = x[4] | (static_cast<uint32_t>(x[5]) << 16);
        y.w = x[6] | (static_cast<uint32_t>(x[7]) << 16);
        *reinterpret_cast<uint4*>(to) = y;
      } else {
        uint2 y = make_uint2(0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y.x |= static_cast<uint32_t>(x[e]) << (8 * e);
          y.y |= static_cast<uint32_t>(x[4 + e]) << (8 * e);
        }
        *reinterpret_cast<uint2*>(to) = y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int q = (e >> 2) * 16 + first + (e & 3);
        if (q >= lo && q < hi) to[e] = v_s[q][w];
      }
    }
  }
}

struct ReadOut {
  uint16_t* k;
  uint16_t* v;
  int64_t ks[3], vs[3];  // element strides: sequence, head, position
  int positions;
};

template <int TYPE, int D>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedCache c, PagedBatch b,
                                                              ReadOut o) {
  using E = typename Stored<TYPE>::type;
  constexpr int S = D / 32;
  constexpr int kLd = D + 16 / sizeof(E);
  __shared__ __attribute__((aligned(16))) E v_s[kPagedBlock][kLd];
  const int blk = blockIdx.x, head = blockIdx.y, sequence = blockIdx.z;
  const int length = min(max(b.lengths[sequence], 0), b.width * c.page);
  const int per_page = c.page / kPagedBlock;
  int page = -1;
  if (blk * kPagedBlock < length) page = paged_page(b, c, sequence, blk / per_page);
  const int p = threadIdx.x >> 3, part = threadIdx.x & 7;
  const int position = blk * kPagedBlock + p;
  const bool there = page >= 0 && position < length;
  uint2 kw[S], vw[S];
#pragma unroll
  for (int j = 0; j < S; ++j) kw[j] = vw[j] = make_uint2(0, 0);
  if (TYPE == kPagedE2m1 && page >= 0) {
    read_e2m1<D>(c, (static_cast<int64_t>(page) * c.kv_heads + head) * per_page + blk % per_page, kw,
                 vw, reinterpret_cast<uint16_t(*)[BlockE2m1<D>::kLd]>(&v_s[0][0]));
    if (!there) {
#pragma unroll
      for (int j = 0; j < S; ++j) kw[j] = vw[j] = make_uint2(0, 0);
    }
  } else if (page >= 0) {  // (uniform)
    const int64_t at = static_cast<int64_t>(page) * c.kv_heads + head;
    const E* const kp =
        static_cast<const E*>(c.key) + (at * per_page + blk % per_page) * (kPagedBlock * D);
    const E* const vp =
        static_cast<const E*>(c.value) + (at * per_page + blk % per_page) * (kPagedBlock * D);
    for (int i = threadIdx.x; i < 4 * D; i += kThreads) {
      const int cc = i & 15, g = (i >> 4) & 3, w = (i >> 6) * 16 + cc;
      E x[8];
      if constexpr (TYPE == kPagedBf16)
        *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(vp + i * 8);
      else
        *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(vp + i * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) v_s[(e >> 2) * 16 + 4 * g + (e & 3)][w] = x[e];
    }
    uint32_t kb = 0, vb = 0;
    if constexpr (TYPE != kPagedBf16) {
      const int64_t e = at * c.page + position % c.page;
      kb = c.key_exponent[e];
      vb = c.value_exponent[e];
    }
    __syncthreads();
    if (there) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const E* const from =
            kp + (((p >> 4) * S + j) * 4 + (part >> 1)) * 128 + (p & 15) * 8 + 4 * (part & 1);
        const E* const turn = &v_s[p][32 * j + 4 * part];
        if constexpr (TYPE == kPagedBf16) {
          kw[j] = *reinterpret_cast<const uint2*>(from);
          vw[j] = *reinterpret_cast<const uint2*>(turn);
        } else {
          float x[4];
          value4<TYPE>(*reinterpret_cast<const uint32_t*>(from), kb, x);
          kw[j] = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
          value4<TYPE>(*reinterpret_cast<const uint32_t*>(turn), vb, x);
          vw[j] = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
        }
      }
    }
  }
  if (position >= o.positions) return;
  uint16_t* const kr = o.k + sequence * o.ks[0] + head * o.ks[1] + position * o.ks[2] + 4 * part;
  uint16_t* const vr = o.v + sequence * o.vs[0] + head * o.vs[1] + position * o.vs[2] + 4 * part;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    *reinterpret_cast<uint2*>(kr + 32 * j) = kw[j];
    *reinterpret_cast<uint2*>(vr + 32 * j) = vw[j];
  }
}

template <typename F>
hipError_t by_width(int head_dim, F launch) {
  switch (head_dim) {
    case 64: launch(std::integral_constant<int, 64>{}); break;
    case 96: launch(std::integral_constant<int, 96>{}); break;
    case 128: launch(std::integral_constant<int, 128>{}); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

bool paged_head_dim_supported(int head_dim) {
  return head_dim == 64 || head_dim == 96 || head_dim == 128;
}

hipError_t launch_paged_append(const PagedCache& cache, int type, int head_dim,
                               const PagedBatch& batch, const uint16_t* k, const uint16_t* v,
                               const int64_t* k_strides, const int64_t* v_strides,
                               const PagedRope& rope, hipStream_t s) {
  if (batch.rows == 0 || batch.batch == 0) return hipSuccess;
  const Rows rows{k, v, {k_strides[0], k_strides[1]}, {v_strides[0], v_strides[1]}, rope};
  // n rows touch at most (n + 30) / 32 + 1 blocks
  const dim3 grid(batch.rows / kPagedBlock + 2 * std::min(batch.batch, batch.rows), cache.kv_heads);
  auto run = [&](auto t) {
    constexpr int TYPE = decltype(t)::value;
    return by_width(head_dim, [&](auto d) {
      constexpr int D = decltype(d)::value;
      if (rope.cos != nullptr)
        paged_append_kernel<TYPE, D, true><<<grid, kThreads, 0, s>>>(cache, batch, rows);
      else
        paged_append_kernel<TYPE, D, false><<<grid, kThreads, 0, s>>>(cache, batch, rows);
    });
  };
  if (type == kPagedBf16) return run(std::integral_constant<int, kPagedBf16>{});
  if (type == kPagedE4m3) return run(std::integral_constant<int, kPagedE4m3>{});
  if (type == kPagedE2m1) return run(std::integral_constant<int, kPagedE2m1>{});
  return run(std::integral_constant<int, kPagedInt8>{});
}

hipError_t launch_paged_read(const PagedCache& cache, int type, int head_dim,
                             const PagedBatch& batch, int positions, uint16_t* k, uint16_t* v,
                             const int64_t* k_strides, const int64_t* v_strides, hipStream_t s) {
  if (positions == 0 || batch.batch == 0) return hipSuccess;
  const ReadOut out{k, v, {k_strides[0], k_strides[1], k_strides[2]},
                    {v_strides[0], v_strides[1], v_strides[2]}, positions};
  const dim3 grid((positions + kPagedBlock - 1) / kPagedBlock, cache.kv_heads, batch.batch);
  auto run = [&](auto t) {
    constexpr int TYPE = decltype(t)::value;
    return by_width(head_dim, [&](auto d) {
      paged_read_kernel<TYPE, decltype(d)::value><<<grid, kThreads, 0, s>>>(cache, batch, out);
    });
  };
  if (type == kPagedBf16) return run(std::integral_constant<int, kPagedBf16>{});
  if (type == kPagedE4m3) return run(std::integral_constant<int, kPagedE4m3>{});
  if (type == kPagedE2m1) return run(std::integral_constant<int, kPagedE2m1>{});
  return run(std::integral_constant<int, kPagedInt8>{});
}

}  // namespace parrot
