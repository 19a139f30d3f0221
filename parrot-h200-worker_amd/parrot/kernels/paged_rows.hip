// Paged attention of some rows per sequence (chunks of a few tokens): tiles of 32 rows
// on the 32-wide matrix instructions, otherwise as the tiles of 16: every wavefront
// takes every fourth key block of the workgroup's share, its operands straight from
// the pages, the next block's keys loaded once its scores are made and the next values
// once these are added; the four wavefronts are merged in LDS.
//
// What bounds it: the chain of dependent loads at a wavefront's start and end, with two
// to four blocks between, and for 8-bit pages their conversion (some 2.7 instructions
// a value of int8, for 32 rows).  Measured, five chunks of 6 tokens after up to 9000 keys,
// 16 heads on 2 of 128 in int8: 17.2 us for 16 MB and 3.2 to 3.9 for the join; in tiles of 16
// rows (three conversions in place of two) 27.8 in all, of 128 22.7.
#include "paged_attention.h"

namespace parrot {
namespace paged {

namespace {

template <int TYPE, int D>
__global__ __launch_bounds__(kWaves * kWave, 2) void paged_rows_kernel(AttendArgs a) {
  constexpr int KU = D / 16, DT = D / 32;
  using raw = typename Piece<TYPE>::raw;
  // (a wavefront's part takes a block's values before the merge, if any is not finite)
  __shared__ __attribute__((aligned(16))) float o_s[kWaves][kRows][D + 4];
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
  if (begin + wave < end) {
    const int kn = (col >> 3) & 1;
    const int kc = 4 * (2 * (col >> 4) + ((col >> 2) & 1)) + (col & 3);
    const int k_off = (kn * (D / 32) * 512 + half * 128 + kc * 8) / 8;  // in pieces
    const int v_off = ((col >> 4) * 512 + half * 128 + (col & 15) * 8) / 8;
    WaveBlocks at(a, sequence, kvh, blocks, begin, end);
    int block = -1;
    raw k[KU] = {}, v[2 * DT] = {};
    uint32_t kbyte = 0, vbytes[4] = {0, 0, 0, 0};
    auto load_keys = [&] {
      if (block < 0) return;
      const raw* from = static_cast<const raw*>(a.cache.key) +
                        int64_t{block} * (kPagedBlock * D / 8) + k_off;
#pragma unroll
      for (int u = 0; u < KU; ++u) k[u] = from[32 * u];
      if constexpr (TYPE != kPagedBf16)
        kbyte = a.cache.key_exponent[int64_t{block} * kPagedBlock + 16 * kn + kc];
    };
    auto load_values = [&] {
      if (block < 0) return;
      const raw* from = static_cast<const raw*>(a.cache.value) +
                        int64_t{block} * (kPagedBlock * D / 8) + v_off;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[2 * t + h] = from[128 * t + 32 * h];
      if constexpr (TYPE != kPagedBf16) {
        const uint8_t* e = a.cache.value_exponent + int64_t{block} * kPagedBlock + 4 * half;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vbytes[j] = *reinterpret_cast<const uint32_t*>(e + 16 * (j & 1) + 8 * (j >> 1));
      }
    };
    block = at.find(begin + wave);
    load_keys();
    load_values();
    bf16x8 qf[KU];
    {
      const uint16_t* row = a.q + mine.token * a.qs[0] + mine.head * a.qs[1] + 8 * half;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        uint4 w = *reinterpret_cast<const uint4*>(row + 16 * u);
        w.x ^= a.q_sign;
        w.y ^= a.q_sign;
        w.z ^= a.q_sign;
        w.w ^= a.q_sign;
        qf[u] = __builtin_bit_cast(bf16x8, w);
      }
    }
    for (int i = begin + wave; i < end; i += kWaves) {
      const bool more = i + kWaves < end;
      const int k0 = blocks.at(i) * kPagedBlock;
      // (of a block without a page no row sees a key)
      const int stored = block >= 0 ? s.stored : 0;
      f32x16 sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
      const float power = TYPE == kPagedBf16 ? 1.0f : piece_power<TYPE>(kbyte);
#pragma unroll
      for (int u = 0; u < KU; ++u)
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(piece_bf16<TYPE>(k[u], power), qf[u], sc, 0, 0,
                                                     0);
      if (more) {
        block = at.find(i + kWaves);
        load_keys();
      }
      bf16x8 vf[2 * DT];
#pragma unroll
      for (int t = 0; t < 2 * DT; ++t) vf[t] = piece_bf16<TYPE>(v[t], 1.0f);
      uint32_t bytes[4] = {vbytes[0], vbytes[1], vbytes[2], vbytes[3]};
      auto byte_of = [&](int e) { return (bytes[e >> 2] >> (8 * (e & 3))) & 0xffu; };
      uint16_t* const v_s = reinterpret_cast<uint16_t*>(&o_s[wave][0][0]);
      // A block that every row of the tile sees whole needs no mask.
      const bool whole = k0 + 31 <= min(first, stored - 1) &&
                         (last - k0 < a.window || k0 + 31 < a.sinks);
      // Values that some row must not see: times a probability of 0 an infinity or a
      // NaN is not 0.  They are left out and added to the rows that see them.
      bool odd = false;
      if (!whole) {
        odd = mask_block<D>(sc, vf, k0, mine.position, stored, a);
        if constexpr (TYPE != kPagedBf16) {
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 16; ++e) bad |= byte_of(e) == kPagedNotFinite;
          odd |= __ballot(bad) != 0;
        }
        if (odd) {
          if constexpr (TYPE != kPagedBf16) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (byte_of(e) == kPagedNotFinite) {  // (such an int8 row holds zeros)
                bytes[e >> 2] &= ~(0xffu << (8 * (e & 3)));
#pragma unroll
                for (int t = 0; t < DT; ++t)
                  vf[2 * t + (e >> 3)][e & 7] = __builtin_bit_cast(__bf16, uint16_t{0x7fc0});
              }
            }
          }
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<bf16x8*>(v_s + 8 * v_off + 1024 * t + 256 * h) = vf[2 * t + h];
          clear_nonfinite(vf);
        }
      }
      raise(st, largest(sc), a.scale_log2);
      bf16x8 pf[2];
      probabilities(st, sc, a.scale_log2, pf, [&](float p, int e) {
        return TYPE == kPagedBf16 ? p : p * __uint_as_float(byte_of(e) << 23);
      });
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < DT; ++t)
          st.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * t + h], pf[h], st.o[t], 0, 0, 0);
      if (odd) add_nonfinite<D>(st, v_s, k0, mine.position, stored, a);
      if (more) load_values();
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

}  // namespace

hipError_t launch_rows(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s) {
  return by_type_and_width(type, head_dim, [&](auto t, auto d) {
    paged_rows_kernel<decltype(t)::value, decltype(d)::value><<<grid, kWaves * kWave, 0, s>>>(a);
  });
}

}  // namespace paged
}  // namespace parrot
