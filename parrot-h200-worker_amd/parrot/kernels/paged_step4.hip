// Paged attention of few rows per sequence over pages of 4 bits: tiles of 16 / G rows, G key
// blocks in one step of a wavefront (G = 4, 2).
//
// A wavefront's time goes with its instructions more than with the pages' bytes (a vector
// instruction of one wavefront takes eight clocks, however few there are on the SIMD), and a
// tile of 16 rows of which a decode step fills four would spend most of them on the other
// twelve columns.  So those columns take other key blocks: column R b + r (R = 16 / G) is
// row r over the step's block b.
//
//   S_b^T = K_b Q^T   for each block, Q's rows repeated over the columns
//                     (v_mfma_f32_16x16x32_bf16), of which columns R b .. are kept: a move
//                     into the banks of four lanes that they are.
//   one softmax of the 128 or 64 keys: eight scores a lane, each column with a maximum and a
//                     sum of its own, raised together in its four lanes
//   O^T += V_b^T P_b^T  for each block, P_b being P with the other columns 0.
//
// At the end the columns of a row are added (in the units of their largest maximum), then
// the wavefronts.  All of a step's blocks are loaded a step ahead, each matrix as soon as the
// registers of the one before are free.
//
// Measured, 8 heads on 2 of 96: 32 sequences in a window of 2048 10.9 us for 12 MB in one launch
// (G = 4: 155 vector instructions a block, tiles of 16 rows 290; a workgroup a CU on a quarter of
// the CUs, since shares and their join take 12.5); 8 sequences of 32000 keys 13.4 us for 51 MB
// (3.8 TB/s) and 3.9 for the join, of 100000 27.4 and 4.1 (160 MB, 5.8 TB/s: the chip's
// memory-side cache holds them); one of 129 keys 4.7.  By the counters of the second a SIMD's
// vector instructions are active for a quarter of the time and the matrix units for 6 %: what
// is left is the launch, the first loads (sequence, table, block: some 4 us), and the last.
// Not kept: 16 wavefronts of two blocks a step (12.0 us for the first).
//
// The stored values are finite whatever a row held (its power of two, which is NaN for byte
// 255, makes the products NaN), so a row that is not seen takes 0 in place of its power and
// cannot reach anything.
#include "paged_attention.h"

namespace parrot {
namespace paged {

namespace {

// Lanes of group b (R of every 16) from `x`, the others from `old`.
template <int R>
__device__ __forceinline__ float group_of(int b, float x, float old) {
  const int xi = __builtin_bit_cast(int, x), oi = __builtin_bit_cast(int, old);
  int y = oi;
  if constexpr (R == 4) {
    if (b == 0) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0x1, false);
    if (b == 1) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0x2, false);
    if (b == 2) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0x4, false);
    if (b == 3) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0x8, false);
  } else {
    static_assert(R == 8, "groups of whole banks");
    if (b == 0) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0x3, false);
    if (b == 1) y = __builtin_amdgcn_update_dpp(oi, xi, 0xe4, 0xf, 0xc, false);
  }
  return __builtin_bit_cast(float, y);
}

// The same value of the column `by` places to the left, around 16.
template <int BY>
__device__ __forceinline__ float rotated(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x),
                                                               0x120 + BY, 0xf, 0xf, false));
}

template <int D, int G, int W>
__global__ __launch_bounds__(W * kWave, W > kWaves ? W / 4 : D < 128 ? 3 : 2)
void paged_step4_kernel(AttendArgs a) {
  constexpr int S = D / 32, T = D / 16, R = kStepRows / G;
  __shared__ __attribute__((aligned(16))) float o_s[W][R][D + 4];
  __shared__ float ml_s[W][2][R];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15, group = col / R, r = col % R;
  const Place place = place_of(a);
  const int kvh = place.kvh, split = place.split;

  auto units_of = [&](const PagedSequence& s) { return (s.count * a.rep + R - 1) / R; };
  int sequence, tile;
  PagedSequence s;
  if (!paged_find(a.batch, a.cache.page, place.tile, units_of, sequence, tile, s)) return;
  const int rows = s.count * a.rep;
  const int row0 = tile * R;
  const TileRow mine = tile_row(s, row0 + r, rows, a.rep, kvh);
  const int first = s.length - s.count + row0 / a.rep;
  const int last = s.length - s.count + (min(row0 + R, rows) - 1) / a.rep;
  const Blocks blocks = tile_blocks(first, last, s.stored, a.window, a.sinks);
  const Share share = split_share(s, rows, R, a.rep, blocks, split, a.splits, a.whole, a.window,
                                  a.sinks);
  if (share.whole && split > 0) return;
  const int begin = share.begin, end = share.end;

  float m = -INFINITY, l = 0.0f;
  f32x4 o[T];
#pragma unroll
  for (int t = 0; t < T; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (begin + wave < end) {
    // The wavefront's blocks are begin + wave + W j; lane i holds where the (64 n + i)-th
    // lies in the cache (-1: nowhere).
    int held = -1;
    int at[G];  // of the step whose blocks are in registers, or on their way
    uint32_t k[G][T], v[G][T], kbytes[G][2], vbytes[2] = {0, 0};
    int there = -1;  // `at` of this lane's group
    auto aim = [&](int j) {
      const int slot = j % kWave;
      if (slot == 0) {
        const int i = begin + wave + W * (j + lane);
        held = i < end ? cache_block(a, sequence, kvh, blocks.at(i)) : -1;
      }
#pragma unroll
      for (int b = 0; b < G; ++b) at[b] = __builtin_amdgcn_readlane(held, slot + b);
      there = __shfl(held, slot + group);
    };
    auto load_keys = [&](int b) {
      if (at[b] < 0) return;
      load_words(static_cast<const uint32_t*>(a.cache.key) + int64_t{at[b]} * (4 * D) + T * lane, k[b]);
      e2m1_key_bytes<D>(a.cache.key_exponent + int64_t{at[b]} * D, col, kbytes[b]);
    };
    auto load_values = [&](int b) {
      if (at[b] < 0) return;
      load_words(static_cast<const uint32_t*>(a.cache.value) + int64_t{at[b]} * (4 * D) + T * lane,
                 v[b]);
    };
    auto load_powers = [&] {
      if (there < 0) return;
      const uint8_t* e = a.cache.value_exponent + int64_t{there} * kPagedBlock + 4 * g;
      vbytes[0] = *reinterpret_cast<const uint32_t*>(e);
      vbytes[1] = *reinterpret_cast<const uint32_t*>(e + 16);
    };
    aim(0);
#pragma unroll
    for (int b = 0; b < G; ++b) load_keys(b);
    load_powers();
#pragma unroll
    for (int b = 0; b < G; ++b) load_values(b);
    bf16x8 qf[S];
    {
      const uint16_t* row = a.q + mine.token * a.qs[0] + mine.head * a.qs[1] + 8 * g;
#pragma unroll
      for (int u = 0; u < S; ++u) {
        uint4 w = *reinterpret_cast<const uint4*>(row + 32 * u);
        w.x ^= a.q_sign;
        w.y ^= a.q_sign;
        w.z ^= a.q_sign;
        w.w ^= a.q_sign;
        qf[u] = __builtin_bit_cast(bf16x8, w);
      }
    }
    // Blocks whole0 .. whole1 - 1 of the tile are seen whole by every row.
    const int low = last >= a.window ? (last - a.window) / kPagedBlock + 1 : 0;
    const int whole0 = blocks.sinks + max(low - blocks.lo, 0);
    const int whole1 =
        min(end, blocks.sinks + min(first + 1, s.stored) / kPagedBlock - blocks.lo);
    const Visible sees = visible_to(mine.position, s.stored, a.window, a.sinks);
    for (int i = begin + wave, j = G; i < end; i += G * W, j += G) {
      // Scores of the step's blocks, each column's of its own block.
      float sc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[e] = -INFINITY;
      int here[G];
      const int of_group = there;
#pragma unroll
      for (int b = 0; b < G; ++b) here[b] = at[b];
      const bool more = i + G * W < end;
      if (more) aim(j);
#pragma unroll
      for (int b = 0; b < G; ++b) {
        if (here[b] >= 0) {
          f32x4 x[2];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            x[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < S; ++u)
              x[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  piece_bf16<kPagedE2m1>(k[b][n * S + u], e2m1_power(kbytes[b], n * S + u)), qf[u],
                  x[n], 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[e] = group_of<R>(b, x[e >> 2][e & 3], sc[e]);
        }
        if (more) load_keys(b);
      }
      float power[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        power[e] = byte_power(vbytes[e >> 2], e & 3);
      if (more) load_powers();
      bool whole = i >= whole0 && i + (G - 1) * W < whole1;
#pragma unroll
      for (int b = 0; b < G; ++b) whole &= here[b] >= 0;
      if (!whole) {
        // (of a block without a page, or past the share, no row sees a key)
        const int mine_i = i + W * group;
        const int k0 = blocks.at(mine_i) * kPagedBlock + 4 * g;
        const bool some = of_group >= 0 && mine_i < end;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool seen = some && sees(k0 + 16 * (e >> 2) + (e & 3));
          sc[e] = seen ? sc[e] : -INFINITY;
          power[e] = seen ? power[e] : 0.0f;
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])),
                       fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
      mx *= a.scale_log2;
      if (__ballot(mx > m + 8.0f) != 0) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][e] *= alpha;
        m = mn;
      }
      const float neg = m == -INFINITY ? 0.0f : -m;
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], a.scale_log2, neg));
      l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      bf16x8 pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = static_cast<__bf16>(p[e] * power[e]);
#pragma unroll
      for (int b = 0; b < G; ++b) {
        if (here[b] >= 0) {
          uint4 w = __builtin_bit_cast(uint4, pf);
          auto of_block = [&](uint32_t x) {
            return __float_as_uint(group_of<R>(b, __uint_as_float(x), 0.0f));
          };
          w = make_uint4(of_block(w.x), of_block(w.y), of_block(w.z), of_block(w.w));
#pragma unroll
          for (int t = 0; t < T; ++t)
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                piece_bf16<kPagedE2m1>(v[b][(t & 1) * S + t / 2], 1.0f),
                __builtin_bit_cast(bf16x8, w), o[t], 0, 0, 0);
        }
        if (more) load_values(b);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // The columns of a row.
  float most = fmaxf(m, rotated<8>(m));
  if constexpr (G == 4) most = fmaxf(most, rotated<4>(most));
  // (one that saw nothing has zeros; a NaN sum has to come through)
  const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - most);
  auto over_groups = [&](float x) {
    x *= f;
    x += rotated<8>(x);
    if constexpr (G == 4) x += rotated<4>(x);
    return x;
  };
  l = over_groups(l);
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const float4 y = make_float4(over_groups(o[t][0]), over_groups(o[t][1]), over_groups(o[t][2]),
                                 over_groups(o[t][3]));
    if (group == 0) *reinterpret_cast<float4*>(&o_s[wave][r][16 * t + 4 * g]) = y;
  }
  if (lane < R) {
    ml_s[wave][0][r] = most;
    ml_s[wave][1][r] = l;
  }
  __syncthreads();
  merge_tile<D, R>(a, o_s, ml_s, s, row0, rows, kvh, split, share);
}

}  // namespace

hipError_t launch_step4(const AttendArgs& a, int head_dim, int tile, bool wide, dim3 grid,
                        hipStream_t s) {
  return by_type_and_width(kPagedE2m1, head_dim, [&](auto, auto d) {
    constexpr int D = decltype(d)::value;
    if (tile == kStepRows / 4)
      paged_step4_kernel<D, 4, kWideWaves><<<grid, kWideWaves * kWave, 0, s>>>(a);
    else if (wide)
      paged_step4_kernel<D, 2, kWideWaves><<<grid, kWideWaves * kWave, 0, s>>>(a);
    else
      paged_step4_kernel<D, 2, kWaves><<<grid, kWaves * kWave, 0, s>>>(a);
  });
}

}  // namespace paged
}  // namespace parrot
