// Paged attention of few rows per sequence (decode steps, short chunks): tiles of 16 rows.
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
//
// Measured, 8 heads on 2 of 96 in e4m3: 8 sequences of 32000 keys 19.6 us for 99 MB
// (5.1 TB/s, what a large copy reaches) and 3.9 for the join of 42 shares; 32 sequences
// in a window of 2048 8.3 us for 23 MB and 3.9; one sequence of 129 keys in bf16 4.6 us.  Not
// kept: registers of two blocks at a time (33 us for the first), four workgroups a CU
// (the registers spill).
//
// Of 4-bit pages (9 to 96 rows a sequence; paged_step4.hip has fewer) a block is a quarter of
// the registers, and two are on their way ahead of the one in hand.  Measured, join included, two
// / one: 8 sequences of 32 rows after 32000 keys, 8 heads on 2 of 96, 24.4 / 25.1 us, 5 of 96 rows after
// 9000, 16 heads on 2 of 128, 19.8 / 20.1, 5 ragged of 48 14.7 / 15.0, 8 of 32 after 16000 20.6 / 20.5, but
// 64 of 20 after 4096, 8 heads on 2 of 96, 26.9 / 25.2.  5 sequences of 48 rows over up to 9000 keys, 16 heads on 2 of 128: 12.4
// us at three blocks a wavefront, and the join 4.0.
#include "paged_attention.h"

namespace parrot {
namespace paged {

namespace {

template <int TYPE, int D>
struct StepBlock {
  using raw = typename Piece<TYPE>::raw;
  static constexpr int N = D / 16;  // pieces of K, and of V, per lane
  raw k[N], v[N];
  uint32_t kbytes[2], vbytes[2];  // exponents of the lane's key rows (4 bits: 2 S bytes); of its
                                  // 8 scores
  int at;                         // which block of the cache; -1: none
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
    const float power = TYPE == kPagedBf16 || TYPE == kPagedE2m1 ? 1.0f
                                                                 : piece_power<TYPE>(b.kbytes[n]);
#pragma unroll
    for (int s = 0; s < S; ++s)
      sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          piece_bf16<TYPE>(b.k[n * S + s], TYPE == kPagedE2m1 ? e2m1_power(b.kbytes, n * S + s) : power),
          qf[s], sc[n], 0, 0, 0);
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
  for (int t = 0; t < T; ++t)  // (a record's words of 4 bits: dims 32 u + 16 o)
    vf[t] = piece_bf16<TYPE>(b.v[TYPE == kPagedE2m1 ? (t & 1) * S + t / 2 : t], 1.0f);
  uint32_t bytes[2] = {b.vbytes[0], b.vbytes[1]};
  auto byte_of = [&](int e) { return (bytes[e >> 2] >> (8 * (e & 3))) & 0xffu; };
  // Values that some row must not see: times a probability of 0 an infinity or a NaN
  // is not 0.  They are left out and added to the rows that see them.
  // (4-bit values are finite themselves: a power of 0 is enough)
  bool odd = false;
  if (TYPE == kPagedE2m1 && !whole) {
    const Visible sees = visible_to(query, stored, a.window, a.sinks);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!sees(key_of(e))) bytes[e >> 2] &= ~(0xffu << (8 * (e & 3)));
  } else if (!whole) {
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
          if (byte_of(e) == kPagedNotFinite) {  // (whatever values such a row holds)
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
    const float y = TYPE == kPagedBf16 ? p[e] : p[e] * byte_power(bytes[e >> 2], e & 3);
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
  const Place place = place_of(a);
  const int kvh = place.kvh, split = place.split;

  auto units_of = [&](const PagedSequence& s) {
    return (s.count * a.rep + kStepRows - 1) / kStepRows;
  };
  int sequence, tile;
  PagedSequence s;
  if (!paged_find(a.batch, a.cache.page, place.tile, units_of, sequence, tile, s)) return;
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
    WaveBlocks at(a, sequence, kvh, blocks, begin, end);
    constexpr int kAhead = TYPE == kPagedE2m1 ? 2 : 1;
    StepBlock<TYPE, D> ahead[kAhead] = {};
    auto load = [&](int at, const void* pages, const uint8_t* exponents, raw(&to)[T],
                    uint32_t(&bytes)[2], auto key) {
      if (at < 0) return;
      const raw* from = static_cast<const raw*>(pages) + int64_t{at} * (kPagedBlock * D / 8);
      if constexpr (TYPE == kPagedE2m1) {
        load_words(from + T * lane, to);
      } else {
#pragma unroll
        for (int u = 0; u < T; ++u) to[u] = from[kWave * u + lane];
      }
      if constexpr (TYPE == kPagedE2m1 && decltype(key)::value) {
        e2m1_key_bytes<D>(exponents + int64_t{at} * D, col, bytes);
      } else if constexpr (TYPE != kPagedBf16) {
        const uint8_t* e = exponents + int64_t{at} * kPagedBlock;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if constexpr (decltype(key)::value) bytes[n] = e[16 * n + col];
          else bytes[n] = *reinterpret_cast<const uint32_t*>(e + 16 * n + 4 * g);
        }
      }
    };
    auto load_keys = [&](StepBlock<TYPE, D>& b) {
      load(b.at, a.cache.key, a.cache.key_exponent, b.k, b.kbytes, std::true_type{});
    };
    auto load_values = [&](StepBlock<TYPE, D>& b) {
      load(b.at, a.cache.value, a.cache.value_exponent, b.v, b.vbytes, std::false_type{});
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (begin + wave + u * kWaves >= end) break;
      ahead[u].at = at.find(begin + wave + u * kWaves);
      load_keys(ahead[u]);
      load_values(ahead[u]);
    }
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
    for (int i0 = begin + wave; i0 < end; i0 += kAhead * kWaves) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kWaves;
        if (i >= end) break;
        StepBlock<TYPE, D>& b = ahead[u];
        const bool more = i + kAhead * kWaves < end;
        // (of a block without a page no row sees a key)
        step_block<TYPE, D>(st, b, qf, blocks.at(i) * kPagedBlock, mine.position, first, last,
                            b.at >= 0 ? s.stored : 0, a,
                            reinterpret_cast<uint16_t*>(&o_s[wave][0][0]), [&] {
                              if (!more) return;
                              b.at = at.find(i + kAhead * kWaves);
                              load_keys(b);
                            });
        if (more) load_values(b);
      }
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

}  // namespace

hipError_t launch_step(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s) {
  return by_type_and_width(type, head_dim, [&](auto t, auto d) {
    paged_step_kernel<decltype(t)::value, decltype(d)::value><<<grid, kWaves * kWave, 0, s>>>(a);
  });
}

}  // namespace paged
}  // namespace parrot
