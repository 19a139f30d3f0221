// Paged attention of many rows per sequence (prompts and their chunks): a wavefront has
// 32 rows, the four of a workgroup share key blocks through LDS.
//
// Each wavefront brings one of a stage's four matrices (K and V of two blocks) from
// the pages while the stage before is computed: bf16 straight into LDS, 8-bit pages
// into registers, from which they are written as bf16, converted once for 128 rows.
// K's second half lies 128 bytes further, so that the 16 lanes of a read's phase, which
// take eight keys of each half, fall into different banks.
//
// What bounds it: a wavefront's chain of LDS reads, products and softmax, some 4340
// clocks a pair of blocks (760 the products, 970 the vector instructions, the rest
// reads, the copies' issue and waits), which three wavefronts a SIMD (2.2 on average)
// overlap in part and whose registers leave no fourth.  So a pair that every row sees whole
// takes one step of the softmax and no mask (4 prompts of 4096, 8 heads on 2 of 96 in
// bf16, window 2048: 114 us without, 102 with), and wavefronts step back for those with
// more left (99).  Measured there 96 us in a trace and 88 to 92 among others, 0.84 to
// 0.88 PFLOP/s of the visible pairs' products; 2 prompts of 4096, 8 heads of 64 in int8, 74 us
// with the join (76 and 6.4 in a trace); 3 chunks of 512 after up to 3500 keys 21.8 and 5.6.
// Not kept: two blocks' scores ahead of the softmax (no change at three workgroups a CU,
// 130 us where registers leave two), workgroups that take a second, short tile (the
// registers leave two a CU), odd shares in reverse order (no change), sums of P by dot
// products of bf16 (eight instructions a block fewer, no change).
#include "attention_lds.h"
#include "paged_attention.h"

namespace parrot {
namespace paged {

namespace {

// A V piece with its positions' powers of two over kUnit (int8: shift = -128 times the power).
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
    const int which = wave >> 1;       // block of a stage, and matrix, that this wavefront brings
    const bool brings_v = wave & 1;
    const char* const matrix = static_cast<const char*>(brings_v ? a.cache.value : a.cache.key);
    // Lane j: which block of the cache the share's j-th is (of the last 64), -1 for none.
    int ids = -1;
    int at0 = -1, at1 = -1;            // of the stage that is brought
    __amdgpu_buffer_rsrc_t from;       // what this wavefront brings of it
    uint4 got[kLoads];                 // 8-bit types
    uint32_t bytes[2] = {0, 0};
    auto aim = [&](int i) {  // at blocks i and i + 1 (past the share: at nothing)
      const int j = (i - begin) % kWave;
      if (j == 0 && i < end) {
        ids = -1;
        if (i + lane < end) ids = cache_block(a, sequence, kvh, blocks.at(i + lane));
      }
      at0 = i < end ? __builtin_amdgcn_readlane(ids, j) : -1;
      at1 = i < end ? __builtin_amdgcn_readlane(ids, j + 1) : -1;
      const int at = which ? at1 : at0;
      from = make_rsrc(matrix + int64_t{max(at, 0)} * (kPagedBlock * D * kBytes),
                       at < 0 ? 0 : kPagedBlock * D * kBytes);
      if constexpr (TYPE != kPagedBf16) {
        if (at < 0) return;
        const int64_t e = int64_t{at} * kPagedBlock;
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
    // Pieces u0 .. u1 - 1 of what was aimed at (zeros for a block without a page).
    auto bring = [&](int u0, int u1, int buf) {
#pragma unroll
      for (int u = u0; u < u1; ++u) {
        if constexpr (TYPE == kPagedBf16)
          buffer_to_lds16(from, &stage[buf][which][brings_v ? kK : 0] + 512 * u +
                                    (!brings_v && u >= S ? kHalf : 0),
                          lane * 16u, 1024u * u);
        else
          got[u] = __builtin_bit_cast(
              uint4, __builtin_amdgcn_raw_buffer_load_b128(from, lane * 16u, 1024u * u, 0));
      }
    };
    auto put = [&](int buf) {  // 8-bit types: what was brought, as bf16
      if constexpr (TYPE != kPagedBf16) {
        if ((which ? at1 : at0) < 0) return;
        uint16_t* const to = &stage[buf][which][brings_v ? kK : 0];
        if (brings_v) {
          float power[8], shift[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            power[e] = piece_power<TYPE>((bytes[e >> 2] >> (8 * (e & 3))) & 0xffu);
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
            p[0] = piece_bf16<TYPE>(make_uint2(got[u].x, got[u].y), piece_power<TYPE>(b & 0xffu));
            p[1] = piece_bf16<TYPE>(make_uint2(got[u].z, got[u].w), piece_power<TYPE>(b >> 8));
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
    // A block's operands.  Before every read of its own the compiler waits for all copies
    // into LDS, the next stage's too, so with bf16 pages the reads and their waits are
    // written out; of 8-bit types it may read early and wait late (84.4 -> 82 us for 2
    // prompts of 4096).
    auto read_k = [&](uint32_t lds, bf16x8(&kf)[KU]) {
      if constexpr (TYPE == kPagedBf16) {
        lds_frags<0, 512>(lds + k_off, kf);
      } else {
        const uint16_t* const from = &stage[0][0][0] + (lds - lds0 + k_off) / 2;
#pragma unroll
        for (int u = 0; u < KU; ++u) kf[u] = *reinterpret_cast<const bf16x8*>(from + 256 * u);
      }
    };
    auto read_v = [&](uint32_t lds, bf16x8(&vf)[2 * DT]) {
      if constexpr (TYPE == kPagedBf16) {
        read_values<0>(lds + v_off, vf);
      } else {
        const uint16_t* const from = &stage[0][0][0] + (lds - lds0 + v_off) / 2;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            vf[2 * t + h] = *reinterpret_cast<const bf16x8*>(from + 1024 * t + 256 * h);
      }
    };
    // True where values that are not finite were left out.
    // (between(n): where a quarter of the next stage is brought)
    auto block = [&](uint32_t lds, int k0, int stored, auto between) -> bool {
      bf16x8 kf[KU], vf[2 * DT], pf[2];
      read_k(lds, kf);
      between(0);
      f32x16 sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
      for (int u = 0; u < KU; ++u)
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u], qf[u], sc, 0, 0, 0);
      if constexpr (TYPE == kPagedBf16) __builtin_amdgcn_sched_barrier(0);
      between(1);
      read_v(lds, vf);
      between(2);
      // A block that every row of the tile sees whole needs no mask.
      const bool whole = k0 + 31 <= min(first, stored - 1) &&
                         (last - k0 < a.window || k0 + 31 < a.sinks);
      // Values that some row must not see: times a probability of 0 an infinity or a
      // NaN is not 0.
      bool odd = false;
      if (!whole) {
        odd = mask_block<D>(sc, vf, k0, mine.position, stored, a);
        if (odd) clear_nonfinite(vf);
      }
      raise(st, largest(sc), a.scale_log2);
      probabilities(st, sc, a.scale_log2, pf, [](float p, int) { return p; });
      between(3);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < DT; ++t)
          st.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * t + h], pf[h], st.o[t], 0, 0, 0);
      return odd;
    };
    // Both blocks of a stage that every row sees whole: one step of the softmax.
    auto both = [&](uint32_t lds, auto between) {
      bf16x8 kf[KU], vf[2 * DT], pf[2];
      f32x16 sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        read_k(lds + 2 * kBlock * b, kf);
        between(2 * b);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[b][e] = 0.0f;
#pragma unroll
        for (int u = 0; u < KU; ++u)
          sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u], qf[u], sc[b], 0, 0, 0);
        if constexpr (TYPE == kPagedBf16) __builtin_amdgcn_sched_barrier(0);
      }
      read_v(lds, vf);
      raise(st, fmaxf(largest(sc[0]), largest(sc[1])), a.scale_log2);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        probabilities(st, sc[b], a.scale_log2, pf, [](float p, int) { return p; });
        between(2 * b + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < DT; ++t)
            st.o[t] =
                __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * t + h], pf[h], st.o[t], 0, 0, 0);
        if (b == 0) {
          if constexpr (TYPE == kPagedBf16) __builtin_amdgcn_sched_barrier(0);
          read_v(lds + 2 * kBlock, vf);
        }
      }
    };
    // The share's blocks that every row of the tile sees whole: from..to - 1.
    const int low = last >= a.window ? (last - a.window) / kPagedBlock + 1 : 0;
    const int whole0 = blocks.sinks + max(low - blocks.lo, 0);
    const int whole1 = min(end, blocks.sinks + (min(first + 1, s.stored)) / kPagedBlock - blocks.lo);
    aim(begin);
    bring(0, kLoads, 0);
    int i = begin, buf = 0;
    // The hardware lets the oldest of equal wavefronts go first, and a CU's last workgroup
    // would be alone at its end.  Those with little left step back for the others, and
    // short ones go first, so that what follows them begins early.
    const int mark1 = 3 * share.most / 8, mark0 = share.most / 6;
    const bool little = end - begin <= 5 * share.most / 8;
    int mark = little ? -1 : mark1;
    if (little) __builtin_amdgcn_s_setprio(3);
    else __builtin_amdgcn_s_setprio(2);
    auto between = [&](int n) { bring(n * kLoads / 4, (n + 1) * kLoads / 4, buf ^ 1); };
    auto next = [&] {  // stage i is there, and i + 2 aimed at
      if constexpr (TYPE == kPagedBf16) {
        // This wavefront's copies have landed; past the barrier everybody's have, and
        // nobody reads the other buffer any more.
        wait_vm_barrier<0>();
      } else {
        put(buf);
        __syncthreads();
      }
      if (end - i <= mark) {
        if (mark == mark0) __builtin_amdgcn_s_setprio(0);
        else __builtin_amdgcn_s_setprio(1);
        mark = mark == mark0 ? -1 : mark0;
      }
      aim(i + 2);
    };
    // Blocks without a page, and those that none of this wavefront's rows sees, are
    // left out (but a stage's first, which brings the next).
    auto seen = [&](int k0) {
      return k0 <= last && (first - (k0 + 31) < a.window || k0 < a.sinks);
    };
    auto easy = [&] { return i >= whole0 && i + 2 <= whole1 && (at0 | at1) >= 0; };
    if (!has) {
#pragma unroll 1
      for (; i < end; i += 2, buf ^= 1) {
        next();
        bring(0, kLoads, buf ^ 1);
      }
    }
    while (i < end) {
#pragma unroll 1
      for (; i < end && !easy(); i += 2, buf ^= 1) {
        const int now1 = at1, stored0 = at0 >= 0 ? s.stored : 0;
        next();
        const uint32_t lds = lds0 + buf * (4 * kBlock);
        const int k0 = blocks.at(i) * kPagedBlock, k1 = blocks.at(i + 1) * kPagedBlock;
        uint32_t odd = block(lds, k0, stored0, between);
        if (now1 >= 0 && seen(k1))
          odd |= 2 * block(lds + 2 * kBlock, k1, s.stored, [](int) {});
#pragma unroll 1
        for (int b = 0; odd != 0; ++b, odd >>= 1)
          if (odd & 1)
            add_nonfinite<D>(st, &stage[buf][b][kK], b ? k1 : k0, mine.position,
                             b ? s.stored : stored0, a);
      }
#pragma unroll 1
      for (; i < end && easy(); i += 2, buf ^= 1) {
        next();
        both(lds0 + buf * (4 * kBlock), between);
      }
    }
    // (the copies of the last step, of nothing, write zeros: not past the workgroup's end)
    if constexpr (TYPE == kPagedBf16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const float l = st.l + __shfl_xor(st.l, 32);
  if (row0 + col >= rows) return;
  const int64_t to = static_cast<int64_t>(mine.token) * a.heads + mine.head;
  if (share.whole) {
    if (a.splits > 1 && half == 0) a.part_ml[to * a.splits] = make_float2(0.0f, kWhole);
    const float f = l == 0.0f ? 0.0f : kUnit<TYPE> / l;
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
              make_float4(st.o[t][e] * kUnit<TYPE>, st.o[t][e + 1] * kUnit<TYPE>,
                          st.o[t][e + 2] * kUnit<TYPE>, st.o[t][e + 3] * kUnit<TYPE>);
    }
  }
}

}  // namespace

hipError_t launch_tiles(const AttendArgs& a, int type, int head_dim, dim3 grid, hipStream_t s) {
  return by_type_and_width(type, head_dim, [&](auto t, auto d) {
    paged_tile_kernel<decltype(t)::value, decltype(d)::value><<<grid, kWaves * kWave, 0, s>>>(a);
  });
}

}  // namespace paged
}  // namespace parrot
