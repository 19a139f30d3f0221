// The launches of paged attention by its plan (paged_share.h), and the join of what the
// workgroups found that a tile's keys were split over.
#include <algorithm>

#include "paged_attention.h"

namespace parrot {

using namespace paged;

namespace {

// A share's part in the joined row: in units of the largest maximum; -1 where it saw
// nothing (a NaN sum has to come through).
__device__ __forceinline__ float share_weight(float2 ml, float m) {
  if (ml.x == -INFINITY) return ml.y == 0.0f ? -1.0f : 1.0f;
  return __builtin_amdgcn_exp2f(ml.x - m);
}

// Rows of no sequence, and those that one share wrote whole, stay as they are.
__device__ __forceinline__ bool joined_already(const AttendArgs& a, int to) {
  const int token = to / a.heads;
  return (token < a.batch.starts[0]) | (token >= a.batch.starts[a.batch.batch]) |
         (a.part_ml[static_cast<int64_t>(to) * a.splits].y == kWhole);
}

// Joins the shares of split tiles where there are many rows: D / 4 threads a row, eight
// shares in flight (of a share that saw nothing the memory may hold anything).
template <int D>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(AttendArgs a) {
  constexpr int kPer = 256 / (D / 4), kAhead = 8;
  const int slot = threadIdx.x / (D / 4), at = threadIdx.x - slot * (D / 4);
  const int to = static_cast<int>(blockIdx.x) * kPer + slot;  // rows * heads fit 30 bits
  if (slot >= kPer || to >= a.batch.rows * a.heads) return;
  const float2* const ml = a.part_ml + static_cast<int64_t>(to) * a.splits;
  const float4* const part =
      reinterpret_cast<const float4*>(a.part) + static_cast<int64_t>(to) * a.splits * (D / 4) + at;
  // (of few shares many rows are whole: 2 prompts of 4096 in int8 81.9 us, asked late 82.8;
  // of six, 3 chunks of 512 rows 30.4 us asked first, late 27.8)
  const bool late = a.splits >= 4;
  if (!late && joined_already(a, to)) return;
  float m = -INFINITY, sum = 0.0f;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c = 0; c < a.splits; c += kAhead) {
    float2 w[kAhead];
    float4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      w[i] = make_float2(-INFINITY, 0.0f);
      if (c + i >= a.splits) continue;  // (the same for all)
      w[i] = ml[c + i];
      x[i] = part[(c + i) * (D / 4)];
    }
    if (late && c == 0 && joined_already(a, to)) return;
    float most = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) most = fmaxf(most, w[i].x);
    // (what came before, in the units of the larger maximum)
    const float back = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - most);
    m = most;
    sum *= back;
    y = make_float4(y.x * back, y.y * back, y.z * back, y.w * back);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float f = share_weight(w[i], m);
      const bool counts = !(f < 0.0f);
      sum += counts ? w[i].y * f : 0.0f;
      y.x += counts ? x[i].x * f : 0.0f;
      y.y += counts ? x[i].y * f : 0.0f;
      y.z += counts ? x[i].z * f : 0.0f;
      y.w += counts ? x[i].w * f : 0.0f;
    }
  }
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(to) * D + 4 * at) =
      make_uint2(pack_bf16x2(y.x * f, y.y * f), pack_bf16x2(y.z * f, y.w * f));
}

// ... and where there are few: a workgroup a row, one share a lane for their weights,
// then D / 4 threads for every tenth share (D = 96).
template <int D>
__global__ __launch_bounds__(256) void paged_join_shares_kernel(AttendArgs a) {
  constexpr int kGroups = 256 / (D / 4);
  __shared__ float w_s[kMaxSplits];
  __shared__ float4 y_s[kGroups][D / 4];
  const int to = blockIdx.x;
  const int group = threadIdx.x / (D / 4), at = threadIdx.x - group * (D / 4);
  const float4* const part =
      reinterpret_cast<const float4*>(a.part) + static_cast<int64_t>(to) * a.splits * (D / 4) + at;
  constexpr int kMine = (kMaxSplits + kGroups - 1) / kGroups;
  float4 x[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k)
    if (group + k * kGroups < a.splits) x[k] = part[(group + k * kGroups) * (D / 4)];
  if (joined_already(a, to)) return;
  if (threadIdx.x < kWave) {
    const int i = threadIdx.x;
    const float2 ml = i < a.splits ? a.part_ml[static_cast<int64_t>(to) * a.splits + i]
                                   : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float f = share_weight(ml, m);
    const float sum = wave_sum(f < 0.0f ? 0.0f : ml.y * f);
    w_s[i] = f < 0.0f ? -1.0f : sum == 0.0f ? 0.0f : f / sum;
  }
  __syncthreads();
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (group < kGroups) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      if (group + k * kGroups >= a.splits) continue;
      const float f = w_s[group + k * kGroups];
      if (f < 0.0f) continue;
      y.x += x[k].x * f;
      y.y += x[k].y * f;
      y.z += x[k].z * f;
      y.w += x[k].w * f;
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
  *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(to) * D + 4 * at) =
      make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

}  // namespace

int paged_attention_splits(int type, int batch, int rows, int heads, int kv_heads, int page,
                           int width, int window, int sinks) {
  return plan(type, batch, rows, heads, kv_heads, page, width, window, sinks).splits;
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
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f *
                 (type == kPagedInt8 ? kUnit<kPagedInt8> : 1.0f);
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.out = out;
  const Plan p = plan(type, batch.batch, batch.rows, heads, cache.kv_heads, cache.page, batch.width,
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
  const hipError_t e = tile == kStepRows ? launch_step(a, type, head_dim, grid, s)
                       : tile == kRows  ? launch_rows(a, type, head_dim, grid, s)
                                        : launch_tiles(a, type, head_dim, tile_grid, s);
  if (e != hipSuccess || splits == 1) return e;
  return by_type_and_width(type, head_dim, [&](auto, auto d) {
    constexpr int D = decltype(d)::value, kPer = 256 / (D / 4);
    const uint32_t rows = static_cast<uint32_t>(batch.rows * heads);
    // (by rows / by shares, in all: 1024 rows after 30000 keys in 64 shares 52.7 / 49.9 us,
    // 4096 in 16 109.4 / 112.1; the join of 12288 rows in 6 8.4 / 13.2)
    if (rows < 2048 || splits >= 32) paged_join_shares_kernel<D><<<rows, 256, 0, s>>>(a);
    else paged_join_rows_kernel<D><<<(rows + kPer - 1) / kPer, 256, 0, s>>>(a);
  });
}

}  // namespace parrot
