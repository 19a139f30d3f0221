// A paged KV cache: its memory, and how a batch of sequences names its parts.
//
// A page holds `page` positions (a multiple of 32) of every kv head, in blocks
// of 32 positions.  A block of D-wide rows is stored in the order in which the
// attention kernels' matrix operands take it, 32 D elements of K and of V:
//   K: [n = 2][s = D / 32][g = 4][c = 16][8]: position 16 n + c, dims 32 s + 8 g ..
//   V: [t = D / 16][g = 4][c = 16][8]: dim 16 t + c, positions
//      {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3}
// (kfrag_index / vfrag_index within one block), so an operand is one
// contiguous piece of a wavefront's load.
//
// 8-bit rows are q 2^(x - 127), x one byte per position and head: the smallest
// power of two that brings the row's largest magnitude inside the type's range.
// A power of two, because q times one is exact in bf16: what is read back, and
// what attention multiplies, is the stored value itself, not a rounding of it.
// For e4m3, a floating type, the choice costs nothing but the bottom of the
// range; for int8 half a bit on average.  Byte 255: the row held a NaN or an
// infinity and reads back as NaN.
//
// 4-bit values (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) lie eight to a
// word, the first in the lowest bits, in records of D / 16 words, one for each of a
// wavefront's lanes 16 g + c:
//   K: [g = 4][c = 16][n = 2][s = D / 32]: position 16 n + c, dims 32 s + 8 g ..
//   V: [g = 4][c = 16][o = 2][u = D / 32]: dim 32 u + 16 o + c, positions
//      {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3}
// so that a lane's whole part of a block is one or two loads.  Bytes: K has one for 32
// dims (the blocks of the microscaling formats), a block's as [c = 16][n = 2][D / 32], V
// one for a row.  Keys have dims that stand out, which would cost the others of the row
// their bits (of a heavy-tailed row, Student's t of 4, the error is 13.0 % of its norm
// by 32 dims and 15.2 by 96; of a normal one 11.2 and 11.4); of V they are few, and one
// power a position is one factor of its probability.  The power leaves the largest
// magnitude above 3.5 and not above 7, and what is above 6 becomes 6: with 6 and 8 in
// place of 7 the error of a normal row is 11.5 and 11.4 % in place of 11.2.
#pragma once

#include "common.h"
#include "paged_share.h"

namespace parrot {

constexpr int kPagedMinExponent = -100;
constexpr uint32_t kPagedNotFinite = 255;

struct PagedCache {
  void* key;               // [pages, kv_heads, page / 32, 32 D] (4 bits: two to a byte)
  void* value;
  uint8_t* key_exponent;   // [pages, kv_heads, page] (8-bit types), [.., page / 32, D] (4 bits)
  uint8_t* value_exponent;
  int64_t pages;
  int page, kv_heads;
};

// Pages that sequences share out among themselves: those with a use of 0 or less are free.
struct PagedPool {
  int32_t* uses;  // [pages]
  int64_t pages;
  int page;
};

// Sequence i: its pages table[i, :width], its whole length lengths[i] (new
// rows included), its new rows starts[i] .. starts[i + 1] of `rows`.
struct PagedBatch {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  int batch, width, rows;
};

// Rotation of keys, and of query rows (q may be null), by their positions' angles
// (those past the tables by the last).  cos null: none.
struct PagedRope {
  const float* cos;  // [positions, D / 2]
  const float* sin;
  int positions, heads;
  const uint16_t* q;
  int64_t qs[2];  // element strides: row, head
  uint16_t* out;  // [rows, heads, D]
};

// Every number of it is bounded here: whatever the device tensors hold, rows
// stay inside the operands and positions inside the table.
__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& b, int page, int i) {
  PagedSequence s;
  s.first = min(max(b.starts[i], 0), b.rows);
  s.count = min(max(b.starts[i + 1], s.first), b.rows) - s.first;
  s.length = max(b.lengths[i], 0);
  s.stored = min(s.length, b.width * page);  // width * page < 2^31, checked on the host
  return s;
}

// The units (tiles, blocks) of the sequences in a row: which sequence unit `unit`
// belongs to, the how manieth of it it is, and the sequence; false past the last.
// Every lane of a wavefront calls it.  units_of(s): sequence s's number.
template <typename F>
__device__ __forceinline__ bool paged_find(const PagedBatch& b, int page, int unit, F units_of,
                                           int& sequence, int& index, PagedSequence& s) {
  const int lane = threadIdx.x & (kWave - 1);
  int base = 0;
  for (int c = 0; c < b.batch; c += kWave) {
    const PagedSequence mine = paged_sequence(b, page, min(c + lane, b.batch - 1));
    const int units = c + lane < b.batch ? units_of(mine) : 0;
    int upto = units;  // sums by DPP: 1, 2, 4, 8 to the right in rows of 16, then across
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x142, 0xa, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x143, 0xc, 0xf, false);
    const int total = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (unit < base + total) {
      const uint64_t hit = __ballot(unit >= base + upto - units && unit < base + upto);
      const int who = __builtin_ctzll(hit);
      sequence = c + who;
      index = unit - base - __builtin_amdgcn_readlane(upto - units, who);
      s.first = __builtin_amdgcn_readlane(mine.first, who);
      s.count = __builtin_amdgcn_readlane(mine.count, who);
      s.length = __builtin_amdgcn_readlane(mine.length, who);
      s.stored = __builtin_amdgcn_readlane(mine.stored, who);
      return true;
    }
    base += total;
  }
  return false;
}

// As paged_find with the units of all sequences in rounds: the last unit of each
// (which sees the most keys), then the last but one, and so on, so that a grid's
// longest workgroups begin first and its shortest end it.
template <typename F>
__device__ __forceinline__ bool paged_find_last(const PagedBatch& b, int page, int unit, F units_of,
                                                int& sequence, int& index, PagedSequence& s) {
  const int lane = threadIdx.x & (kWave - 1);
  auto sum = [](int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return __builtin_amdgcn_readlane(v, kWave - 1);
  };
  auto units_at = [&](int c, PagedSequence& mine) {
    mine = paged_sequence(b, page, min(c + lane, b.batch - 1));
    return c + lane < b.batch ? units_of(mine) : 0;
  };
  PagedSequence mine;
  int units = units_at(0, mine);
  auto first_rounds = [&](int rounds) {  // units of that many rounds
    int all = sum(min(units, rounds));
    for (int c = kWave; c < b.batch; c += kWave) {
      PagedSequence other;
      all += sum(min(units_at(c, other), rounds));
    }
    return all;
  };
  // The round: the largest number of rounds that lie before the unit.
  int low = 0, high = unit + 1;  // first_rounds(low) <= unit; a round has one unit at least
  if (first_rounds(high) <= unit) return false;
  while (high - low > 1) {
    const int mid = low + (high - low) / 2;
    if (first_rounds(mid) <= unit) low = mid;
    else high = mid;
  }
  int left = unit - first_rounds(low);
  for (int c = 0; c < b.batch; c += kWave) {
    if (c > 0) units = units_at(c, mine);
    uint64_t who = __ballot(units > low);
    const int n = __popcll(who);
    if (left < n) {
      for (; left > 0; --left) who &= who - 1;
      const int at = __builtin_ctzll(who);
      sequence = c + at;
      index = __builtin_amdgcn_readlane(units, at) - 1 - low;
      s.first = __builtin_amdgcn_readlane(mine.first, at);
      s.count = __builtin_amdgcn_readlane(mine.count, at);
      s.length = __builtin_amdgcn_readlane(mine.length, at);
      s.stored = __builtin_amdgcn_readlane(mine.stored, at);
      return true;
    }
    left -= n;
  }
  return false;
}

// Four-bit keys: the powers' bytes of positions c and 16 + c, D / 32 each, in memory's order
// (what is above them is anything).  Words as they are loaded: whoever puts them together
// here waits for them here.
template <int D>
__device__ __forceinline__ void e2m1_key_bytes(const uint8_t* bytes, int c, uint32_t (&to)[2]) {
  if constexpr (D == 64) {
    to[0] = *reinterpret_cast<const uint32_t*>(bytes + 4 * c);
  } else if constexpr (D == 96) {
    struct __attribute__((packed, aligned(2))) Word {
      uint32_t w;
    };
    to[0] = reinterpret_cast<const Word*>(bytes + 6 * c)->w;
    to[1] = *reinterpret_cast<const uint16_t*>(bytes + 6 * c + 4);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(bytes + 8 * c);
    to[0] = w.x;
    to[1] = w.y;
  }
}

// 2^(byte i - 127) as the conversions of 4-bit values take it: they read the eight bits of
// the exponent (255: NaN) and no others.
__device__ __forceinline__ float e2m1_power(const uint32_t (&bytes)[2], int i) {
  const uint32_t w = bytes[i / 4];
  return __uint_as_float(i % 4 < 3 ? w << (23 - 8 * (i % 4)) : w >> 1);
}

// The bytes of a 4-bit key's N groups, as words that are used as they come (e2m1_key_bytes).
template <int N>
__device__ __forceinline__ void load_row_bytes(const uint8_t* from, uint32_t (&to)[2]) {
  if constexpr (N == 4) {
    to[0] = *reinterpret_cast<const uint32_t*>(from);
  } else {
    struct __attribute__((packed, aligned(1))) Two {
      uint16_t w;
    };
    to[0] = reinterpret_cast<const Two*>(from)->w;
    if constexpr (N == 3) to[1] = from[2];
  }
}

template <int N>
__device__ __forceinline__ float row_power(const uint32_t (&bytes)[2], int i) {
  return e2m1_power(bytes, N == 3 && i == 2 ? 4 : i);
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// Bytes 0 and 1, or 2 and 3, of a word of 4-bit values times a power, as bf16 (exact).
template <int HALF>
__device__ __forceinline__ uint2 e2m1_bf16x4(uint32_t w, float power) {
  return make_uint2(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 2 * HALF)),
      __builtin_bit_cast(uint32_t,
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 2 * HALF + 1)));
}

// The page of a position's block, or -1 where the table names none.
__device__ __forceinline__ int paged_page(const PagedBatch& b, const PagedCache& c, int sequence,
                                          int at) {
  const int p = b.table[static_cast<int64_t>(sequence) * b.width + at];
  return p >= 0 && p < c.pages ? p : -1;
}

// Host side: launchers (shapes are validated by the C-ABI layer).
bool paged_head_dim_supported(int head_dim);  // 64, 96, 128
hipError_t launch_paged_append(const PagedCache& cache, int type, int head_dim,
                               const PagedBatch& batch, const uint16_t* k, const uint16_t* v,
                               const int64_t* k_strides, const int64_t* v_strides,
                               const PagedRope& rope, hipStream_t s);
hipError_t launch_paged_read(const PagedCache& cache, int type, int head_dim,
                             const PagedBatch& batch, int positions, uint16_t* k, uint16_t* v,
                             const int64_t* k_strides, const int64_t* v_strides, hipStream_t s);
size_t paged_extend_workspace_bytes(int64_t pages, int batch, int rows);
hipError_t launch_paged_extend(const PagedPool& pool, const PagedBatch& batch, const int32_t* fresh,
                               int64_t* slots, int32_t* positions, void* workspace, hipStream_t s);
hipError_t launch_paged_release(const PagedPool& pool, const PagedBatch& batch, const int32_t* to,
                                int window, int sinks, hipStream_t s);
int paged_attention_splits(int type, int batch, int rows, int heads, int kv_heads, int page,
                           int width, int window, int sinks);
size_t paged_attention_workspace_bytes(int splits, int rows, int heads, int head_dim);
hipError_t launch_paged_attention(const PagedCache& cache, int type, int head_dim,
                                  const PagedBatch& batch, const uint16_t* q,
                                  const int64_t* q_strides, int heads, int window, int sinks,
                                  float scale, void* workspace, uint16_t* out, hipStream_t s);

}  // namespace parrot
