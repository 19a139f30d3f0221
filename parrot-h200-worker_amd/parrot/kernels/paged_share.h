// How paged attention's work is cut: the tiles, the key blocks that a tile's rows see,
// and the shares of them that workgroups take, as plain functions of the sizes.  The
// kernels and their launches go by them, and a host program can walk a whole launch.
#pragma once

#include <algorithm>
#include <cstdint>

#include "extents.h"

namespace parrot {

enum PagedType { kPagedBf16 = 0, kPagedE4m3 = 1, kPagedInt8 = 2 };

constexpr int kPagedBlock = 32;  // positions of a block

struct PagedSequence {
  int first;   // its first new row
  int count;   // new rows
  int length;  // positions, as given
  int stored;  // positions that its pages can hold
};

namespace paged {

constexpr int kWaves = 4;
constexpr int kRows = 32;                  // rows of a wavefront's tile
constexpr int kStepRows = 16;              // rows of a workgroup's tile, few per sequence
constexpr int kTileRows = kWaves * kRows;  // ... many
constexpr int kMaxSplits = 64;             // a lane each in the join

// (by value: with std::min's references the compiler orders the kernels otherwise, 115.6 us
// for 114.9 for 4 prompts of 4096 in e4m3, 8 heads on 2 of 96)
PARROT_EXTENT int lesser(int a, int b) { return a < b ? a : b; }
PARROT_EXTENT int greater(int a, int b) { return a > b ? a : b; }

// The key blocks that a tile's rows see, in order: the first `sinks` blocks,
// then those from `lo` on.
struct Blocks {
  int sinks, lo, count;
  PARROT_EXTENT int at(int i) const { return i < sinks ? i : lo + i - sinks; }
};

PARROT_EXTENT Blocks tile_blocks(int first, int last, int stored, int window, int sinks) {
  Blocks r{0, 0, 0};
  last = lesser(last, stored - 1);
  if (last < 0) return r;
  // (a window past the first position reaches every key; first - window + 1 fits)
  r.lo = first >= window ? lesser((first - window + 1) / kPagedBlock, last / kPagedBlock + 1) : 0;
  // sinks > 0 only count where the window has left them
  r.sinks = lesser(
      static_cast<int>((static_cast<int64_t>(sinks) + kPagedBlock - 1) / kPagedBlock), r.lo);
  r.count = r.sinks + last / kPagedBlock - r.lo + 1;
  return r;
}

// The key blocks of a split: at least kMinShare, as many for each wavefront, and as many
// as `splits` of them need for the tile and for the sequence's last rows; all, where
// those see no more than `whole`.  The last rows see the most without a window, which
// makes shares of one size for a sequence's tiles.  With one, or past the table's end, a
// tile before them may see more (the last may be short: 5 rows of 4 heads in tiles of 16
// see 65, then 64 blocks of a window of 2048), and takes larger shares.  A tile that one
// share covers writes its output itself; its partial sums say so (kWhole).
constexpr int kMinShare = 8;
constexpr float kWhole = -1.0f;  // in place of a sum

struct Share {
  int begin, end;
  bool whole;
  int most;  // key blocks of the longest share of the tile and the sequence's last rows
};

PARROT_EXTENT Share split_share(const PagedSequence& s, int rows, int tile, int rep,
                                const Blocks& blocks, int split, int splits, int whole,
                                int window, int sinks) {
  const int row0 = (rows - 1) / tile * tile;
  const Blocks last = tile_blocks(s.length - s.count + row0 / rep, s.length - 1, s.stored, window,
                                  sinks);
  const int most = greater(last.count, blocks.count);
  if (splits == 1) return {0, blocks.count, true, most};
  const int even = ((most + splits - 1) / splits + kWaves - 1) / kWaves * kWaves;
  const int share = most <= whole ? most : greater(even, kMinShare);
  const int begin = lesser(split * share, blocks.count);
  return {begin, lesser(begin + share, blocks.count), blocks.count <= share,
          lesser(share, most)};
}

struct Plan {
  int tile, splits, whole;
};

// Tiles: of 16 rows where a sequence has no more than 32 on average (most of a larger
// tile would be empty).  Of 32 while there is little to do, four blocks of 32 keys for
// each of the chip's 1024 wavefront schedulers, eight of 8-bit keys: each wavefront
// takes its own, straight from the pages, and none waits for another.  Beyond, of 128,
// which share what they read and convert.  32 / 128 rows, 8 heads on 2 of 96 (us):
//   bf16: 1 sequence of 500 keys, 1024 rows per kv head (1500 blocks) 9.1 / 15.0, 4 of
//   2000, 128 (2000) 12.6 / 14.9, 16 of 1000, 96 (3000) 17.6 / 17.8, 4 of 2000, 256 (4100)
//   21.6 / 20.8, 1 of 4000, 1024 (8500) 28.2 / 27.1, 32 of 4000, 48 (16000) 48.8 / 34.2
//   int8: 4 of 2000, 256 (4100) 21.5 / 23.8, 16 of 1000, 256 (8200) 27.1 / 25.2, 1 of 4000,
//   1024 (8500) 32.4 / 29.9
// Splits, where a tile may see more keys than are faster without the join's launch: 768
// for 16 and 32 rows (one sequence, 8 heads on 2 of 96, one launch / split, us: 512 keys
// 6.0 / 8.4, 768 7.1 / 8.1, 1024 8.2 / 8.3, 1536 10.4 / 8.4; 64 sequences of 8 kv heads of
// 64 in int8 768 17.3 / 18.1, 1024 21.3 / 21.1), and for 128 rows the more the more
// workgroups there are without (16: 384 12.8 / 14.2, 512 15.6 / 14.2; 104: 768 21.4 / 23.0,
// 1024 27.0 / 26.4).  For 16 rows no more workgroups than are resident at once, three a CU
// (8 sequences of 32000 keys 24.5 us, of 1024 workgroups 27.2), each with 256 keys at
// least (384: 24.5 and, of 32 rows with a window, 12.8 for 12.7); for larger tiles about
// 1024, which evens out the causal ones (2 prompts of 4096 92.5 us, of 768 102), each with
// 384 keys (3 chunks of 512 rows after 3500 keys 32.2 us, of 256 keys 35.5, of 512 33.2).
inline Plan plan(int type, int batch, int rows, int heads, int kv_heads, int page, int width,
                 int window, int sinks) {
  const int rep = heads / kv_heads;
  // The most keys a tile can see: its table's, or the window, the sinks and
  // the tile's own span.
  auto keys_of = [&](int tile) {
    const int64_t keys = static_cast<int64_t>(width) * page;
    return window < INT32_MAX ? std::min<int64_t>(keys, int64_t{window} + sinks + tile + 64) : keys;
  };
  const int64_t all = static_cast<int64_t>(rows) * rep, n = std::max(std::min(batch, rows), 1);
  const int64_t work = n * ((all + n * kRows - 1) / (n * kRows)) * kv_heads *
                       ((keys_of(kRows) + kPagedBlock - 1) / kPagedBlock);
  const int tile = all <= 2 * kStepRows * n                          ? kStepRows
                   : work <= (type == kPagedBf16 ? 4096 : 8192) ? kRows
                                                                     : kTileRows;
  const int64_t keys = keys_of(tile);
  const int64_t tiles = (static_cast<int64_t>(rows) * rep + tile - 1) / tile;
  const int64_t units = std::max<int64_t>({tiles, std::min(batch, rows), 1}) * kv_heads;
  const int64_t line = tile == kTileRows ? std::min<int64_t>(384 + 4 * units, 1024) : 768;
  const bool step = tile == kStepRows;
  const int64_t want = step ? std::max<int64_t>(768 / units, 1) : (1024 + units - 1) / units;
  const int64_t least = step ? 256 : 384;
  const int64_t splits =
      keys <= line ? 1 : std::min<int64_t>({want, (keys + least - 1) / least, kMaxSplits});
  return {tile, static_cast<int>(splits), static_cast<int>(line / kPagedBlock)};
}

}  // namespace paged
}  // namespace parrot
