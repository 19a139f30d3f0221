// How paged attention's work is cut: the tiles, the key blocks that a tile's rows see,
// and the shares of them that workgroups take, as plain functions of the sizes.  The
// kernels and their launches go by them, and a host program can walk a whole launch.
#pragma once

#include <algorithm>
#include <cstdint>

#include "extents.h"

namespace parrot {

enum PagedType { kPagedBf16 = 0, kPagedE4m3 = 1, kPagedInt8 = 2, kPagedE2m1 = 4 };

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
constexpr int kWideWaves = 8;

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

PARROT_EXTENT int even_share(int blocks, int splits) {
  return greater(((blocks + splits - 1) / splits + kWaves - 1) / kWaves * kWaves, kMinShare);
}

PARROT_EXTENT Share split_share(const PagedSequence& s, int rows, int tile, int rep,
                                const Blocks& blocks, int split, int splits, int whole,
                                int window, int sinks) {
  const int row0 = (rows - 1) / tile * tile;
  const Blocks last = tile_blocks(s.length - s.count + row0 / rep, s.length - 1, s.stored, window,
                                  sinks);
  const int most = greater(last.count, blocks.count);
  if (splits == 1) return {0, blocks.count, true, most};
  const int share = most <= whole ? most : even_share(most, splits);
  const int begin = lesser(split * share, blocks.count);
  return {begin, lesser(begin + share, blocks.count), blocks.count <= share,
          lesser(share, most)};
}

struct Plan {
  int tile, splits, whole;
  bool wide;  // workgroups of kWideWaves wavefronts (tiles of fewer than 16 rows)
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
// Of 4-bit pages: tiles of 8 rows where a sequence has no more than 8 on average (two key
// blocks a step, paged_step4.hip), and workgroups of eight wavefronts, with four blocks a step
// for up to 4 rows, where one of them is as fast as the split and its join (us, 8 heads on 2 of
// 96, one wide / split: 1 sequence of 1536 keys 9.1 / 9.4; 16 of 2048 10.8 / 10.8; 32 of 2048
// 10.9 / 12.5, 4096 15.6 / 14.9; 64 of 4096 15.9 / 20.4, 8000 27.5 / 26.5; 128 of 16000 76 / 82;
// 16 heads on 2 of 128: 4 of 1024 8.6 / 9.6, 2048 11.6 / 9.8, 32 of 2048 12.0 / 13.0).  One fills
// a CU, so from three quarters of the CUs on the question is how full their last round is (to
// 8192 keys: a table so wide may hold one sequence as long and many short ones).  Short
// sequences leave most of its wavefronts nothing (512 of 129 keys 22.4 us, by four 12.1).
// Splits are as wide where each CU's one has 512 keys or more and few are left over (join
// included, wide / four wavefronts: 8 sequences of 4000 keys 10.2 / 9.3, 8000 10.3 / 10.6, 16000
// 12.9 / 15.6, 32000 17.1 / 18.5, 64000 24.4 / 25.8; 32 of 16000 24.3 / 26.3, 48, which leave 64
// CUs none, 34.4 / 32.2; 1 of 8000 9.8 / 9.0; 16 heads on 2 of 128: 4 of 8000 10.9 / 9.9, of 20000
// 12.6 / 14.7).  Tiles of 16 rows up to 96 on average: their registers are two blocks ahead, and
// the third conversion of what two larger tiles convert twice costs less than the rows that
// those leave empty (5 sequences of 9000 keys, 48 rows, 16 heads on 2 of 128 18.3 / 22.8 in tiles
// of 32; 5 x 96 rows 21.1 / 23.8, of 128; 2 x 128 rows after 4000 15.0 / 13.3).
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
  const bool few = type == kPagedE2m1 && all <= kStepRows / 2 * n;
  if (few) {
    const bool fewer = all <= kStepRows / 4 * n;
    const int tile = fewer ? kStepRows / 4 : kStepRows / 2;
    const int64_t keys = keys_of(tile), tiles = std::max<int64_t>((all + tile - 1) / tile, n);
    const int64_t units = tiles * kv_heads, rounds = (units + 255) / 256;
    const int64_t most = (fewer ? 2176 : 1152) + 16 * units;
    if (keys > 768 && units < 768 &&
        (units < 192 ? keys <= most : 4 * units >= 768 * rounds && keys <= 8192))
      return {tile, 1, static_cast<int>(keys / kPagedBlock + 1), true};
  }
  const int tile = few                                                   ? kStepRows / 2
                   : all <= (type == kPagedE2m1 ? 6 : 2) * kStepRows * n ? kStepRows
                   : work <= (type == kPagedBf16 ? 4096 : 8192) ? kRows
                                                                     : kTileRows;
  const int64_t keys = keys_of(tile);
  const int64_t tiles = (static_cast<int64_t>(rows) * rep + tile - 1) / tile;
  const int64_t units = std::max<int64_t>({tiles, std::min(batch, rows), 1}) * kv_heads;
  const int64_t line = tile == kTileRows ? std::min<int64_t>(384 + 4 * units, 1024) : 768;
  const bool step = tile <= kStepRows;
  const bool wide = few && units <= 64 && keys * units >= 1 << 17;
  const int64_t want = wide   ? 256 / units
                       : step ? std::max<int64_t>(768 / units, 1)
                              : (1024 + units - 1) / units;
  const int64_t least = wide ? 512 : step ? 256 : 384;
  const int64_t splits =
      keys <= line ? 1 : std::min<int64_t>({want, (keys + least - 1) / least, kMaxSplits});
  return {tile, static_cast<int>(splits), static_cast<int>(line / kPagedBlock), wide};
}

// Workgroups for the tiles of all sequences, ceil(n rep / tile) for one of n rows: no more
// than one each besides those that all rows fill, and no more than those of each row alone
// (those without a tile end at once, but take room until they do: 8 sequences of 32000 keys by
// eight empty ones beside eight 21.6 us, without 15.9).
inline int64_t grid_tiles(int rows, int batch, int rep, int tile) {
  return std::min(static_cast<int64_t>(rows) * rep / tile + std::min(batch, rows),
                  static_cast<int64_t>(rows) * ((rep + tile - 1) / tile));
}

// A tile, kv head and share.
struct Place {
  int tile, kvh, split;
};

// Workgroup x of a line: the shares fastest, then the kv heads, the tiles slowest.
PARROT_EXTENT Place line_place(int x, int kv_heads, int splits) {
  const int t = x / splits, tile = t / kv_heads;
  return {tile, t - tile * kv_heads, x - t * splits};
}

// Whether the workgroups lie in a line, in place of a grid with the tiles fastest and the
// shares slowest.  Workgroups go to the eight XCDs in turn, so where a tile has a multiple of
// eight of them, the same share of a sequence's tiles is on one XCD, whose L2 then has the keys
// for the second; and those without a tile come last, in place of taking the room of others.
// For batches of several rows a sequence, of 8 and 16 bits more than one tile's (us, grid / line;
// 8 kv heads of 64, or 8 or 16 heads on 2 of 96 or 128):
//              16 x 5 rows   64 x 5 in a   8 x 4 after   2 x 60 after  16 x 24 after  16 x 6 after
//              after 2000    window of     16000 of 128  3000 of 64    4000 of 64     9000 of 128
//                            3000
//     bf16     16.0 / 11.5   49.1 / 29.1   46.4 / 34.7   11.6 / 10.2   43.6 / 26.8    (128 rows a tile)
//     e4m3     13.0 / 11.2   31.7 / 24.9   28.5 / 23.0   12.3 / 10.6   26.9 / 20.9    (128)
//     int8     14.3 / 12.3   34.4 / 30.7   30.9 / 27.4   13.2 / 11.4   28.8 / 25.9    (128)
//     4 bits   11.8 / 10.8   23.7 / 22.1   21.9 / 20.1   12.4 / 11.5   20.8 / 19.2    31.3 / 24.2
// (but, a tile each, 16 x 8 after 4000 of 64 26.3 / 27.4 in bf16, 18.6 / 19.0, 20.3 / 20.7 and 8 x 3
// after 16000, 8 heads on 4 of 128, 46.8 / 52.4, 27.8 / 29.1, 30.0 / 30.7; in 4 bits 16 x 2 after 4000
// of 96 12.9 / 10.1).  Ragged contexts go either way in 4 bits (5, 6 and 12 chunks of 6 rows of
// up to 9000, 9000 and 5000, 16 heads on 2 of 128: 14.2 / 14.9, 16.5 / 15.3, 19.0 / 16.8).
// A window cuts shares of unlike length, and the grid has the short ones last.  So with one, and
// two tiles a sequence in 4 bits, the line needs the gain of the L2 (tiles of other numbers of
// workgroups: 32 x 5 in one of 2048 of 96 23.9 / 23.8 in bf16, 19.4 / 20.2, 21.3 / 22.2 and 16.8 / 17.1
// in 4 bits; 32 x 4 in one of 1000, 16 heads on 2 of 128, 19.2 / 20.4, 13.9 / 15.6, 15.3 / 17.1, 13.4 /
// 14.1), and below 16 bits, which have less to gain, shares that all have blocks (64 x 5 in one of 1000,
// four shares of 12, 12, 9 and no blocks, 22.6 / 18.7 in bf16, 17.1 / 17.9, 18.4 / 20.8, 14.1 / 16.1; in
// one of 2048, 20 to 5 blocks, 36.4 / 24.1, 24.7 / 22.3, 26.3 / 26.8, 19.7 / 19.7).  In 4 bits of one tile
// a sequence, or three and more, windows gain (64 x 3 in one of 2048 15.1 / 14.6, 64 x 5, 16 heads on
// 2 of 128, 26.9 / 24.5).
// One row a sequence has no tile too many (in 4 bits 8 of 32000 keys 17.1 / 17.8).  A line is as
// long as a grid may be; past 2^20 workgroups the order is nothing.  Tiles of 128 keep theirs,
// longest first (2 prompts of 4096 68.8 / 75.7).
inline bool tiles_last(const Plan& p, int type, int batch, int rows, int rep, int kv_heads,
                       int positions, int window, int sinks, int64_t workgroups) {
  const int64_t all = static_cast<int64_t>(rows) * rep, one = int64_t{kStepRows} * batch;
  if (rows <= batch || workgroups > 1 << 20 || (type != kPagedE2m1 && all <= one)) return false;
  if (window >= positions || (type == kPagedE2m1 && (all <= one || all > 2 * one))) return true;
  if (p.splits * kv_heads % 8 != 0 || type == kPagedBf16) return p.splits * kv_heads % 8 == 0;
  const int blocks =
      static_cast<int>((int64_t{window} + sinks + kPagedBlock - 1) / kPagedBlock + 1);
  return (p.splits - 1) * even_share(blocks, p.splits) < blocks;
}

}  // namespace paged
}  // namespace parrot
