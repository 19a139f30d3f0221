"""The shares of key blocks that paged attention's workgroups take cover what each
tile's rows see: the kernels' own functions, compiled for the host and walked
through whole launches."""
import subprocess
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "parrot-h200-worker_amd" / "parrot" / "kernels"

WALK = r"""
#include "paged_share.h"
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>
using namespace parrot;
using namespace parrot::paged;

// Every tile of every sequence: its shares begin at its first block, follow each other and
// end at its last, and its blocks hold every key that a row of it sees.
struct Walk {
  int type, heads, kv_heads, page, width, window, sinks;
  std::vector<int> news, lengths;
  bool fail(const char* what, int i, int row0, const Plan& p, int count, int end) const {
    std::printf("%s: type %d, %d heads on %d, page %d, width %d, window %d, sinks %d, %d sequences, "
                "%d new of %d, row %d, tile %d, splits %d: %d blocks, to %d\n", what, type, heads,
                kv_heads, page, width, window, sinks, static_cast<int>(news.size()), news[i],
                lengths[i], row0, p.tile, p.splits, count, end);
    return false;
  }
  bool covered(int* split_tiles) const {
    int total = 0;
    for (int n : news) total += n;
    const Plan p = plan(type, static_cast<int>(news.size()), total, heads, kv_heads, page, width,
                        window, sinks);
    const int rep = heads / kv_heads;
    for (size_t i = 0; i < news.size(); ++i) {
      const PagedSequence s{0, news[i], lengths[i], std::min(lengths[i], width * page)};
      const int rows = s.count * rep, before = s.length - s.count;
      for (int row0 = 0; row0 < rows; row0 += p.tile) {
        const int first = before + row0 / rep;
        const int last = before + (std::min(row0 + p.tile, rows) - 1) / rep;
        const Blocks b = tile_blocks(first, last, s.stored, window, sinks);
        for (int k = 1; k < b.count; ++k)
          if (b.at(k) <= b.at(k - 1)) return fail("order", i, row0, p, b.count, k);
        for (int q : {first, last}) {  // the blocks between are those of the rows between
          const int newest = std::min(q, s.stored - 1), low = q >= window ? q - window + 1 : 0;
          for (int key : {low, newest, 0, std::min(sinks, newest + 1) - 1}) {
            if (key < 0 || key > newest || (key < low && key >= sinks)) continue;
            bool there = false;
            for (int k = 0; k < b.count && !there; ++k) there = b.at(k) == key / kPagedBlock;
            if (!there) return fail("key", i, row0, p, b.count, key);
          }
        }
        int end = 0;
        const Share one = split_share(s, rows, p.tile, rep, b, 0, p.splits, p.whole, window, sinks);
        for (int split = 0; split < (one.whole ? 1 : p.splits); ++split) {
          const Share x = split_share(s, rows, p.tile, rep, b, split, p.splits, p.whole, window, sinks);
          if (x.whole != one.whole || x.begin != end || x.end < x.begin || x.end > b.count)
            return fail("share", i, row0, p, b.count, end);
          if (x.end - x.begin > x.most) return fail("most", i, row0, p, x.most, x.end - x.begin);
          end = x.end;
        }
        if (end != b.count) return fail("lost", i, row0, p, b.count, end);
        *split_tiles += !one.whole;
      }
    }
    return true;
  }
};

Walk same(int type, int heads, int kv_heads, int page, int n, int news, int length, int window, int sinks,
          int width = 0) {
  return {type, heads, kv_heads, page, width ? width : (length + page - 1) / page, window, sinks,
          std::vector<int>(n, news), std::vector<int>(n, length)};
}

int main() {
  int split = 0;
"""


def _run(tmp_path, body):
    source, program = tmp_path / "walk.cpp", tmp_path / "walk"
    source.write_text(WALK + body + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{KERNELS}", str(source), "-o",
                    str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_short_last_tiles(tmp_path):
    """A sequence's last tile may span fewer positions than the others, and so see fewer
    of a window's blocks: short chunks, chunks of prompts and whole prompts."""
    _run(tmp_path, """
  for (const Walk& w : {same(0, 8, 2, 64, 64, 5, 4096, 2048, 0), same(1, 8, 2, 64, 36, 5, 4096, 2048, 0),
                        same(0, 8, 2, 64, 4, 1025, 4096, 2048, 0),
                        same(0, 8, 2, 64, 1, 465, 1465, 1000, 0), same(2, 8, 8, 64, 16, 337, 1337, 1024, 0),
                        same(0, 16, 2, 32, 1, 1172, 1172, 1000, 0)})
    if (!w.covered(&split)) return 1;
  return split > 0 ? 0 : 2;""")


def test_tables_shorter_than_the_lengths(tmp_path):
    """The last rows' window may lie past what the table holds, where they see less than
    the rows before them, or nothing."""
    _run(tmp_path, """
  for (int type : {0, 2})
    for (int news : {5, 40, 2000})
      for (int width : {1, 16, 32, 48, 50})
        for (int window : {1, 300, 1000, INT32_MAX})
          if (!same(type, 8, 2, 64, 1, news, 3200, window, 5, width).covered(&split)) return 1;
  return split > 0 ? 0 : 2;""")


def test_every_batch(tmp_path):
    """Batches of all kinds: head layouts, ragged chunks and lengths, windows, sinks, pages,
    tables that hold the lengths and tables that do not."""
    _run(tmp_path, """
  std::mt19937 rng(1);
  auto pick = [&](int low, int high) {  // spread over the logarithm
    std::uniform_real_distribution<double> u(std::log(low), std::log(high + 0.999));
    return std::min(static_cast<int>(std::exp(u(rng))), high);
  };
  const int layouts[][2] = {{8, 2}, {8, 8}, {16, 2}, {12, 4}, {4, 1}, {6, 2}, {5, 1}, {32, 32}, {7, 1}};
  for (int run = 0; run < 6000; ++run) {
    Walk w;
    w.type = static_cast<int>(rng() % 3);
    w.heads = layouts[run % 9][0], w.kv_heads = layouts[run % 9][1];
    w.page = 32 << (rng() % 3);
    w.window = rng() % 4 == 0 ? INT32_MAX : pick(1, 4096);
    w.sinks = rng() % 2 ? 0 : pick(1, 300);
    const int batch = pick(1, 64), most = rng() % 2 ? pick(1, 8) : pick(1, std::max(1, 8192 / batch));
    const int context = pick(1, 9000);
    int longest = 0;
    for (int i = 0; i < batch; ++i) {
      w.news.push_back(rng() % 5 ? static_cast<int>(rng() % most) + 1 : rng() % 2 ? most : 0);
      w.lengths.push_back(w.news[i] + static_cast<int>(rng() % context));
      if (rng() % 40 == 0) w.lengths[i] = w.news[i] / 2;  // rows before position 0
      longest = std::max(longest, w.lengths[i]);
    }
    w.width = (longest + w.page - 1) / w.page;
    if (rng() % 8 == 0) w.width = w.width * static_cast<int>(rng() % 8) / 8;
    if (!w.covered(&split)) return 1;
  }
  return split > 10000 ? 0 : 2;""")
