"""The shares of key blocks that attention over pages of 4 bits takes cover what each tile's
rows see, and its grids all tiles: the kernels' own functions, walked on the host."""
from test_paged_share_cpu import _run


def test_every_batch(tmp_path):
    """Batches of all kinds, from single rows to prompts: tiles of 4, 8, 16, 32 and 128 rows."""
    _run(tmp_path, """
  std::mt19937 rng(2);
  auto pick = [&](int low, int high) {  // spread over the logarithm
    std::uniform_real_distribution<double> u(std::log(low), std::log(high + 0.999));
    return std::min(static_cast<int>(std::exp(u(rng))), high);
  };
  const int layouts[][2] = {{8, 2}, {8, 8}, {16, 2}, {12, 4}, {4, 1}, {6, 2}, {5, 1}, {32, 32}, {7, 1}};
  int tiles[129] = {0}, wide = 0, wide_splits = 0;
  for (int run = 0; run < 8000; ++run) {
    Walk w;
    w.type = 4;
    w.heads = layouts[run % 9][0], w.kv_heads = layouts[run % 9][1];
    w.page = 32 << (rng() % 3);
    w.window = rng() % 4 == 0 ? INT32_MAX : pick(1, 4096);
    w.sinks = rng() % 2 ? 0 : pick(1, 300);
    const int batch = pick(1, 300), most = rng() % 3 ? pick(1, 4) : pick(1, std::max(1, 8192 / batch));
    const int context = pick(1, rng() % 4 ? 12000 : 100000);
    int longest = 0, rows = 0;
    for (int i = 0; i < batch; ++i) {
      w.news.push_back(rng() % 5 ? static_cast<int>(rng() % most) + 1 : rng() % 2 ? most : 0);
      w.lengths.push_back(w.news[i] + static_cast<int>(rng() % context));
      if (rng() % 40 == 0) w.lengths[i] = w.news[i] / 2;  // rows before position 0
      longest = std::max(longest, w.lengths[i]);
      rows += w.news[i];
    }
    w.width = (longest + w.page - 1) / w.page;
    if (rng() % 8 == 0) w.width = w.width * static_cast<int>(rng() % 8) / 8;
    if (!w.covered(&split)) return 1;
    const int rep = w.heads / w.kv_heads;
    const Plan p = plan(4, batch, rows, w.heads, w.kv_heads, w.page, w.width, w.window, w.sinks);
    int64_t all = 0;
    for (int n : w.news) all += (static_cast<int64_t>(n) * rep + p.tile - 1) / p.tile;
    if (all > grid_tiles(rows, batch, rep, p.tile)) return 3;
    if (p.wide && (p.tile > 8 || (p.tile == 4 && p.splits != 1))) return 4;
    wide_splits += p.wide && p.splits > 1;
    ++tiles[p.tile];
    wide += p.wide;
  }
  for (int t : {4, 8, 16, 32, 128})
    if (tiles[t] < 20) return 5;
  std::printf("%d shares, %d wide, %d of them split\\n", split, wide, wide_splits);
  return split > 10000 && wide > 100 && wide < 4000 && wide_splits >= 20 ? 0 : 2;""")


def test_grids(tmp_path):
    """Every tile of every batch has a workgroup, of any type."""
    _run(tmp_path, """
  std::mt19937 rng(3);
  for (int run = 0; run < 200000; ++run) {
    const int batch = 1 + rng() % 20, rep = 1 + rng() % 40, tile = 4 << (rng() % 6);
    int rows = rng() % 5;  // (some of nobody)
    int64_t all = 0;
    for (int i = 0; i < batch; ++i) {
      const int n = rng() % 4 ? rng() % 4 : rng() % 300;
      rows += n;
      all += (static_cast<int64_t>(n) * rep + tile - 1) / tile;
    }
    if (all > grid_tiles(rows, batch, rep, tile)) return 1;
  }
  return split;""")
