// Runs the walk of the 4-bit cache's attention blocks (csrc/kv4_walk.h) on the host:
// every block of a call, its rings' producers and consumers, with lengths that stay and
// with lengths that change at every read.
//   kv4_walk_check <seed> <calls>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv4_walk.h"

using namespace mri::kv4;

struct Args {
  struct {
    int batch, heads;
    size_t cap;
  } c;
  int n_tokens, group, rows, n_rows, row_groups, keys, pad, splits;
  std::vector<int> lens;
  bool change;
  mutable std::mt19937* rng;
  int len(int b) const {
    if (b < 0 || b >= c.batch) std::printf("length of entry %d of %d\n", b, c.batch), std::exit(1);
    if (change) return static_cast<int>((*rng)() % 3 ? (*rng)() % (c.cap + 1) : (*rng)() % 2 ? 0 : c.cap);
    return lens[b];
  }
};

#define CHECK(x) \
  if (!(x)) std::printf("line %d: %s (seed %u, call %d)\n", __LINE__, #x, seed, call), std::exit(1)

int main(int, char** argv) {
  const unsigned seed = static_cast<unsigned>(std::atoi(argv[1]));
  std::mt19937 rng(seed);
  auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
  for (int call = 0; call < std::atoi(argv[2]); ++call) {
    Args a;
    a.c = {pick(1, 9), pick(1, 5), static_cast<size_t>(64 * pick(1, 20))};
    a.group = pick(1, 8);
    a.n_tokens = rng() % 2 ? 1 : pick(1, 40);
    a.rows = a.group * a.n_tokens;
    const bool few = a.rows <= 8;
    const int tile = few ? 8 : 16, tiles = (a.rows + tile - 1) / tile, most = pick(3, 4);
    a.row_groups = (tiles + most - 1) / most;
    const int row_tiles = (tiles + a.row_groups - 1) / a.row_groups;
    a.row_groups = (tiles + row_tiles - 1) / row_tiles;
    a.n_rows = row_tiles * tile;
    a.keys = few ? 32 : 64;
    a.pad = few ? 12 : 2;
    a.splits = few ? 4 : 1;
    a.change = call % 2;
    a.rng = &rng;
    for (int b = 0; b < a.c.batch; ++b) a.lens.push_back(pick(0, 3) ? pick(0, static_cast<int>(a.c.cap)) : 0);
    const unsigned grid = static_cast<unsigned>(pick(1, 60)), least = 128 / static_cast<unsigned>(a.keys);
    const unsigned pairs = static_cast<unsigned>(a.c.batch * a.row_groups);
    // Stages seen of each unit, and blocks that arrived at it.
    std::vector<std::vector<int>> seen(pairs * a.c.heads);
    std::vector<int> arrived(grid), expected(grid);
    for (unsigned block = 0; block < grid; ++block) {
      unsigned total = 0;
      std::vector<unsigned> before;
      for (unsigned p = 0; p < pairs; ++p) {
        before.push_back(total);
        total += static_cast<unsigned>(unit_tiles(a, static_cast<int>(p / a.row_groups), static_cast<int>(p % a.row_groups)) * a.c.heads);
      }
      before.push_back(total);
      Plan plan;
      share_out(a, total, block, grid, least, plan);
      CHECK(plan.blocks >= 1 && plan.blocks <= grid && plan.count >= 0);
      for (unsigned p = 0; p < pairs; ++p)  // a thread a pair
        if (plan.x0 >= before[p] && plan.x0 - before[p] < before[p + 1] - before[p]) {
          const bool found = find_first(a, plan.x0, before[p], p, p + 1, plan.first);
          CHECK(found || a.change);
        }
      if (plan.count == 0) continue;
      CHECK(a.change || plan.first.b < a.c.batch);
      // The rings' producers: (unit, stage) in the order of their copies.
      struct Copy {
        int b, rg, h, stage;
      };
      std::vector<std::vector<Copy>> copies(a.splits);
      for (int ring = 0; ring < a.splits; ++ring) {
        Unit v = plan.first;
        for (int next = ring; (next = seek_stage(a, v, next, plan.count)) < plan.count; next += a.splits) {
          const int stage = next - (v.end - v.tiles + a.pad);
          CHECK(v.b < a.c.batch && v.rg < a.row_groups && v.h < a.c.heads);
          CHECK(stage >= 0 && static_cast<size_t>(stage + 1) * a.keys <= a.c.cap);
          CHECK(next % a.splits == ring && next < v.end);
          copies[ring].push_back({v.b, v.rg, v.h, stage});
          CHECK(copies[ring].size() <= static_cast<size_t>(plan.count));
        }
      }
      std::vector<size_t> used(a.splits, 0);
      Unit u = plan.first;
      int x = 0, unit_begin, seg_end, segments = 0;
      while (next_segment(a, u, x, plan.count, unit_begin, seg_end)) {
        CHECK(++segments <= plan.count);
        CHECK(u.b < a.c.batch && u.rg < a.row_groups && u.h < a.c.heads && x < seg_end && seg_end <= plan.count);
        const int c0 = owner_of(plan, plan.x0 + static_cast<unsigned>(unit_begin)), c1 = owner_of(plan, plan.x0 + static_cast<unsigned>(u.end - 1));
        CHECK(c0 >= 0 && c0 <= c1 && static_cast<unsigned>(c1) < plan.blocks);
        for (int ring = 0; ring < a.splits; ++ring)
          for (int y = x + (a.splits + ring - x % a.splits) % a.splits; y < seg_end; y += a.splits) {
            const int stage = y - unit_begin;
            CHECK(stage >= 0 && static_cast<size_t>(stage + 1) * a.keys <= a.c.cap);
            if (a.change) continue;
            CHECK(used[ring] < copies[ring].size());
            const Copy& c = copies[ring][used[ring]++];
            CHECK(c.b == u.b && c.rg == u.rg && c.h == u.h && c.stage == stage);
            auto& s = seen[(u.b * a.row_groups + u.rg) * a.c.heads + u.h];
            if (static_cast<int>(s.size()) <= stage) s.resize(stage + 1);
            ++s[stage];
          }
        if (!a.change) {
          CHECK(c0 <= static_cast<int>(block) && static_cast<int>(block) <= c1);
          CHECK((x == unit_begin && seg_end == u.end) == (c0 == c1));
          if (c0 != c1) {
            ++arrived[c0];
            CHECK(expected[c0] == 0 || expected[c0] == c1 - c0 + 1);
            expected[c0] = c1 - c0 + 1;
          }
        }
        x = seg_end;
        next_unit(a, u);
      }
      for (int ring = 0; ring < a.splits && !a.change; ++ring) CHECK(used[ring] == copies[ring].size());
    }
    if (a.change) continue;
    CHECK(arrived == expected);
    for (int b = 0; b < a.c.batch; ++b)
      for (int rg = 0; rg < a.row_groups; ++rg)
        for (int h = 0; h < a.c.heads; ++h) {
          const auto& s = seen[(b * a.row_groups + rg) * a.c.heads + h];
          CHECK(static_cast<int>(s.size()) == unit_tiles(a, b, rg) - a.pad);
          for (int n : s) CHECK(n == 1);
        }
  }
  std::puts("ok");
}
