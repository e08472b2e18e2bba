// mk_product_plan.h — which tile a product runs on and in how many parts along K:
// the host's choice, from sizes alone (no HIP headers, so that it can be checked
// without a GPU).
#pragma once
#include <stdint.h>

#include <algorithm>

namespace mk {

enum ProductTile : int { kProd32 = 0, kProd64 = 1, kProd64w = 2, kProd128 = 3, kProd256 = 4, kProdTiles = 5 };
constexpr int kProductTickets = 1024;  // tiles of a launch whose K is cut into parts, at most

// The tile shapes and what they cost, in us.  A launch runs in rounds of per_cu x CUs workgroups; a round takes
//   round + K/16 x slope(x),  slope = one + load min(x, 1) + more max(x - 1, 0),  x = the round's workgroups per CU
// (a full chip clocks lower and shares its caches).  `start` comes once, `area` for a million results (their stores),
// and where the last round's tiles are cut: meet + part per part, and `exchange` for a MB of partial sums.  Fitted to
// 923 launches of 79 shapes of 1 .. 8192 rows, 64 .. 8192 columns and K on one MI355X; the tile and cut that it picks
// take 2 % longer than the best of those tried in the mean (worst 33 %).
struct ProductShape {
  int bm, bn, per_cu, waves_n;
  double start, round, one, load, more, meet, part, area, exchange;
};
constexpr ProductShape kProductShapes[kProdTiles] = {
    {32, 128, 2, 2, 4.10, 0.00, 0.078, 0.002, 0.061, 0.63, 0.41, 10.2, 0.55},
    {64, 64, 2, 1, 2.25, 2.20, 0.069, 0.020, 0.038, 0.73, 0.39, 0.58, 0.33},
    {64, 128, 2, 2, 3.52, 1.10, 0.071, 0.044, 0.069, 1.10, 0.39, 0.56, 0.39},
    {128, 128, 2, 2, 1.60, 2.87, 0.098, 0.120, 0.045, 2.06, 0.53, 0.46, 0.36},
    {256, 256, 1, 4, 6.59, 0.85, 0.142, 0.293, 0.0, 5.56, 2.01, 0.74, 0.14},
};

struct ProductPlan {
  int tile, split;
  int64_t tiles, whole;  // without the parts; tiles that are not cut
  double us;
};

// M rows (ragged 1: in `groups` groups, about as many each), `cols` columns of B (SwiGLU: gate and up together), K
// (ragged 2: of all groups).  cut: whether K may be cut.
inline ProductPlan plan_product(int64_t M, int64_t cols, int64_t K, int64_t groups, int ragged, bool right_grad,
                                bool cut, int cus) {
  ProductPlan best = {};
  bool found = false;
  for (int i = 0; i < kProdTiles; ++i) {
    const ProductShape& s = kProductShapes[i];
    // (tiles of 32 rows stream weights of groups more slowly: 64 tokens' 27 experts of 7168 x 4096 242 us, 214 with 64)
    if ((right_grad || ragged) && s.bm == 32) continue;
    const int64_t tn = (cols + s.bn - 1) / s.bn;
    // a group's rows fill its last tile by half in the mean; of the tallest, rows that are not there cost little
    const int64_t spare = ragged == 1 ? (groups - 1) * (s.bm == 256 ? 64 : s.bm / 2) : 0;
    const int64_t tm = (M + spare + s.bm - 1) / s.bm;
    const int64_t tiles = tm * tn * (ragged == 2 ? groups : 1), slots = (int64_t)s.per_cu * cus;
    const double k16 = (double)(ragged == 2 ? K / std::max<int64_t>(groups, 1) : K) / 16;
    // whole rounds, and the last one's tiles in parts
    const int64_t rest = tiles % slots, rounds = tiles / slots;
    for (int split = 1; split <= 16; ++split) {
      // groups' sums have lengths that the host does not know, rows' tiles a number that it does not: not cut
      if (split > 1 && (!cut || ragged || rest == 0 || rest * split > slots || rest > kProductTickets || k16 < 8.0 * split))
        break;
      const double x = (double)(rest * split) / cus;
      double t = s.start + (double)rounds * (s.round + k16 * (s.one + s.load + s.more * (s.per_cu - 1)));
      if (rest) t += s.round + k16 / split * (s.one + s.load * std::min(x, 1.0) + s.more * std::max(x - 1.0, 0.0));
      t += s.area * 1e-6 * (double)M * (double)cols * (ragged == 2 ? (double)groups : 1.0);
      if (split > 1) t += s.meet + s.part * split + s.exchange * 4e-6 * (double)(rest * split) * s.bm * s.bn;
      if (!found || t < best.us) {
        found = true;
        best = {i, split, tiles, split > 1 ? tiles - rest : tiles, t};
      }
    }
  }
  return best;
}

}  // namespace mk
