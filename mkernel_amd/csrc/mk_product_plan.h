// mk_product_plan.h — which tile a product runs on and in how many parts along K:
// the host's choice, from sizes alone (no HIP headers, so that it can be checked
// without a GPU).
#pragma once
#include <stdint.h>

#include <algorithm>

namespace mk {

enum ProductTile : int { kProd32 = 0, kProd64 = 1, kProd128 = 2, kProd256 = 3, kProdTiles = 4 };
constexpr int kProductTickets = 1024;  // tiles of a launch whose K is cut into parts, at most

struct ProductShape {
  int bm, bn, per_cu, waves_n;
  double start, per_k16, meet;  // us: of a round, of 16 of K with every CU busy, of a tile's parts
};
constexpr ProductShape kProductShapes[kProdTiles] = {
    {32, 128, 2, 2, 2.5, 0.030, 3.0},
    {64, 128, 2, 2, 2.5, 0.045, 4.0},
    {128, 128, 2, 2, 3.0, 0.110, 5.0},
    {256, 256, 1, 4, 6.0, 0.205, 12.0},
};

struct ProductPlan {
  int tile, split;
  int64_t tiles;  // without the parts
  double us;
};

// M rows (ragged: in `groups` groups, about as many each), `cols` columns of B (SwiGLU: gate and up together), K
// (ragged sums: of all groups).  right_grad: no tiles of 32 rows.  cut: whether K may be cut.
inline ProductPlan plan_product(int64_t M, int64_t cols, int64_t K, int64_t groups, int ragged, bool right_grad,
                                bool cut, int cus) {
  ProductPlan best = {};
  bool found = false;
  for (int i = 0; i < kProdTiles; ++i) {
    const ProductShape& s = kProductShapes[i];
    if (right_grad && s.bm == 32) continue;
    const int64_t tn = (cols + s.bn - 1) / s.bn;
    // a group's rows fill its last tile by half in the mean
    const int64_t tm = ragged == 1 ? (M + (groups - 1) * (s.bm / 2) + s.bm - 1) / s.bm : (M + s.bm - 1) / s.bm;
    const int64_t tiles = tm * tn * (ragged == 2 ? groups : 1);
    const double k16 = (double)(ragged == 2 ? K / std::max<int64_t>(groups, 1) : K) / 16;
    for (int split = 1; split <= 16; ++split) {
      // groups' sums have lengths that the host does not know, rows' tiles a number that it does not: not cut
      if (split > 1 && (!cut || ragged || tiles * split > 2 * (int64_t)s.per_cu * cus || tiles > kProductTickets ||
                        k16 < 8.0 * split))
        break;
      const int64_t slots = (int64_t)s.per_cu * cus, g = tiles * split;
      const double rounds = (double)((g + slots - 1) / slots);
      double t = rounds * (s.start + k16 / split * s.per_k16) + (split > 1 ? s.meet + 0.5 * split : 0.0);
      if (!found || t < best.us) {
        found = true;
        best = {i, split, tiles, t};
      }
    }
  }
  return best;
}

}  // namespace mk
