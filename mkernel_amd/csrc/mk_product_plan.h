// mk_product_plan.h — which tile a product runs on and in how many parts along K:
// the host's choice, from sizes and the number of CUs (no HIP headers, so that it
// can be checked without a GPU).
#pragma once
#include <stdint.h>

#include <algorithm>

namespace mk {

enum ProductTile : int { kProd32 = 0, kProd64 = 1, kProd64w = 2, kProd128 = 3, kProd256 = 4, kProd128w = 5, kProdTiles = 6 };
constexpr int kProductTickets = 256;  // tiles of a launch whose K is cut into parts, at most
constexpr int kTicketStride = 32;     // words between them: a line each

// The tile shapes and what they cost, in us.  A launch runs in rounds of per_cu x CUs workgroups; a round takes
//   round + K/16 x slope(x),  slope = one + load min(x, 1) + more max(x - 1, 0),  x = the round's workgroups per CU
// (a full chip clocks lower and shares its caches).  `start` comes once, `area` for a million results (their stores),
// and where the last round's tiles are cut: meet + part per part, and `exchange` for a MB of partial sums.  Fitted to
// 1392 launches of 79 shapes of 1 .. 8192 rows, 64 .. 8192 columns and K on one MI355X; among these the tile and cut
// that it picks take 4 % longer than the best of those tried in the mean (worst 33 %).  Odd sizes and short sums take 25
// to 60 % longer than it says (1003 x 2811 x 1501 22 us and 28, a gradient 1024 x 520 x 5003 14 and 22).
struct ProductShape {
  int bm, bn, per_cu;
  double start, round, one, load, more, meet, part, area, exchange;
};
constexpr ProductShape kProductShapes[kProdTiles] = {
    {32, 128, 2, 3.68, 0.00, 0.076, 0.015, 0.129, 0.95, 0.39, 5.42, 0.13},
    {64, 64, 2, 2.97, 0.84, 0.071, 0.012, 0.052, 1.17, 0.34, 0.69, 0.17},
    {64, 128, 2, 3.81, 0.00, 0.071, 0.040, 0.084, 1.46, 0.30, 0.53, 0.30},
    {128, 128, 2, 2.66, 1.12, 0.099, 0.113, 0.079, 1.94, 0.32, 0.47, 0.29},
    {256, 256, 1, 4.95, 1.00, 0.141, 0.266, 0.0, 4.41, 1.32, 0.86, 0.13},
    {128, 256, 2, 5.37, 0.00, 0.167, 0.073, 0.231, 2.95, 0.90, 0.36, 0.31},
};

// One row or two go to the kernel that has all of K in one workgroup where K is short, or where B would have to be laid
// out anew (which takes three times the bytes).
inline bool product_few_rows(int64_t M, int64_t N, int64_t K, bool aligned) {
  return M <= 2 && N >= 8 && (M * K <= 2048 || !aligned);
}

struct ProductPlan {
  int tile, split;
  int64_t tiles, whole;  // without the parts; tiles that are not cut
  double us;
};

// M rows (ragged 1: in `groups` groups, about as many each), `cols` columns of B (SwiGLU: gate and up together), K
// (ragged 2: of all groups).  plain: results go as they are.
// cut: whether K may be cut.
inline ProductPlan plan_product(int64_t M, int64_t cols, int64_t K, int64_t groups, int ragged, bool right_grad,
                                bool plain, bool cut, int cus) {
  ProductPlan best = {};
  bool found = false;
  for (int i = 0; i < kProdTiles; ++i) {
    const ProductShape& s = kProductShapes[i];
    // (tiles of 32 rows stream weights of groups more slowly: 64 tokens' 27 experts of 7168 x 4096 242 us, 214 with 64)
    if ((right_grad || ragged) && s.bm == 32) continue;
    if (i == kProd128w && !(right_grad && plain)) continue;
    const int64_t tn = (cols + s.bn - 1) / s.bn;
    // a group's rows fill its last tile by half in the mean; of the tallest, rows that are not there cost little
    const int64_t spare = ragged == 1 ? (groups - 1) * (s.bm == 256 ? 64 : s.bm / 2) : 0;
    const int64_t tm = (M + spare + s.bm - 1) / s.bm;
    const int64_t tiles = tm * tn * (ragged == 2 ? groups : 1), slots = (int64_t)s.per_cu * cus;
    const double k16 = (double)(ragged == 2 ? K / std::max<int64_t>(groups, 1) : K) / 16;
    // whole rounds, and the last one's tiles in parts
    const int64_t rest = tiles % slots, rounds = tiles / slots;
    for (int split : {1, 2, 3, 4, 6, 8, 12, 16}) {
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
