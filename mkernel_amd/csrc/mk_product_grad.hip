// mk_product_grad.hip — the products of a backward pass (mk_product.h): of the
// activations (rows against the rows of the weights) and of the weights (columns
// against columns), without a transposed copy of either.
#include "mk_product.h"

namespace mk {

hipError_t launch_product_left_grad(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream) {
  switch (epi) {
    case kProdStore: return launch_product_tile<true, true, kProdStore>(p, tile, grid, stream);
    case kProdPlain: return launch_product_tile<true, true, kProdPlain>(p, tile, grid, stream);
    case kProdSwigluGrad: return launch_product_tile<true, true, kProdSwigluGrad>(p, tile, grid, stream);
  }
  return hipErrorInvalidValue;
}

namespace {
template <int EPI>
hipError_t right_grad(const ProductParams& p, int tile, int64_t grid, hipStream_t stream) {
  switch (tile) {
    case kProd64: return launch_product_cfg<ProdTile64, void, false, false, EPI>(p, grid, stream);
    case kProd64w: return launch_product_cfg<ProdTile64w, void, false, false, EPI>(p, grid, stream);
    case kProd128: return launch_product_cfg<ProdTile128, void, false, false, EPI>(p, grid, stream);
    case kProd256: return launch_product_cfg<ProdTile256, void, false, false, EPI>(p, grid, stream);
    case kProd128w:
      // (what the other epilogues keep in registers does not fit beside a second workgroup: 60 of them spilled, 575 us
      // instead of 383 for 32 experts of 2048 x 7168.  Adding to these experts' bf16 dW takes 798 us on the other
      // tiles, to an fp32 one 1141; storing 390 and 511)
      if constexpr (EPI != kProdStore) return launch_product_cfg<ProdTile128w, void, false, false, EPI>(p, grid, stream);
  }
  return hipErrorInvalidValue;
}
}  // namespace

hipError_t launch_product_right_grad(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream) {
  switch (epi) {
    case kProdStore: return right_grad<kProdStore>(p, tile, grid, stream);
    case kProdPlain: return right_grad<kProdPlain>(p, tile, grid, stream);
    case kProdPlain32: return right_grad<kProdPlain32>(p, tile, grid, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mk
