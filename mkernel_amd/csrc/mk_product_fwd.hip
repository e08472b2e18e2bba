// mk_product_fwd.hip — forward products (mk_product.h): rows of activations
// against weights as they are stored, [K, N].
#include "mk_product.h"

namespace mk {

hipError_t launch_product_forward(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream) {
  switch (epi) {
    case kProdStore: return launch_product_tile<true, false, kProdStore>(p, tile, grid, stream);
    case kProdPlain: return launch_product_tile<true, false, kProdPlain>(p, tile, grid, stream);
    case kProdSwiglu: return launch_product_tile<true, false, kProdSwiglu>(p, tile, grid, stream);
    case kProdStats: return launch_product_tile<true, false, kProdStats>(p, tile, grid, stream);
    case kProdDlogits: return launch_product_tile<true, false, kProdDlogits>(p, tile, grid, stream);
    case kProdDlogits3: return launch_product_tile<true, false, kProdDlogits3>(p, tile, grid, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mk
