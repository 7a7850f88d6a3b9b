// product_kernel's instances for f16 operands.
#include "ffn_product_tiles.h"

namespace bvml_ffn {

hipError_t launch_tiles_f16(const Product& a, const ProductPlan& p, int layout, bool gated,
                           hipStream_t s) {
    return launch_tiles<kF16>(a, p, layout, gated, s);
}
hipError_t launch_gradients_f16(const Gradients& g, int tile, hipStream_t s) {
    return launch_gradient_tiles<kF16>(g, tile, s);
}

}  // namespace bvml_ffn
