// product_kernel's instances for bf16 operands.
#include "ffn_product_tiles.h"

namespace bvml_ffn {

hipError_t launch_tiles_bf16(const Product& a, const ProductPlan& p, int layout, bool gated,
                           hipStream_t s) {
    return launch_tiles<kBF16>(a, p, layout, gated, s);
}
hipError_t launch_gradients_bf16(const Gradients& g, int tile, hipStream_t s) {
    return launch_gradient_tiles<kBF16>(g, tile, s);
}

}  // namespace bvml_ffn
