// product_kernel's instances for bf16 operands.
#include "ffn_product_tiles.h"

namespace bvml_ffn {

hipError_t launch_tiles_bf16(const Product& a, const ProductPlan& p, int layout, bool gated,
                           hipStream_t s) {
    return launch_tiles<kBF16>(a, p, layout, gated, s);
}

}  // namespace bvml_ffn
