// product_kernel's instances for e4m3 operands.
#include "ffn_product_tiles.h"

namespace bvml_ffn {

hipError_t launch_tiles_e4m3(const Product& a, const ProductPlan& p, int layout, bool gated,
                           hipStream_t s) {
    return launch_tiles<kE4M3>(a, p, layout, gated, s);
}

}  // namespace bvml_ffn
