// Launches product_kernel for one element type: every tile, layout and copy
// that plan_product can name.  Included by ffn_product_{f16,bf16,e4m3}.hip,
// a translation unit each so that they compile side by side.
#pragma once

#include "ffn_kernels.h"
#include "ffn_product.h"

namespace bvml_ffn {

template <int kIn, int BM, int BN, int S, bool PT, bool QT, bool G, bool D>
hipError_t launch_one(const Product& a, hipStream_t s) {
    const long long groups = groups_of(a);
    if (groups > kMostGroups) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((product_kernel<kIn, BM, BN, S, PT, QT, G, D>), dim3((unsigned)groups),
                       dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int kIn, bool PT, bool QT, bool G>
hipError_t launch_layout(const Product& a, const ProductPlan& p, hipStream_t s) {
    if (!p.dma) {
        if constexpr (!G) {
            if (p.tile == kTileSquare) return launch_one<kIn, 64, 64, 2, PT, QT, G, false>(a, s);
        }
        return launch_one<kIn, 128, 128, 2, PT, QT, G, false>(a, s);
    }
    switch (p.tile) {
        case kTile256: return launch_one<kIn, 256, 256, 2, PT, QT, G, true>(a, s);
        case kTile128: return launch_one<kIn, 128, 128, 2, PT, QT, G, true>(a, s);
        case kTile128Deep: return launch_one<kIn, 128, 128, 4, PT, QT, G, true>(a, s);
        case kTile64: return launch_one<kIn, 64, 128, 3, PT, QT, G, true>(a, s);
        default:
            // (half of 64 columns is no 32 x 32 block for each of two waves)
            if constexpr (G)
                return hipErrorInvalidConfiguration;
            else
                return launch_one<kIn, 64, 64, 4, PT, QT, G, true>(a, s);
    }
}

template <int kIn, int BM, int BN, int S>
hipError_t launch_both(const Gradients& g, hipStream_t s) {
    hipLaunchKernelGGL((gradients_kernel<kIn, BM, BN, S>), dim3((unsigned)groups_of(g)), dim3(256),
                       0, s, g);
    return hipGetLastError();
}

template <int kIn>
hipError_t launch_gradient_tiles(const Gradients& g, int tile, hipStream_t s) {
    switch (tile) {
        case kTile256: return launch_both<kIn, 256, 256, 2>(g, s);
        case kTile128: return launch_both<kIn, 128, 128, 2>(g, s);
        case kTile128Deep: return launch_both<kIn, 128, 128, 4>(g, s);
        case kTile64: return launch_both<kIn, 64, 128, 3>(g, s);
        default: return launch_both<kIn, 64, 64, 4>(g, s);
    }
}

template <int kIn>
hipError_t launch_tiles(const Product& a, const ProductPlan& p, int layout, bool gated,
                        hipStream_t s) {
    if constexpr (kIn != kE4M3) {
        if (layout == kInputGrad) return launch_layout<kIn, false, true, false>(a, p, s);
        if (layout == kWeightGrad) return launch_layout<kIn, true, true, false>(a, p, s);
    }
    return gated ? launch_layout<kIn, false, false, true>(a, p, s)
                 : launch_layout<kIn, false, false, false>(a, p, s);
}

}  // namespace bvml_ffn
