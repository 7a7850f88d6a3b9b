// Launches product_kernel for one element type: every tile, layout and copy
// that plan_product can name.  Included by ffn_product_{f16,bf16,e4m3}.hip,
// a translation unit each so that they compile side by side.
#pragma once

#include "ffn_kernels.h"
#include "ffn_product.h"

namespace bvml_ffn {

template <int kIn, int BM, int BN, int WM, int WN, bool PT, bool QT, bool G, bool D>
hipError_t launch_one(const Product& a, int splits, hipStream_t s) {
    Product c = a;
    const int cols = G ? BN / 2 : BN;
    c.tiles_m = (a.M + BM - 1) / BM;
    c.tiles_n = ((G ? a.R / 2 : a.R) + cols - 1) / cols;
    const long long tiles = (long long)c.tiles_m * c.tiles_n;
    if (tiles > 0x7fffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((product_kernel<kIn, BM, BN, WM, WN, PT, QT, G, D>),
                       dim3((unsigned)tiles, (unsigned)splits), dim3(64 * WM * WN), 0, s, c);
    return hipGetLastError();
}

template <int kIn, bool PT, bool QT, bool G>
hipError_t launch_layout(const Product& a, const ProductPlan& p, hipStream_t s) {
    if (!p.dma) return launch_one<kIn, 128, 128, 2, 2, PT, QT, G, false>(a, p.splits, s);
    switch (p.tile) {
        case kTile256: return launch_one<kIn, 256, 256, 2, 2, PT, QT, G, true>(a, p.splits, s);
        case kTile128: return launch_one<kIn, 128, 128, 2, 2, PT, QT, G, true>(a, p.splits, s);
        default: return launch_one<kIn, 64, 128, 2, 2, PT, QT, G, true>(a, p.splits, s);
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
