// The feed-forward library's kernels as its C entry points call them.
// Private to libbvml_ffn.so.
#pragma once

#include "ffn_common.h"

namespace bvml_ffn {

// Workgroups of 256 threads that a launch holds: fewer than 2^32 threads.
constexpr long long kMostGroups = (1LL << 24) - 1;

// Which operand lies with k across its rows (ffn_product.h).
enum Layout { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };

// A product's operands and sums; its kernel, tile and split are chosen by
// plan_product.
struct ProductCall {
    const void* p;
    const void* q;
    long long ldp, ldq;  // elements from row to row
    int M, R, K;
    int in_type;
    int layout;
    bool gated;
    bool padded_p;  // P's rows end on 16 bytes, zeros from K (columns: from M) on
    Epilogue e;
};

// 256 x 256; 128 x 128 with two LDS slots (two workgroups a CU) or four (one);
// 64 x 128 with three and 64 x 64 with four (two a CU; the latter not gated); the
// few-rows kernel.
enum Tile { kTile256 = 0, kTile128 = 1, kTile128Deep = 2, kTile64 = 3, kTileSquare = 4, kTileRows = 5 };

struct ProductPlan {
    int tile;    // a Tile
    bool dma;    // copies go straight to LDS
    int whole;   // tiles that one workgroup sums
    int splits;  // workgroups for each of the others, joined by a second launch
};

// The kernel for a product of these sizes (dma: dma_fits of its operands).
ProductPlan plan_product(int M, int R, int K, int in_type, int layout, bool gated, bool dma);
bool dma_fits(const ProductCall& c);
// bytes of partial sums the plan needs, with and without direct copies
long long product_workspace(int M, int R, int K, int in_type, int layout, bool gated);
hipError_t launch_product(const ProductCall& c, void* workspace, hipStream_t s);

// out[c] = the sum of `parts` rows of `cols` floats, of `type` (out null: none).
struct ColumnSum {
    const float* part;
    int parts, cols;
    void* out;
    int type;
};

// Both gradients of one product from the same dz: x's (c.p = dz, c.q = W) and W's
// (c.p = dz, c.q = x), in one launch where their operands go straight to LDS.
struct GradientsPlan {
    int tile;
    bool weight_first;  // the weight's workgroups take longer
    // tiles of each that one workgroup sums, workgroups for each of the others
    int input_whole, input_splits, weight_whole, weight_splits;
};
GradientsPlan plan_gradients(int M, int R, int K);
long long gradients_workspace(int M, int R, int K);
// `sums` goes along with them
hipError_t launch_gradients(const ProductCall& input, const ProductCall& weight,
                            const ColumnSum& sums, void* workspace, hipStream_t s);

// One translation unit an element type (ffn_product_*.hip).
struct Product;
hipError_t launch_tiles_f16(const Product& a, const ProductPlan& p, int layout, bool gated,
                            hipStream_t s);
hipError_t launch_tiles_bf16(const Product& a, const ProductPlan& p, int layout, bool gated,
                             hipStream_t s);
hipError_t launch_tiles_e4m3(const Product& a, const ProductPlan& p, int layout, bool gated,
                             hipStream_t s);
struct Gradients;
hipError_t launch_gradients_f16(const Gradients& g, int tile, hipStream_t s);
hipError_t launch_gradients_bf16(const Gradients& g, int tile, hipStream_t s);

struct NormCall {
    const void* x;
    const void* residual;
    const void* weight;
    long long ldx, ldr, ldy, lds;
    int rows, cols;
    float eps;
    int x_type, w_type, y_type;
    void* y;
    void* stream_out;
    float* scale;
    float* rstd;
};
hipError_t launch_norm(const NormCall& c, hipStream_t s);

struct NormGradCall {
    const void* dy;
    const void* stream_in;
    const void* weight;
    const float* rstd;
    const void* dstream;
    long long lddy, lds, ldds, lddx;
    int rows, cols;
    int dy_type, x_type, w_type;
    void* dx;
    void* dweight;
    float* workspace;
};
long long norm_grad_workspace(int rows, int cols);
hipError_t launch_norm_grad(const NormGradCall& c, hipStream_t s);

// dz = dy act'(z) (linear) or [dy up act'(gate), dy act(gate)] (gated), in
// 16 bits with rows of ldd elements (zeros beyond the last column), and the
// sums of its columns.
struct SlopeCall {
    const void* dy;
    const void* z;  // null: dz = dy
    long long lddy, ldz, ldd;
    int rows, N;
    bool gated;
    int dy_type, type, act;
    void* dz;    // null: only the sums
    void* db;    // null: only dz
    float* workspace;
};
hipError_t launch_column_sum(const ColumnSum& c, hipStream_t s);
long long slope_workspace(int rows, int R);
// (*sums: what is left to do for db)
hipError_t launch_slope(const SlopeCall& c, ColumnSum* sums, hipStream_t s);

}  // namespace bvml_ffn
