// Which kernel a product takes, the few-rows kernel, and the second launch
// that joins a split sum.

#include "ffn_kernels.h"
#include "ffn_product.h"

namespace bvml_ffn {

namespace {

// ---------------------------------------------------------------------------
// few rows (serving): the weights are read once, by 16 waves a workgroup
// that share 16 rows of W (gated: 16 of each half) and divide k; their sums
// meet in LDS.  Bound by reading W: every lane has its 16-byte pieces of
// kAhead k groups in flight.  The matrix instruction's other operand holds up to 16 rows
// of x at a time, so a row costs what sixteen cost.
// ---------------------------------------------------------------------------
template <int kIn, int kBlocks, bool kGated, bool kWhole>
__global__ __launch_bounds__(kBlocks == 4 ? 512 : 1024) void rows_kernel(Product a) {
    constexpr int kWaves = kBlocks == 4 ? 8 : 16;
    constexpr int kHalves = kGated ? 2 : 1;
    constexpr int kSize = kIn == kE4M3 ? 1 : 2, kPiece = 16 / kSize, kStep = 128 / kSize;
    constexpr int kAhead = kBlocks == 4 ? 1 : 2;
    __shared__ v4f sums[kWaves][kHalves][kBlocks][64];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int g = lane >> 4, i16 = lane & 15;
    const int N = a.e.N, n0 = blockIdx.x * 16;
    const int row = n0 + i16 < N ? n0 + i16 : N - 1;
    const char* q[kHalves];
    const char* p[kBlocks];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) q[h] = a.q + (long long)(row + h * N) * a.ldq;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const int m = 16 * b + i16;
        p[b] = a.p + (long long)(m < a.M ? m : a.M - 1) * a.ldp;
    }
    v4f acc[kHalves][kBlocks];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[h][b] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    // a lane's piece of k: zeros beyond the row's end
    auto piece = [&](const char* at, int k) {
        v4i v = {0, 0, 0, 0};
        const int n = a.K - k;
        if (n >= kPiece) {
            __builtin_memcpy(&v, at + (long long)k * kSize, 16);
        } else if (!kWhole && n > 0) {
            if constexpr (kSize == 2) {
                uint16_t h[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    h[i] = i < n ? reinterpret_cast<const uint16_t*>(at)[k + i] : (uint16_t)0;
                __builtin_memcpy(&v, h, 16);
            } else {
                uint8_t h[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    h[i] = i < n ? reinterpret_cast<const uint8_t*>(at)[k + i] : (uint8_t)0;
                __builtin_memcpy(&v, h, 16);
            }
        }
        return v;
    };
    for (int s = w; s < a.steps; s += kWaves * kAhead) {
        v4i qv[kAhead][kHalves][2], pv[kAhead][kBlocks][2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (s + u * kWaves) * kStep + g * kPiece;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int h = 0; h < kHalves; ++h) qv[u][h][c] = piece(q[h], k + c * 4 * kPiece);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) pv[u][b][c] = piece(p[b], k + c * 4 * kPiece);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    if constexpr (kIn == kE4M3) {
                        acc[h][b] = multiply8(
                            __builtin_shufflevector(qv[u][h][0], qv[u][h][1], 0, 1, 2, 3, 4, 5, 6, 7),
                            __builtin_shufflevector(pv[u][b][0], pv[u][b][1], 0, 1, 2, 3, 4, 5, 6, 7),
                            acc[h][b]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            acc[h][b] = multiply16<kIn>(qv[u][h][c], pv[u][b][c], acc[h][b]);
                    }
                }
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) sums[w][h][b][lane] = acc[h][b];
    __syncthreads();
    if (w >= kBlocks) return;
    float v[kHalves][4];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        v4f t = sums[0][h][w][lane];
#pragma unroll
        for (int j = 1; j < kWaves; ++j) t += sums[j][h][w][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[h][r] = t[r];
    }
    const int m = 16 * w + i16, n = n0 + 4 * g;
    if constexpr (kGated)
        finish_one_gated<4>(a.e, type16_of(kIn, a.e), m, n, v[0], v[1]);
    else
        finish_one<4>(a.e, type16_of(kIn, a.e), m, n, v[0]);
}

// Sums a split product's parts, in their order, and finishes them.
template <bool kGated>
__global__ __launch_bounds__(256) void join_kernel(Epilogue e, int in_type, int splits) {
    const int per = (e.N + 3) / 4;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long m = t / per;
    if (m >= e.M) return;
    const int n = (int)(t % per) * 4, c = e.N - n;
    const int R = kGated ? 2 * e.N : e.N;
    float v[4], u[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = u[r] = 0.0f;
    for (int s = 0; s < splits; ++s) {
        const long long at = ((long long)s * e.M + m) * R + n;
        float x[4];
        load_row<4>(e.part, kF32, at, c, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += x[r];
        if constexpr (kGated) {
            load_row<4>(e.part, kF32, at + e.N, c, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) u[r] += x[r];
        }
    }
    if constexpr (kGated)
        finish_one_gated<4>(e, type16_of(in_type, e), (int)m, n, v, u);
    else
        finish_one<4>(e, type16_of(in_type, e), (int)m, n, v);
}

int step_of(int in_type) { return in_type == kE4M3 ? 128 : 64; }
int size_of(int in_type) { return in_type == kE4M3 ? 1 : 2; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

Product product_of(const ProductCall& c) {
    Product a;
    a.p = static_cast<const char*>(c.p);
    a.q = static_cast<const char*>(c.q);
    a.ldp = c.ldp * size_of(c.in_type);
    a.ldq = c.ldq * size_of(c.in_type);
    a.M = c.M;
    a.K = c.K;
    a.R = c.R;
    a.tiles_m = a.tiles_n = 0;
    a.steps = (int)ceil_div(c.K, step_of(c.in_type));
    a.per_split = a.steps;
    a.e = c.e;
    return a;
}

template <int kIn, bool kGated>
hipError_t launch_rows_of(const Product& a, bool whole, hipStream_t s) {
    const int blocks = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const dim3 grid((unsigned)((a.e.N + 15) / 16));
#define BVML_FFN_ROWS(B)                                                                     \
    if (whole)                                                                               \
        hipLaunchKernelGGL((rows_kernel<kIn, B, kGated, true>), grid, dim3(B == 4 ? 512 : 1024), \
                           0, s, a);                                                         \
    else                                                                                     \
        hipLaunchKernelGGL((rows_kernel<kIn, B, kGated, false>), grid,                       \
                           dim3(B == 4 ? 512 : 1024), 0, s, a);
    if (blocks == 1) {
        BVML_FFN_ROWS(1)
    } else if (blocks == 2) {
        BVML_FFN_ROWS(2)
    } else {
        BVML_FFN_ROWS(4)
    }
#undef BVML_FFN_ROWS
    return hipGetLastError();
}

hipError_t launch_rows(const ProductCall& c, hipStream_t s) {
    const Product a = product_of(c);
    const bool whole = c.K % (16 / size_of(c.in_type)) == 0;
    if (c.gated) {
        if (c.in_type == kF16) return launch_rows_of<kF16, true>(a, whole, s);
        if (c.in_type == kBF16) return launch_rows_of<kBF16, true>(a, whole, s);
        return launch_rows_of<kE4M3, true>(a, whole, s);
    }
    if (c.in_type == kF16) return launch_rows_of<kF16, false>(a, whole, s);
    if (c.in_type == kBF16) return launch_rows_of<kBF16, false>(a, whole, s);
    return launch_rows_of<kE4M3, false>(a, whole, s);
}

}  // namespace

bool dma_fits(const ProductCall& c) {
    const int piece = 16 / size_of(c.in_type);
    // rows that begin on 16 bytes, and whole pieces along them
    if (!on16(c.p) || !on16(c.q) || c.ldp % piece != 0 || c.ldq % piece != 0) return false;
    if (c.layout == kForward) return c.K % piece == 0;
    const int along = c.layout == kInputGrad ? c.K : c.M;
    return (along % piece == 0 || c.padded_p) && c.R % piece == 0;
}

ProductPlan plan_product(int M, int R, int K, int in_type, int layout, bool gated, bool dma) {
    ProductPlan p{kTileRows, dma, 1};
    if (layout == kForward && M <= 64) return p;
    const int n = gated ? R / 2 : R;
    auto tiles = [&](int b) { return ceil_div(M, b) * ceil_div(n, gated ? b / 2 : b); };
    const long long steps = ceil_div(K, step_of(in_type));
    p.tile = !dma ? kTile128 : tiles(256) >= 160 ? kTile256 : tiles(128) >= 128 ? kTile128 : kTile64;
    const int b = p.tile == kTile256 ? 256 : p.tile == kTile128 ? 128 : 64;
    const long long room = p.tile == kTile256 ? 256 : 512;
    if (tiles(b) > 0 && tiles(b) * 2 <= room) {
        long long s = room / tiles(b);
        if (s > steps / 4) s = steps / 4;
        if (s > 16) s = 16;
        if (s > 1) p.splits = (int)ceil_div(steps, ceil_div(steps, s));
    }
    return p;
}

long long product_workspace(int M, int R, int K, int in_type, int layout, bool gated) {
    int splits = 1;
    for (const bool dma : {false, true}) {
        const ProductPlan p = plan_product(M, R, K, in_type, layout, gated, dma);
        if (p.splits > splits) splits = p.splits;
    }
    return splits > 1 ? (long long)splits * M * R * 4 : 0;
}

hipError_t launch_product(const ProductCall& c, void* workspace, hipStream_t s) {
    const ProductPlan p =
        plan_product(c.M, c.R, c.K, c.in_type, c.layout, c.gated, dma_fits(c));
    if (p.tile == kTileRows) return launch_rows(c, s);
    Product a = product_of(c);
    a.per_split = (int)ceil_div(a.steps, p.splits);
    if (p.splits > 1) a.e.part = static_cast<float*>(workspace);
    hipError_t err = c.in_type == kF16    ? launch_tiles_f16(a, p, c.layout, c.gated, s)
                     : c.in_type == kBF16 ? launch_tiles_bf16(a, p, c.layout, c.gated, s)
                                          : launch_tiles_e4m3(a, p, c.layout, c.gated, s);
    if (err != hipSuccess || p.splits == 1) return err;
    const long long threads = (long long)c.M * ((a.e.N + 3) / 4);
    const dim3 grid((unsigned)ceil_div(threads, 256));
    if (c.gated)
        hipLaunchKernelGGL(join_kernel<true>, grid, dim3(256), 0, s, a.e, c.in_type, p.splits);
    else
        hipLaunchKernelGGL(join_kernel<false>, grid, dim3(256), 0, s, a.e, c.in_type, p.splits);
    return hipGetLastError();
}

}  // namespace bvml_ffn
