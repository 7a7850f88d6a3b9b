// Which kernel a product takes, the two kernels for few rows, and the second
// launch that joins a split sum.

#include "ffn_kernels.h"
#include "ffn_product.h"

namespace bvml_ffn {

namespace {

// 16 bytes of a row from element k on: zeros beyond its end (`end` 0 for no
// row at all, so that absent rows cost no loads).
template <int kSize, bool kWhole>
__device__ __forceinline__ v4i row_piece(const char* at, int k, int end) {
    constexpr int kPiece = 16 / kSize;
    v4i v = {0, 0, 0, 0};
    const int n = end - k;
    if (n >= kPiece) {
        __builtin_memcpy(&v, at + (long long)k * kSize, 16);
    } else if (!kWhole && n > 0) {
        at = apart(at);
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
}

// ---------------------------------------------------------------------------
// few rows (5 to 32, serving): the weights are read once, by workgroups of 8
// waves that share 16 rows of W (gated: 16 of each half) and divide k; their
// sums meet in LDS.  Bound by reading W and, at these sizes, by the latency of
// doing so: every lane has its 16-byte pieces of kAhead k groups in flight,
// and what the epilogue adds is asked for first.  The matrix instruction's
// other operand holds up to 16 rows of x.  Every workgroup reads all of x, a
// 64-byte run of a row at a time, which is what more rows cost.  Weights from
// memory: 16 x 4096 x 4096 10.8 us, 3.1 TB/s; 16 x 1280 x 1280 4.7.  (16 waves:
// 16 x 5120 x 1280 11.0 us for 11.2, 12 x 1024 x 1024 3.8 for 3.6: not kept.)
// ---------------------------------------------------------------------------
constexpr int kRowsWaves = 8;

template <int kIn, int kBlocks, bool kGated, bool kWhole>
__global__ __launch_bounds__(64 * kRowsWaves) void rows_kernel(Product a) {
    constexpr int kHalves = kGated ? 2 : 1, kWaves = kRowsWaves;
    constexpr int kSize = kIn == kE4M3 ? 1 : 2, kPiece = 16 / kSize, kStep = 128 / kSize;
    constexpr int kAhead = kBlocks > 1 || kGated ? 2 : 5;
    __shared__ v4f sums[kWaves][kHalves][kBlocks][64];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int g = lane >> 4, i16 = lane & 15;
    const int N = a.e.N, n0 = blockIdx.x * 16;
    const int row = n0 + i16 < N ? n0 + i16 : N - 1;
    const char* q[kHalves];
    const char* p[kBlocks];
    int pend[kBlocks];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) q[h] = a.q + (long long)(row + h * N) * a.ldq;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const int m = 16 * b + i16;
        p[b] = a.p + (long long)(m < a.M ? m : a.M - 1) * a.ldp;
        pend[b] = m < a.M ? a.K : 0;
    }
    v4f acc[kHalves][kBlocks];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[h][b] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    // wave b finishes rows 16 b .. of x
    const int type16 = type16_of(kIn, a.e), m = 16 * w + i16, n = n0 + 4 * g;
    Single<4, kGated> terms;
    if (w < kBlocks) terms.load(a.e, type16, m, n);
    for (int s = w; s < a.steps; s += kWaves * kAhead) {
        v4i qv[kAhead][kHalves][2], pv[kAhead][kBlocks][2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (s + u * kWaves) * kStep + g * kPiece;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int h = 0; h < kHalves; ++h) qv[u][h][c] = row_piece<kSize, kWhole>(q[h], k + c * 4 * kPiece, a.K);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) pv[u][b][c] = row_piece<kSize, kWhole>(p[b], k + c * 4 * kPiece, pend[b]);
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
    float v[2][4];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        v4f t = sums[0][h][w][lane];
#pragma unroll
        for (int j = 1; j < kWaves; ++j) t += sums[j][h][w][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[h][r] = t[r];
    }
    terms.finish(a.e, type16, m, n, v[0], v[1]);
}

// ---------------------------------------------------------------------------
// one to four rows: a wave takes kRows rows of W (gated: of each half) and the
// lanes their k, 16 adjacent bytes a lane, so that every load is whole cache
// lines of one row and the work spreads over every CU.  Products and sums
// are fp32 on the vector units: at so few rows the weights' way from memory
// is all that counts.  Weights from memory: 1 x 4096 x 4096 7.6 us, 4.4 TB/s;
// 1 x 5120 x 1280 5.1.  The kernel above takes 7.7 for 4.6 with the latter in the
// caches, and wins from 5 rows on (8 x 1280 x 5120: 6.1 us, this one 7.9).
// ---------------------------------------------------------------------------
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// c + the 4 bytes' products
template <int kIn>
__device__ __forceinline__ float dot4(int a, int b, float c) {
    if constexpr (kIn == kBF16) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, a),
                                               __builtin_bit_cast(v2b, b), c, false);
    } else if constexpr (kIn == kF16) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, a), __builtin_bit_cast(v2h, b), c,
                                      false);
    } else {
        const v2f a0 = __builtin_amdgcn_cvt_pk_f32_fp8(a, false);
        const v2f a1 = __builtin_amdgcn_cvt_pk_f32_fp8(a, true);
        const v2f b0 = __builtin_amdgcn_cvt_pk_f32_fp8(b, false);
        const v2f b1 = __builtin_amdgcn_cvt_pk_f32_fp8(b, true);
        c = __builtin_fmaf(a0[0], b0[0], c);
        c = __builtin_fmaf(a0[1], b0[1], c);
        c = __builtin_fmaf(a1[0], b1[0], c);
        return __builtin_fmaf(a1[1], b1[1], c);
    }
}

// The wave's sum, to every lane: within rows of 16 lanes, then across them.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                             0, __builtin_bit_cast(int, v), kCtrl, kRowMask, 0xf,
                                             kRowMask == 0xf));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast 15 to rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);  // row_bcast 31 to rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <int kIn, int kM, int kRows, bool kGated, bool kWhole>
__global__ __launch_bounds__(256) void dot_kernel(Product a) {
    constexpr int kHalves = kGated ? 2 : 1;
    constexpr int kSize = kIn == kE4M3 ? 1 : 2, kPiece = 16 / kSize;
    constexpr int kAhead = kM * kHalves * kRows >= 8 ? 3 : 5;
    const int lane = threadIdx.x & 63;
    const int N = a.e.N, n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows;
    if (n0 >= N) return;
    const char* q[kHalves][kRows];
    const char* p[kM];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            q[h][r] = a.q + (long long)((n0 + r < N ? n0 + r : N - 1) + h * N) * a.ldq;
#pragma unroll
    for (int m = 0; m < kM; ++m) p[m] = a.p + (long long)(m < a.M ? m : a.M - 1) * a.ldp;
    // lane m kRows + r finishes row m, column n0 + r
    const int type16 = type16_of(kIn, a.e), mine = lane / kRows, n = n0 + lane % kRows;
    Single<1, kGated> terms;
    if (mine < kM) terms.load(a.e, type16, mine, n);
    float acc[kHalves][kM][kRows];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int r = 0; r < kRows; ++r) acc[h][m][r] = 0.0f;

    for (int k0 = lane * kPiece; k0 < a.K; k0 += 64 * kPiece * kAhead) {
        v4i qv[kAhead][kHalves][kRows], pv[kAhead][kM];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = k0 + u * 64 * kPiece;
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    qv[u][h][r] = row_piece<kSize, kWhole>(q[h][r], k, a.K);
#pragma unroll
            for (int m = 0; m < kM; ++m) pv[u][m] = row_piece<kSize, kWhole>(p[m], k, a.K);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int m = 0; m < kM; ++m)
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[h][m][r] = dot4<kIn>(qv[u][h][r][i], pv[u][m][i], acc[h][m][r]);
    }
    float v[1] = {0.0f}, w[1] = {0.0f};
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float t = wave_sum(acc[h][m][r]);
                if (lane == m * kRows + r) (h ? w : v)[0] = t;
            }
    if (mine < kM) terms.finish(a.e, type16, mine, n, v, w);
}

// Sums the parts of the split tiles, in their order, and finishes them: a
// thread 8 columns of a row, blockIdx.y the tile.  Bound by latency, so eight
// loads of parts are on their way together: 4 tiles of 256 x 256 in 16 parts 6 us,
// 10 one part after another; 64 x 1280 in 10 parts 4.7 and 5.4 (gated, twice the
// values a part: four parts 5.7, eight 7.4).  The order is fixed, so equal
// inputs give equal bits; atomic sums would not.
template <bool kGated>
__global__ __launch_bounds__(256) void join_kernel(Product a, int in_type, int bm, int bn) {
    constexpr int kHalves = kGated ? 2 : 1, kInFlight = 8 / kHalves;  // parts on their way
    const int cols = kGated ? bn / 2 : bn, per = cols / 8;
    const int t = blockIdx.x * 256 + threadIdx.x;
    const int row = t / per, col = t % per * 8;
    if (row >= bm) return;
    int tm, tn;
    tile_of(a.whole + blockIdx.y, a.tiles_m, a.tiles_n, tm, tn);
    const int m = tm * bm + row, n = tn * cols + col;
    if (m >= a.M || n >= a.e.N) return;
    const float* from = a.e.part + (long long)blockIdx.y * a.splits * bm * bn + row * bn + col;
    const int type16 = type16_of(in_type, a.e);
    Single<8, kGated> terms;
    terms.load(a.e, type16, m, n);
    v4f sum[kHalves][2] = {};
    for (int s = 0; s < a.splits; s += kInFlight) {
        v4f x[kInFlight][kHalves][2];
#pragma unroll
        for (int t = 0; t < kInFlight; ++t) {
            // beyond the last: that one again, not added
            const int at = s + t < a.splits ? s + t : a.splits - 1;
            const v4f* const p = reinterpret_cast<const v4f*>(from + (long long)at * bm * bn);
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[t][h][i] = p[h * (cols / 4) + i];
        }
#pragma unroll
        for (int t = 0; t < kInFlight; ++t) {
            const bool in = s + t < a.splits;
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[h][i][j] += in ? x[t][h][i][j] : 0.0f;
        }
    }
    float v[8], u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = sum[0][i / 4][i % 4];
        u[i] = sum[kHalves - 1][i / 4][i % 4];
    }
    terms.finish(a.e, type16, m, n, v, u);
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
    a.whole = 0;
    a.splits = 1;
    a.per_split = a.steps;
    a.e = c.e;
    return a;
}

template <int kIn, int kBlocks, bool kGated>
hipError_t launch_rows_one(const Product& a, bool whole, hipStream_t s) {
    const dim3 grid((unsigned)((a.e.N + 15) / 16)), block(64 * kRowsWaves);
    if (whole)
        hipLaunchKernelGGL((rows_kernel<kIn, kBlocks, kGated, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((rows_kernel<kIn, kBlocks, kGated, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <int kIn, int kM, int kRows, bool kGated>
hipError_t launch_dot_one(const Product& a, bool whole, hipStream_t s) {
    const dim3 grid((unsigned)((a.e.N + 4 * kRows - 1) / (4 * kRows))), block(256);
    if (whole)
        hipLaunchKernelGGL((dot_kernel<kIn, kM, kRows, kGated, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((dot_kernel<kIn, kM, kRows, kGated, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <int kIn, bool kGated>
hipError_t launch_rows_of(const Product& a, bool whole, hipStream_t s) {
    if (a.M == 1) return launch_dot_one<kIn, 1, 1, kGated>(a, whole, s);
    if (a.M == 2) return launch_dot_one<kIn, 2, 1, kGated>(a, whole, s);
    if (a.M <= 4) {
        // A wave of two columns reads x half as often, and that is what counts
        // from 3 rows on, once two workgroups a CU are left: 4 x 1280 x 8192 7.3
        // to 6.3 us; 1 x 1280 x 5120 takes 4.3 either way, and 4 x 5120 x 2048 7.3
        // for 6.5.  Gated waves have two columns as it is: four take 4 x 1280 x 5120
        // from 7.3 to 7.6 (all with the weights in the caches; from memory the
        // latter takes 10.5).
        if constexpr (!kGated) {
            if (a.e.N >= 4096) return launch_dot_one<kIn, 4, 2, kGated>(a, whole, s);
        }
        return launch_dot_one<kIn, 4, 1, kGated>(a, whole, s);
    }
    return a.M <= 16 ? launch_rows_one<kIn, 1, kGated>(a, whole, s)
                     : launch_rows_one<kIn, 2, kGated>(a, whole, s);
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

namespace {

// What a tile costs, in us, measured on bf16 products of 1,280 to 8,192 terms
// (8-bit ones are chosen by the same figures):
// `fixed` for its first copies and its epilogue, `step` for 128 bytes of k with
// the card full and `idle` with half of that at most.
// `room`: workgroups on the card at once, one or two a CU.
// `across`: what an operand read across its rows adds to a step.
struct TileCost {
    int bm, bn, room;
    double fixed, step, idle, across;
};
constexpr TileCost kCosts[] = {
    {256, 256, 256, 9.0, 1.42, 1.03, 0.06},  // 4096^2 x 8192 at 1350 TFLOP/s
    {128, 128, 512, 5.0, 0.87, 0.65, 0.12},  // 1130
    {128, 128, 256, 4.0, 0.47, 0.45, 0.12},  // 2048^2 x 5120: 45 us, 59 with two slots
    {64, 128, 512, 3.0, 0.55, 0.33, 0.12},   // 2048 x 1024 x 5120: 29 us, 34 with 64 x 64
    {64, 64, 512, 2.8, 0.40, 0.19, 0.09},    // 512 x 1280 x 5120: 18 us, 26 with 64 x 128
};
// The two of them that also copy through registers, then: a step's copies wait
// for their loads (64 x 5120 x 1280: 22 us in one part, 64 x 64 tiles 15).
constexpr TileCost kCopied128{128, 128, 512, 4.9, 1.20, 0.87, 0.03};
constexpr TileCost kCopiedSquare{64, 64, 512, 3.3, 0.66, 0.58, 0.10};

// With part of the card's room taken, 0 to 1.  Up to one workgroup a CU costs
// `idle`; the first second one makes its CU the last to finish (64 x 64 tiles
// of 5,120 terms: 256 of them 19 us, 384 33, 512 34).  Where one fills a CU, the
// step grows with the CUs at work.
double step_cost(const TileCost& c, double full) {
    if (full <= 0.5) return c.idle;
    const double over = 2.0 * full - 1.0;
    return c.idle + (c.step - c.idle) * (c.room > 256 ? 0.8 + 0.2 * over : over);
}
// The few-rows kernel: always up to kDotRows rows, possible up to kFewRows. Its
// cost from 5 rows on, measured as above: rounds of a workgroup a CU, a step of
// which takes longer with every row (16 x 4096 x 4096: 10.9 us, 32 rows 14.4).  The
// tiles' costs are of operands that the caches hold; so few rows' weights
// mostly come from memory, which takes a tile's first steps kCold longer.
constexpr int kDotRows = 4, kFewRows = 32;
constexpr double kCold = 1.2;
double rows_cost(int M, int n, long long steps, bool gated) {
    const double step = gated ? 0.15 + 0.0027 * M + (M > 16 ? 0.022 : 0.0)
                              : 0.095 + 0.0024 * M + (M > 16 ? 0.015 : 0.0);
    return (gated ? 2.75 : 2.5) + ceil_div(n, 16 * 256) * steps * step;
}
// A second launch, and a byte of a part written and read.
constexpr double kJoin = 5.0, kJoinBytes = 8.0 / 4e6;

ProductPlan search_product(int M, int R, int K, int in_type, int layout, bool gated, bool dma) {
    const int n = gated ? R / 2 : R;
    const long long steps = ceil_div(K, step_of(in_type));
    ProductPlan best{kTile128, dma, 0, 1};
    double least = 1e30;
    if (layout == kForward && M <= kFewRows) {
        // (without direct copies the tiles lose to it at all of these rows)
        best = {kTileRows, dma, 0, 1};
        if (!dma || M <= kDotRows) return best;
        least = rows_cost(M, n, steps, gated) - kCold;
    }
    for (int tile = kTile256; tile <= kTileSquare; ++tile) {
        if (gated && tile == kTileSquare) continue;
        if (!dma && tile != kTile128 && tile != kTileSquare) continue;
        const TileCost& c = dma                ? kCosts[tile]
                            : tile == kTile128 ? kCopied128
                                               : kCopiedSquare;
        const long long tiles = ceil_div(M, c.bm) * ceil_div(n, gated ? c.bn / 2 : c.bn);
        // rounds of a full card, then what is left over: one workgroup a tile
        // or, where that leaves CUs idle, several that share its terms
        const long long left = tiles % c.room;
        const double slower = 1.0 + layout * c.across;
        const double rounds = (double)(tiles / c.room) * (c.fixed + steps * c.step * slower);
        for (int s = 1; s <= 64; ++s) {
            if (s > 1 && (left * s > c.room || steps < 4 * s)) break;
            const long long each = ceil_div(steps, s);
            if (s > 1 && ceil_div(steps, each) != s) continue;  // a part with nothing
            double t = rounds;
            if (left > 0) {
                const double full = (double)(left * s) / c.room;
                t += c.fixed + each * step_cost(c, full) * slower;
            }
            if (s > 1) t += kJoin + (double)(left * s) * c.bm * c.bn * kJoinBytes;
            if (t < least) {
                least = t;
                best = {tile, dma, (int)(s > 1 ? tiles - left : tiles), s};
            }
        }
    }
    return best;
}

}  // namespace

// (A call asks three times, for its workspace with and without direct copies
// and for its launch, and a search takes 0.4 us: a thread keeps its last
// plans, by their sizes.)
ProductPlan plan_product(int M, int R, int K, int in_type, int layout, bool gated, bool dma) {
    if (layout == kForward && M <= kDotRows) return {kTileRows, dma, 0, 1};
    struct Known {
        int M, R, K, kind;
        ProductPlan plan;
    };
    thread_local Known known[64] = {};
    const int kind = ((in_type * 4 + layout) * 2 + gated) * 2 + dma;
    const unsigned h = (unsigned)M * 31u + (unsigned)R * 17u + (unsigned)K + (unsigned)kind;
    Known& k = known[h % 64u];
    if (k.M != M || k.R != R || k.K != K || k.kind != kind)
        k = {M, R, K, kind, search_product(M, R, K, in_type, layout, gated, dma)};
    return k.plan;
}

namespace {
long long parts_of(int M, int R, bool gated, const ProductPlan& p) {
    if (p.tile == kTileRows || p.splits == 1) return 0;
    const TileCost& c = kCosts[p.tile];
    const int n = gated ? R / 2 : R;
    return ceil_div(M, c.bm) * ceil_div(n, gated ? c.bn / 2 : c.bn) - p.whole;
}
}  // namespace

long long product_workspace(int M, int R, int K, int in_type, int layout, bool gated) {
    long long most = 0;
    for (const bool dma : {false, true}) {
        const ProductPlan p = plan_product(M, R, K, in_type, layout, gated, dma);
        const long long parts = parts_of(M, R, gated, p) * p.splits;
        if (parts == 0) continue;
        const long long bytes = parts * kCosts[p.tile].bm * kCosts[p.tile].bn * 4;
        if (bytes > most) most = bytes;
    }
    return most;
}

namespace {

// A product's tiles as the plan has them.
void lay_out(Product& a, const ProductCall& c, int tile, int whole, int splits, void* workspace) {
    const TileCost& t = kCosts[tile];
    a.tiles_m = (int)ceil_div(c.M, t.bm);
    a.tiles_n = (int)ceil_div(c.gated ? c.R / 2 : c.R, c.gated ? t.bn / 2 : t.bn);
    a.whole = whole;
    a.splits = splits;
    a.per_split = (int)ceil_div(a.steps, splits);
    a.e.part = static_cast<float*>(workspace);
}

hipError_t join(const Product& a, const ProductCall& c, int tile, hipStream_t s) {
    const long long parts = (long long)a.tiles_m * a.tiles_n - a.whole;
    if (parts == 0) return hipSuccess;
    const TileCost& t = kCosts[tile];
    const int cols = c.gated ? t.bn / 2 : t.bn;
    const dim3 grid((unsigned)ceil_div(t.bm * cols / 8, 256), (unsigned)parts);
    if (c.gated)
        hipLaunchKernelGGL(join_kernel<true>, grid, dim3(256), 0, s, a, c.in_type, t.bm, t.bn);
    else
        hipLaunchKernelGGL(join_kernel<false>, grid, dim3(256), 0, s, a, c.in_type, t.bm, t.bn);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_product(const ProductCall& c, void* workspace, hipStream_t s) {
    const ProductPlan p =
        plan_product(c.M, c.R, c.K, c.in_type, c.layout, c.gated, dma_fits(c));
    if (p.tile == kTileRows) return launch_rows(c, s);
    Product a = product_of(c);
    lay_out(a, c, p.tile, p.whole, p.splits, workspace);
    const hipError_t e = c.in_type == kF16    ? launch_tiles_f16(a, p, c.layout, c.gated, s)
                         : c.in_type == kBF16 ? launch_tiles_bf16(a, p, c.layout, c.gated, s)
                                              : launch_tiles_e4m3(a, p, c.layout, c.gated, s);
    return e == hipSuccess ? join(a, c, p.tile, s) : e;
}

namespace {

// When n1 jobs of t1 and then n2 of t2 <= t1 are done on `room` slots, each
// slot taking the next job as it comes free.
double done_by(long long n1, double t1, long long n2, double t2, int room) {
    const long long a = n1 / room, over = n1 % room;
    const double early = a * t1, late = over > 0 ? early + t1 : early;
    // room - over slots come free at `early`, the others at `late`; what fits by T
    auto fit = [&](double T) {
        const double x = (T - early) / t2 + 1e-9, y = (T - early - t1) / t2 + 1e-9;
        return (room - over) * (x > 0 ? (long long)x : 0) + over * (y > 0 ? (long long)y : 0);
    };
    if (fit(late) >= n2) return late;
    // T one job after a slot of either kind came free
    double best = 1e30;
    for (int kind = 0; kind < (over > 0 ? 2 : 1); ++kind) {
        const double from = kind == 0 ? early : early + t1;
        long long lo = 0, hi = n2 / (over > 0 && kind == 1 ? over : room - over) + 1;
        while (lo < hi) {
            const long long k = (lo + hi) / 2;
            if (fit(from + k * t2) >= n2) hi = k;
            else lo = k + 1;
        }
        const double T = from + lo * t2;
        if (T < best) best = T;
    }
    return best > late ? best : late;
}

GradientsPlan search_gradients(int M, int R, int K) {
    static const int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    GradientsPlan best{kTile128, false, 0, 1, 0, 1};
    double least = 1e30;
    const long long si = ceil_div(R, 64), sw = ceil_div(M, 64);  // steps of a tile
    for (int tile = kTile256; tile <= kTileSquare; ++tile) {
        const TileCost& c = kCosts[tile];
        const double bytes = (double)c.bm * c.bn * kJoinBytes;
        const long long cols = ceil_div(K, c.bn);
        const long long ti = ceil_div(M, c.bm) * cols, tw = ceil_div(R, c.bm) * cols;
        auto time = [&](long long steps, int across) {
            return c.fixed + steps * c.step * (1.0 + across * c.across);
        };
        auto may = [&](long long tiles, long long steps, int s) {
            return s == 1 || (steps >= 4 * s && ceil_div(steps, ceil_div(steps, s)) == s &&
                              tiles * s <= 2 * c.room);
        };
        // every tile of a product in s parts
        for (const int a : kSplits) {
            if (!may(ti, si, a)) continue;
            for (const int b : kSplits) {
                if (!may(tw, sw, b)) continue;
                const double x = time(ceil_div(si, a), 1), w = time(ceil_div(sw, b), 2);
                double t = w > x ? done_by(tw * b, w, ti * a, x, c.room)
                                 : done_by(ti * a, x, tw * b, w, c.room);
                if (a > 1) t += kJoin + ti * a * bytes;
                if (b > 1) t += kJoin + tw * b * bytes;
                if (t < least) {
                    least = t;
                    best = {tile, w > x, a > 1 ? 0 : (int)ti, a, b > 1 ? 0 : (int)tw, b};
                }
            }
        }
        // or the shorter product's last tiles, those beyond whole rounds
        const double x = time(si, 1), w = time(sw, 2);
        const bool first = w > x;
        const long long longs = first ? tw : ti, shorts = first ? ti : tw;
        const long long steps = first ? si : sw;
        for (long long rest = 1; rest < shorts && rest <= c.room / 2; rest += rest < 8 ? 1 : rest / 4) {
            const double t0 = done_by(longs, first ? w : x, shorts - rest, first ? x : w, c.room);
            if (t0 >= least) continue;
            for (const int s : kSplits) {
                if (s == 1 || !may(rest, steps, s)) continue;
                const double one = time(ceil_div(steps, s), first ? 1 : 2);
                const double t = t0 + one * ceil_div(rest * s, c.room) + kJoin + rest * s * bytes;
                if (t < least) {
                    least = t;
                    best = first ? GradientsPlan{tile, true, (int)(ti - rest), s, (int)tw, 1}
                                 : GradientsPlan{tile, false, (int)ti, 1, (int)(tw - rest), s};
                }
            }
        }
    }
    return best;
}

}  // namespace

// (The search takes some tens of microseconds: a thread keeps its last plans,
// by their sizes.)
GradientsPlan plan_gradients(int M, int R, int K) {
    struct Known {
        int M, R, K;
        GradientsPlan plan;
    };
    thread_local Known known[64] = {};
    Known& k = known[((unsigned)M * 31u + (unsigned)R * 17u + (unsigned)K) % 64u];
    if (k.M != M || k.R != R || k.K != K) k = {M, R, K, search_gradients(M, R, K)};
    return k.plan;
}

namespace {
long long part_bytes(long long tiles, int whole, int splits, int tile) {
    return splits == 1 ? 0 : (tiles - whole) * splits * kCosts[tile].bm * kCosts[tile].bn * 4;
}
}  // namespace

long long gradients_workspace(int M, int R, int K) {
    if (M == 0) return 0;
    const GradientsPlan p = plan_gradients(M, R, K);
    const TileCost& c = kCosts[p.tile];
    const long long cols = ceil_div(K, c.bn);
    return part_bytes(ceil_div(M, c.bm) * cols, p.input_whole, p.input_splits, p.tile) +
           part_bytes(ceil_div(R, c.bm) * cols, p.weight_whole, p.weight_splits, p.tile);
}

hipError_t launch_gradients(const ProductCall& input, const ProductCall& weight,
                            const ColumnSum& sums, void* workspace, hipStream_t s) {
    auto apart = [&]() {
        hipError_t e = sums.out ? launch_column_sum(sums, s) : hipSuccess;
        if (e == hipSuccess && input.M > 0) e = launch_product(input, workspace, s);
        return e == hipSuccess ? launch_product(weight, workspace, s) : e;
    };
    if (input.M == 0 || !dma_fits(input) || !dma_fits(weight)) return apart();
    const GradientsPlan p = plan_gradients(input.M, input.K, input.R);
    Gradients g{product_of(input), product_of(weight), p.weight_first, sums};
    lay_out(g.input, input, p.tile, p.input_whole, p.input_splits, workspace);
    const long long ti = (long long)g.input.tiles_m * g.input.tiles_n;
    lay_out(g.weight, weight, p.tile, p.weight_whole, p.weight_splits,
            static_cast<char*>(workspace) + part_bytes(ti, p.input_whole, p.input_splits, p.tile));
    if (groups_of(g) > kMostGroups) return apart();
    hipError_t e = input.in_type == kF16 ? launch_gradients_f16(g, p.tile, s)
                                         : launch_gradients_bf16(g, p.tile, s);
    if (e == hipSuccess) e = join(g.input, input, p.tile, s);
    if (e == hipSuccess) e = join(g.weight, weight, p.tile, s);
    return e;
}

}  // namespace bvml_ffn
