// RMS norm with the residual's addition, and its gradient.
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   with n = s rstd and a = dy w:  ds = dstream + rstd (a - n mean(a n)),
//                                  dw = sum over rows of dy n
//
// Bound by memory: a row is read once into registers, its sum of squares (and
// for 8-bit output its largest magnitude) taken across the team of threads
// that hold it, and every output written from the registers.  Statistics and
// sums are fp32.  A team is a workgroup of a wave for every 512 columns; rows
// of one wave share a workgroup of four (BVML_FFN_TEAMS below, with the times).
//
// 4805 x 1280 from fp32 to 8 bits, the sum stored too: 14.7 us, 5.4 TB/s.  The
// gradient of 65541 x 1024: 119 us, 4.5 TB/s, with 5 of them the weight's sums.

#include "ffn_kernels.h"

namespace bvml_ffn {

namespace {

constexpr int kVec = 8;  // columns a thread takes at a time
constexpr float kE4M3Max = 448.0f;
constexpr float kTiny = 1.17549435e-38f;  // 2^-126
constexpr float kMost = 3.40282347e+38f;  // the largest finite number

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Across the team: every thread gets the sum (the largest).  `turn` picks the
// LDS slot, so that two reductions need one barrier each.
template <int kTeam, typename T, typename Op>
__device__ __forceinline__ T reduce(T v, Op op, T* slots) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = op(v, (T)__shfl_xor(v, d));
    if constexpr (kTeam > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[w] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int j = 1; j < kTeam / 64; ++j) v = op(v, slots[j]);
    }
    return v;
}

// A launch holds fewer than 2^32 threads along x: workgroups beyond kMostX go
// along y, and those beyond the last row return.
constexpr long long kMostX = 1 << 20;
dim3 grid_of(long long groups) {
    if (groups <= kMostX) return dim3((unsigned)groups);
    return dim3((unsigned)kMostX, (unsigned)((groups + kMostX - 1) / kMostX));
}

template <int kTeam, int kV>
__global__ __launch_bounds__(kTeam == 64 ? 256 : kTeam) void norm_kernel(NormCall c) {
    __shared__ float sum_slots[kTeam / 64];
    __shared__ uint32_t max_slots[kTeam / 64];
    const int t = threadIdx.x % kTeam;
    const long long group = (long long)blockIdx.y * kMostX + blockIdx.x;
    const long long row = kTeam == 64 ? group * 4 + (threadIdx.x >> 6) : group;
    if (row >= c.rows) return;  // whole teams
    float v[kV][kVec];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const int col = (k * kTeam + t) * kVec, left = c.cols - col;
        if (left > 0) {
            load_row<kVec>(c.x, c.x_type, row * c.ldx + col, left, v[k]);
            if (c.residual) {
                float r[kVec];
                load_row<kVec>(c.residual, c.x_type, row * c.ldr + col, left, r);
#pragma unroll
                for (int i = 0; i < kVec; ++i) v[k][i] += r[i];
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) sum += v[k][i] * v[k][i];
        }
    }
    sum = reduce<kTeam>(sum, [](float a, float b) { return a + b; }, sum_slots);
    const float rstd = 1.0f / __builtin_sqrtf(sum / (float)c.cols + c.eps);
    if (c.rstd && t == 0) c.rstd[row] = rstd;
    // the largest |y|, compared as bits: a NaN is above every number
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const int col = (k * kTeam + t) * kVec, left = c.cols - col;
        if (left > 0) {
            if (c.stream_out) store_row<kVec>(c.stream_out, c.x_type, row * c.lds + col, left, v[k]);
            float w[kVec];
            if (c.weight) {
                load_row<kVec>(c.weight, c.w_type, col, left, w);
            } else {
#pragma unroll
                for (int i = 0; i < kVec; ++i) w[i] = 1.0f;
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                v[k][i] = v[k][i] * rstd * w[i];
                if (i < left)
                    most = umax(most, __builtin_bit_cast(uint32_t, v[k][i]) & 0x7fffffffu);
            }
            if (c.y_type != kE4M3)
                store_row<kVec>(c.y, c.y_type, row * c.ldy + col, left, v[k]);
        }
    }
    if (c.y_type != kE4M3) return;
    most = reduce<kTeam>(most, umax, max_slots);
    const float top = __builtin_bit_cast(float, most) / kE4M3Max;
    const float scale = top < kTiny ? kTiny : top;  // (a NaN stays)
    if (t == 0) c.scale[row] = scale;
    // y / scale to nearest: the product with the rounded reciprocal, which alone
    // puts some ties a step apart, and what it leaves of y (16.7 us with the
    // quotient's own instructions for 4805 x 1280, 15.9 so).  An infinite scale
    // has quotients of 0: nothing is taken off.
    const float inverse = 1.0f / scale;
    const float minus = scale > kMost ? 0.0f : -scale;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const int col = (k * kTeam + t) * kVec, left = c.cols - col;
        if (left <= 0) continue;
        float q[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const float near = v[k][i] * inverse;
            q[i] = __builtin_fmaf(__builtin_fmaf(near, minus, v[k][i]), inverse, near);
        }
        int packed[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], 0, false);
            packed[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], p, true);
        }
        uint8_t* to = static_cast<uint8_t*>(c.y) + row * c.ldy + col;
        if (left >= kVec) {
            __builtin_memcpy(to, packed, 8);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (i < left) to[i] = (uint8_t)((uint32_t)packed[i / 4] >> (8 * (i % 4)));
        }
    }
}

// A team walks rows `teams` apart and keeps its columns' part of the weight's
// gradient in registers; a workgroup leaves one partial row, and a second
// launch sums those in their order: no atomics, equal bits for equal inputs.
template <int kTeam, int kV>
__global__ __launch_bounds__(kTeam == 64 ? 256 : kTeam) void norm_grad_kernel(NormGradCall c) {
    constexpr int kTeams = kTeam == 64 ? 4 : 1;
    __shared__ float slots[2][kTeam / 64];
    __shared__ float sums[kTeam == 64 ? 3 : 1][kTeam == 64 ? kV * 64 * kVec : 1];
    const int t = threadIdx.x % kTeam, team = kTeam == 64 ? threadIdx.x >> 6 : 0;
    float dw[kV][kVec];
#pragma unroll
    for (int k = 0; k < kV; ++k)
#pragma unroll
        for (int i = 0; i < kVec; ++i) dw[k][i] = 0.0f;
    int turn = 0;
    for (long long row = (long long)blockIdx.x * kTeams + team; row < c.rows;
         row += (long long)gridDim.x * kTeams) {
        float n[kV][kVec], a[kV][kVec];
        const float rstd = c.rstd[row];
        float dot = 0.0f;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const int col = (k * kTeam + t) * kVec, left = c.cols - col;
            if (left > 0) {
                float w[kVec];
                load_row<kVec>(c.dy, c.dy_type, row * c.lddy + col, left, a[k]);
                load_row<kVec>(c.stream_in, c.x_type, row * c.lds + col, left, n[k]);
                if (c.weight) {
                    load_row<kVec>(c.weight, c.w_type, col, left, w);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) w[i] = 1.0f;
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    n[k][i] *= rstd;
                    dw[k][i] += a[k][i] * n[k][i];
                    a[k][i] *= w[i];
                    dot += a[k][i] * n[k][i];
                }
            }
        }
        dot = reduce<kTeam>(dot, [](float x, float y) { return x + y; }, slots[turn]);
        turn ^= 1;
        const float mean = dot / (float)c.cols;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const int col = (k * kTeam + t) * kVec, left = c.cols - col;
            if (left > 0) {
                float d[kVec];
                if (c.dstream) {
                    load_row<kVec>(c.dstream, c.x_type, row * c.ldds + col, left, d);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) d[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) d[i] += rstd * (a[k][i] - n[k][i] * mean);
                store_row<kVec>(c.dx, c.x_type, row * c.lddx + col, left, d);
            }
        }
    }
    if (!c.dweight) return;
    if constexpr (kTeam == 64) {
        if (team != 0)
#pragma unroll
            for (int k = 0; k < kV; ++k)
#pragma unroll
                for (int i = 0; i < kVec; ++i) sums[team - 1][(k * 64 + t) * kVec + i] = dw[k][i];
        __syncthreads();
        if (team != 0) return;
#pragma unroll
        for (int k = 0; k < kV; ++k)
#pragma unroll
            for (int i = 0; i < kVec; ++i)
#pragma unroll
                for (int j = 0; j < 3; ++j) dw[k][i] += sums[j][(k * 64 + t) * kVec + i];
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const int col = (k * kTeam + t) * kVec, left = c.cols - col;
        if (left > 0)
            store_row<kVec>(c.workspace, kF32, (long long)blockIdx.x * c.cols + col, left, dw[k]);
    }
}

// How a row is dealt out, as (threads of a team, 8-column pieces of each): a
// wave for every 512 columns, so that a thread has one piece, a row's loads are
// all on their way at once, and the gradient, which holds four values a
// column, keeps its waves on the SIMD.  us, bf16, with what else could be:
//               1 x 1280  norm      192 threads 2.7   a wave, 3 pieces 4.2
//           16384 x 1280                        30.4                  31.5   256 threads 33.9
//           16384 x 2048            256         39.8          4       45.2
//            8192 x 2560            320         29.8  256, 2          31.1
//            4805 x 1280  gradient  192         21.6  64, 3           24.1
//            8192 x 2560            320         42.1  256, 2          52.8   512 threads 43.5
//            4096 x 5120            640         43.6  512, 2          57.3   1024 threads 60.2
// (and 512, 2 for the norm of 4096 x 5120: 31.9, 640 threads 33.0).  Up to
// 1,024 columns the norm's teams are of 128 (16384 x 1024: 22.3, a wave's two
// pieces 23.9; one row 2.6 and 3.3), the gradient's of a wave, four of which
// leave one partial row (37.4 with its sum, 38.8).
#define BVML_FFN_TEAMS(GO, UP_TO_1024)           \
    switch ((cols + 511) / 512) {                \
        case 0: case 1: GO(64, 1) break;         \
        case 2: UP_TO_1024 break;                \
        case 3: GO(192, 1) break;                \
        case 4: GO(256, 1) break;                \
        case 5: GO(320, 1) break;                \
        case 6: GO(384, 1) break;                \
        case 7: case 8: GO(512, 1) break;        \
        case 9: case 10: GO(640, 1) break;       \
        case 11: case 12: GO(768, 1) break;      \
        case 13: case 14: case 15: case 16:      \
            GO(1024, 1) break;                   \
        default:                                 \
            if (cols <= 16384) { GO(1024, 2) }   \
            else { GO(1024, 4) }                 \
    }

// Workgroups of the gradient: as many a CU as stay on it together, found by the
// step in time beyond them (8192 x 2560: 1,280 workgroups 42 us, 1,536 52; fewer
// hide less, 768 47), or one where rows are long and partial rows cost more
// (700 x 32000: 76 us, two 89).
int grad_blocks(int rows, int cols) {
    const int waves = (cols + 511) / 512;
    const int each = waves <= 2    ? 4
                     : waves == 3  ? 10
                     : waves == 4  ? 8
                     : waves <= 6  ? 5
                     : waves <= 8  ? 4
                     : waves <= 16 ? 2
                                   : 1;
    const int most = 256 * each;
    const long long teams = waves <= 2 ? (rows + 3LL) / 4 : rows;
    return teams < most ? (int)teams : most;
}

}  // namespace

hipError_t launch_norm(const NormCall& c, hipStream_t s) {
    const int cols = c.cols;
#define BVML_FFN_GO(T, V)                                                                 \
    hipLaunchKernelGGL((norm_kernel<T, V>), grid_of(T == 64 ? (c.rows + 3) / 4 : c.rows), \
                       dim3(T == 64 ? 256 : T), 0, s, c);
    BVML_FFN_TEAMS(BVML_FFN_GO, BVML_FFN_GO(128, 1))
#undef BVML_FFN_GO
    return hipGetLastError();
}

long long norm_grad_workspace(int rows, int cols) {
    return (long long)grad_blocks(rows, cols) * cols * 4;
}

hipError_t launch_norm_grad(const NormGradCall& c, hipStream_t s) {
    const int cols = c.cols, blocks = grad_blocks(c.rows, cols);
    if (blocks > 0) {
#define BVML_FFN_GO(T, V)                                                              \
    hipLaunchKernelGGL((norm_grad_kernel<T, V>), dim3((unsigned)blocks),               \
                       dim3(T == 64 ? 256 : T), 0, s, c);
        BVML_FFN_TEAMS(BVML_FFN_GO, BVML_FFN_GO(64, 2))
#undef BVML_FFN_GO
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return c.dweight ? launch_column_sum({c.workspace, blocks, cols, c.dweight, c.w_type}, s)
                     : hipSuccess;
}

}  // namespace bvml_ffn
