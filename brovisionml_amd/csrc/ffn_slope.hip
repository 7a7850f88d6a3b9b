// The activation's part of the gradients: dz from dy and the saved
// pre-activations, with the sums of dz's columns (the bias's gradient) on the
// way, and the sum of partial rows that this and the norm's gradient end with.
//
//   dz = dy act'(z), or [dh u act'(g), dh act(g)] with z = [g u]
//
// Bound by memory: dy and z are read once, dz written once; a workgroup takes
// 256 columns by a run of rows, keeps its columns' sums in fp32 registers and
// leaves one partial row.  Partial rows are summed in their order, so equal
// inputs give equal bits.  Gated 16389 x 4096, 671 MB: 119 us, 5.6 TB/s; 4805 x
// 5120, 148 MB: 32 us.
//
// dz is rounded to the operands' 16 bits, for the matrix cores multiply those:
// the gradients' error is that rounding beside their own (a factor of 1.4).

#include "ffn_kernels.h"
#include "ffn_sums.h"

namespace bvml_ffn {

namespace {

constexpr int kVec = 8;        // columns a thread
constexpr int kLanes = 32;     // threads along the columns
constexpr int kRows = 8;       // threads along the rows
constexpr int kMostParts = 256;
constexpr int kSumRuns = 32;

template <bool kGated, int kAhead>
__global__ __launch_bounds__(256) void slope_kernel(SlopeCall c, int rows_each) {
    constexpr int kHalves = kGated ? 2 : 1;
    __shared__ float sums[kRows][kHalves][kLanes * kVec];
    const int x = threadIdx.x % kLanes, y = threadIdx.x / kLanes;
    const int n = (blockIdx.x * kLanes + x) * kVec, left = c.N - n;
    const int R = kGated ? 2 * c.N : c.N;
    const int r0 = blockIdx.y * rows_each;
    // (the last run's end may be beyond what an int holds)
    const int r1 = c.rows - r0 < rows_each ? c.rows : r0 + rows_each;
    float s[kHalves][kVec];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < kVec; ++i) s[h][i] = 0.0f;
    if (left > 0) {
        // kAhead rows at a time, so that their loads are in flight together
        for (int r = r0 + y; r < r1; r += kRows * kAhead) {
            float dy[kAhead][kVec], z[kAhead][kVec], up[kGated ? kAhead : 1][kVec];
#pragma unroll
            for (int t = 0; t < kAhead; ++t) {
                const long long at = kAhead == 1 || r + t * kRows < r1 ? r + t * kRows : r;
                load_row<kVec>(c.dy, c.dy_type, at * c.lddy + n, left, dy[t]);
                if (kGated || c.z) load_row<kVec>(c.z, c.type, at * c.ldz + n, left, z[t]);
                if constexpr (kGated) load_row<kVec>(c.z, c.type, at * c.ldz + c.N + n, left, up[t]);
            }
#pragma unroll
            for (int t = 0; t < kAhead; ++t) {
                const long long at = r + t * kRows;
                if (kAhead > 1 && at >= r1) break;
                float d[kVec], du[kVec];
                // (the activations of the whole vector at once take fewer
                // branches but more registers, which the gated form has none
                // left of at 8 waves a SIMD: 16,389 x 8,192 119 us, 128 with
                // it; 4,805 x 5,120 ungated 34 without, 31 with it)
                if constexpr (kGated && kAhead == 1) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        float value, slope;
                        act_slope1(c.act, z[t][i], value, slope);
                        d[i] = dy[t][i] * up[t][i] * slope;
                        du[i] = dy[t][i] * value;
                    }
                } else {
                    float value[kVec], slope[kVec];
                    if (kGated || c.z) act_slope<kVec>(c.act, z[t], value, slope);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        d[i] = dy[t][i];
                        if (kGated || c.z) d[i] *= slope[i];
                        if constexpr (kGated) {
                            d[i] *= up[t][i];
                            du[i] = dy[t][i] * value[i];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    s[0][i] += d[i];
                    if constexpr (kGated) s[1][i] += du[i];
                }
                if (!c.dz) continue;
                store_row<kVec>(c.dz, c.type, at * c.ldd + n, left, d);
                if constexpr (kGated) store_row<kVec>(c.dz, c.type, at * c.ldd + c.N + n, left, du);
                // the zeros between the last column and the row's end
                if (left <= kVec)
                    for (int i = R; i < c.ldd; ++i)
                        static_cast<uint16_t*>(c.dz)[at * c.ldd + i] = 0;
            }
        }
    }
    if (!c.db) return;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < kVec; ++i) sums[y][h][x * kVec + i] = s[h][i];
    __syncthreads();
    const int col = blockIdx.x * kLanes * kVec + threadIdx.x;
    if (col >= c.N) return;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < kRows; ++j) t += sums[j][h][threadIdx.x];
        c.workspace[(long long)blockIdx.y * R + h * c.N + col] = t;
    }
}

__global__ __launch_bounds__(32 * kSumRuns) void column_sum_kernel(ColumnSum c) {
    __shared__ float sums[kSumRuns][32];
    column_sum<kSumRuns>(c, blockIdx.x, sums);
}

// (in 64 bits: rows may be close to the largest int)
long long rows_each_of(long long rows) {
    const long long each = (rows + kMostParts - 1) / kMostParts;
    const long long whole = (each + kRows - 1) / kRows * kRows;
    return whole < 16 ? 16 : whole;
}
int parts_of(long long rows) {
    const long long each = rows_each_of(rows);
    return (int)((rows + each - 1) / each);
}

}  // namespace

hipError_t launch_column_sum(const ColumnSum& c, hipStream_t s) {
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((c.cols + 31) / 32)), dim3(32 * kSumRuns),
                       0, s, c);
    return hipGetLastError();
}

long long slope_workspace(int rows, int R) {
    return (long long)parts_of(rows) * R * 4;
}

hipError_t launch_slope(const SlopeCall& c, ColumnSum* sums, hipStream_t s) {
    const int each = (int)rows_each_of(c.rows), parts = parts_of(c.rows);
    const int R = c.gated ? 2 * c.N : c.N;
    *sums = {c.workspace, parts, R, c.db, c.type};
    if (parts == 0) return hipSuccess;
    const dim3 grid((unsigned)((c.N + kLanes * kVec - 1) / (kLanes * kVec)), (unsigned)parts);
    // two rows at a time where the workgroups do not fill the card: 1,205 x
    // 5,460 gated 15 to 12 us, but 16,389 x 8,192 120 to 135
    const bool few = (long long)grid.x * grid.y < 1024;
#define BVML_FFN_SLOPE(G, A) \
    hipLaunchKernelGGL((slope_kernel<G, A>), grid, dim3(256), 0, s, c, each)
    if (c.gated) {
        if (few) BVML_FFN_SLOPE(true, 2);
        else BVML_FFN_SLOPE(true, 1);
    } else {
        if (few) BVML_FFN_SLOPE(false, 2);
        else BVML_FFN_SLOPE(false, 1);
    }
#undef BVML_FFN_SLOPE
    return hipGetLastError();
}

}  // namespace bvml_ffn
