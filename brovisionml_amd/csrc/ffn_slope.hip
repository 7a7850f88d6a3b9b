// The activation's part of the gradients: dz from dy and the saved
// pre-activations, with the sums of dz's columns (the bias's gradient) on the
// way, and the sum of partial rows that this and the norm's gradient end with.
//
// Bound by memory: dy and z are read once, dz written once; a workgroup takes
// 256 columns by a run of rows, keeps its columns' sums in fp32 registers and
// leaves one partial row.  Partial rows are summed in their order, so equal
// inputs give equal bits.

#include "ffn_kernels.h"

namespace bvml_ffn {

namespace {

constexpr int kVec = 8;        // columns a thread
constexpr int kLanes = 32;     // threads along the columns
constexpr int kRows = 8;       // threads along the rows
constexpr int kMostParts = 256;

template <bool kGated>
__global__ __launch_bounds__(256) void slope_kernel(SlopeCall c, int rows_each) {
    constexpr int kHalves = kGated ? 2 : 1;
    __shared__ float sums[kRows][kHalves][kLanes * kVec];
    const int x = threadIdx.x % kLanes, y = threadIdx.x / kLanes;
    const int n = (blockIdx.x * kLanes + x) * kVec, left = c.N - n;
    const int R = kGated ? 2 * c.N : c.N;
    const int r0 = blockIdx.y * rows_each;
    const int r1 = r0 + rows_each < c.rows ? r0 + rows_each : c.rows;
    float s[kHalves][kVec];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < kVec; ++i) s[h][i] = 0.0f;
    if (left > 0) {
        for (int r = r0 + y; r < r1; r += kRows) {
            float dy[kVec], z[kVec], d[kVec];
            load_row<kVec>(c.dy, c.dy_type, (long long)r * c.lddy + n, left, dy);
            if constexpr (kGated) {
                float up[kVec], du[kVec];
                load_row<kVec>(c.z, c.type, (long long)r * c.ldz + n, left, z);
                load_row<kVec>(c.z, c.type, (long long)r * c.ldz + c.N + n, left, up);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    float value, slope;
                    act_slope1(c.act, z[i], value, slope);
                    d[i] = dy[i] * up[i] * slope;
                    du[i] = dy[i] * value;
                    s[0][i] += d[i];
                    s[1][i] += du[i];
                }
                if (c.dz) {
                    store_row<kVec>(c.dz, c.type, (long long)r * c.ldd + n, left, d);
                    store_row<kVec>(c.dz, c.type, (long long)r * c.ldd + c.N + n, left, du);
                }
            } else {
                if (c.z) load_row<kVec>(c.z, c.type, (long long)r * c.ldz + n, left, z);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    float value, slope = 1.0f;
                    if (c.z) act_slope1(c.act, z[i], value, slope);
                    d[i] = dy[i] * slope;
                    s[0][i] += d[i];
                }
                if (c.dz) store_row<kVec>(c.dz, c.type, (long long)r * c.ldd + n, left, d);
            }
            // the zeros between the last column and the row's end
            if (c.dz && left <= kVec)
                for (int i = R; i < c.ldd; ++i)
                    static_cast<uint16_t*>(c.dz)[(long long)r * c.ldd + i] = 0;
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

// out[c] = sum over the parts: 32 interleaved runs of them, then the runs.
// Bound by latency: a thread has eight of its loads in flight (1,024 rows of
// 1,024 columns: 39 us with one at a time by 8 runs).
constexpr int kRuns = 32, kInFlight = 8;
__global__ __launch_bounds__(32 * kRuns) void column_sum_kernel(const float* part, int parts,
                                                                int cols, void* out, int type) {
    __shared__ float sums[kRuns][32];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    const int col = blockIdx.x * 32 + x;
    float t = 0.0f;
    if (col < cols) {
        const float* p = part + col;
        int r = y;
        for (; r + (kInFlight - 1) * kRuns < parts; r += kInFlight * kRuns) {
            float v[kInFlight];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) v[i] = p[(long long)(r + i * kRuns) * cols];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) t += v[i];
        }
        for (; r < parts; r += kRuns) t += p[(long long)r * cols];
    }
    sums[y][x] = t;
    __syncthreads();
    if (y != 0 || col >= cols) return;
#pragma unroll
    for (int j = 1; j < kRuns; ++j) t += sums[j][x];
    if (type == kF32)
        static_cast<float*>(out)[col] = t;
    else
        static_cast<uint16_t*>(out)[col] = to16(t, type);
}

int rows_each_of(int rows) {
    const int each = (rows + kMostParts - 1) / kMostParts;
    const int whole = (each + kRows - 1) / kRows * kRows;
    return whole < 32 ? 32 : whole;
}

}  // namespace

hipError_t launch_column_sum(const float* part, int parts, int cols, void* out, int type,
                             hipStream_t s) {
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(32 * kRuns), 0, s, part,
                       parts, cols, out, type);
    return hipGetLastError();
}

long long slope_workspace(int rows, int R) {
    const int each = rows_each_of(rows);
    return (long long)((rows + each - 1) / each) * R * 4;
}

hipError_t launch_slope(const SlopeCall& c, hipStream_t s) {
    const int each = rows_each_of(c.rows), parts = (c.rows + each - 1) / each;
    const int R = c.gated ? 2 * c.N : c.N;
    if (parts > 0) {
        const dim3 grid((unsigned)((c.N + kLanes * kVec - 1) / (kLanes * kVec)), (unsigned)parts);
        if (c.gated)
            hipLaunchKernelGGL(slope_kernel<true>, grid, dim3(256), 0, s, c, each);
        else
            hipLaunchKernelGGL(slope_kernel<false>, grid, dim3(256), 0, s, c, each);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return c.db ? launch_column_sum(c.workspace, parts, R, c.db, c.type, s) : hipSuccess;
}

}  // namespace bvml_ffn
