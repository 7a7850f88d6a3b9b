// Sums of columns over partial rows: what the gradients of a bias and of a
// norm's weight end with.  Private to libbvml_ffn.so.
#pragma once

#include "ffn_kernels.h"

namespace bvml_ffn {

// 32 columns a workgroup of 32 kRuns threads: kRuns interleaved runs of the
// parts, each in its order, then the runs.  Bound by latency: a thread has
// eight of its loads in flight (1,024 rows of 1,024 columns: 4.7 us; 39 with
// one at a time; sixteen gain nothing), the last ones too.
template <int kRuns>
__device__ __forceinline__ void column_sum(const ColumnSum& c, int block, float (*sums)[32]) {
    constexpr int kInFlight = 8;
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    const int col = block * 32 + x;
    float t = 0.0f;
    if (col < c.cols) {
        const float* p = c.part + col;
        for (int r = y; r < c.parts; r += kInFlight * kRuns) {
            float v[kInFlight];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) {
                const int at = r + i * kRuns;  // beyond the last: that one again, not added
                v[i] = p[(long long)(at < c.parts ? at : c.parts - 1) * c.cols];
            }
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) t += r + i * kRuns < c.parts ? v[i] : 0.0f;
        }
    }
    sums[y][x] = t;
    __syncthreads();
    if (y != 0 || col >= c.cols) return;
#pragma unroll
    for (int j = 1; j < kRuns; ++j) t += sums[j][x];
    if (c.type == kF32)
        static_cast<float*>(c.out)[col] = t;
    else
        static_cast<uint16_t*>(c.out)[col] = to16(t, c.type);
}

}  // namespace bvml_ffn
