// colsum.cuh -- the last step of a weight's gradient: per-block partial column sums
// (float32) added in block order, so that the result depends on nothing but the inputs.
#pragma once

#include <stdint.h>

#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int CR_COLS = 16, CR_ROWS = 32;

// out[n] = sum_b part[b][n], n < N: CR_ROWS threads per column take every CR_ROWS-th block,
// their sums are added in order.  Columns from `split` on go to out2 (two weights' partial
// sums side by side).
template <typename T>
__global__ void __launch_bounds__(CR_COLS* CR_ROWS) k_col_reduce(const float* __restrict__ part, int blocks, int64_t N,
                                                                 int64_t split, T* __restrict__ out,
                                                                 T* __restrict__ out2) {
    __shared__ float sums[CR_ROWS][CR_COLS + 1];
    grid_wait();
    grid_trigger();
    const int x = threadIdx.x % CR_COLS, y = threadIdx.x / CR_COLS;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * CR_COLS + x;
    float s = 0.0f;
    if (n < N) {
#pragma unroll 8
        for (int b = y; b < blocks; b += CR_ROWS) s += part[static_cast<int64_t>(b) * N + n];
    }
    sums[y][x] = s;
    __syncthreads();
    if (y == 0 && n < N) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < CR_ROWS; ++i) t += sums[i][x];
        if (n < split) out[n] = round_to<T>(t);
        else out2[n - split] = round_to<T>(t);
    }
}

}  // namespace ravel
