// Sums of a workgroup's parts: what each workgroup of a pass over rows leaves per
// column, added up in a fixed order.
#pragma once

#include "ts_hip_internal.h"

namespace tship {

// out[c] = the parts' sum over g, f64: 16 columns a workgroup, 16 groups of parts
static __global__ __launch_bounds__(kBlock) void sum_parts(const float *__restrict__ part, size_t parts, size_t cols,
                                                    float *__restrict__ out) {
    __shared__ double lds[16][17];
    const int j = threadIdx.x & 15, q = threadIdx.x >> 4;
    const size_t c = static_cast<size_t>(blockIdx.x) * 16 + j;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 8
        for (size_t g = q; g < parts; g += 16) s += part[g * cols + c];
    }
    lds[q][j] = s;
    __syncthreads();
    if (q == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += lds[k][j];
        out[c] = static_cast<float>(s);
    }
}

}  // namespace tship
