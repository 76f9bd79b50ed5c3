// Sums of a workgroup's parts: what each workgroup of a pass over rows leaves per
// column, added up in a fixed order.
#pragma once

#include "ts_hip_internal.h"

namespace tship {

// out[c] = the sum over g of part[g][c], in f64; blocks workgroups of at
// least kBlock threads, 16 columns each, 16 groups of parts side by side.
struct PartSums {
    const float *part;
    size_t parts, cols;
    float *out;
    int blocks;
};
inline PartSums part_sums(const float *part, size_t parts, size_t cols, float *out) {
    return {part, parts, cols, out, static_cast<int>((cols + 15) / 16)};
}

constexpr int kPartSumsLds = 16 * 17;  // doubles

__device__ __forceinline__ void part_sums_block(const PartSums &p, int block, double *lds) {
    const int j = threadIdx.x & 15, q = threadIdx.x >> 4;
    const size_t c = static_cast<size_t>(block) * 16 + j;
    double s = 0.0;
    if (c < p.cols && q < 16) {  // (threads past kBlock only reach the barrier)
#pragma unroll 8
        for (size_t g = q; g < p.parts; g += 16) s += p.part[g * p.cols + c];
    }
    if (q < 16) lds[q * 17 + j] = s;
    __syncthreads();
    if (q == 0 && c < p.cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += lds[k * 17 + j];
        p.out[c] = static_cast<float>(s);
    }
}

}  // namespace tship
