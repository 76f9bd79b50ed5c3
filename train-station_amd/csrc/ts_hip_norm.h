// What the norms over rows share (ts_hip_norm.hip, ts_hip_layer_norm.hip): a row
// held in registers by W waves, four neighbouring columns a lane and NV such quads.
#pragma once

#include <type_traits>

#include "ts_hip_pack8.h"
#include "ts_hip_parts.h"

namespace tship {

constexpr size_t kMaxHeldCols = 16384;  // 16 waves of 64 lanes of four quads

__device__ __forceinline__ void load4(const float *p, size_t c, size_t cols, float (&v)[4]) {
    if (c + 4 <= cols) {
        const pk4u_t q = *reinterpret_cast<const pk4u_t *>(p + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? p[c + e] : 0.0f;
    }
}

__device__ __forceinline__ void store4(float *p, size_t c, size_t cols, const float (&v)[4]) {
    if (c + 4 <= cols) {
        *reinterpret_cast<pk4u_t *>(p + c) = pk4u_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) p[c + e] = v[e];
    }
}

// The sum over the W waves of a row, in every lane; lds: N * W doubles of this row.
template <int W, int N>
__device__ __forceinline__ void row_sum(double (&s)[N], double *lds) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = wave_sum(s[n]);
    if (W == 1) return;
    const int wave = (threadIdx.x >> 6) % W;
    __syncthreads();  // the last row's reads
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) lds[n * W + wave] = s[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        s[n] = 0.0;
#pragma unroll
        for (int w = 0; w < W; ++w) s[n] += lds[n * W + w];
    }
}

// r = up * f with up a power of two (as fp32 has them) and f in [1, 2) where r is
// one of fp32's range, within a few binades of it for what rows can give beyond.
struct RowScale {
    float up;
    double f;
};
__device__ __forceinline__ RowScale row_scale(double r) {
    const int e = min(max(static_cast<int>(__double_as_longlong(r) >> 52 & 0x7ff) - 1023, -126), 127);  // (inf, NaN: 127)
    const double down = __longlong_as_double(static_cast<long long>(1023 - e) << 52);
    return {__uint_as_float(static_cast<unsigned>(e + 127) << 23), r * down};
}

template <int W>
constexpr int kNormThreads = W < 4 ? 256 : 64 * W;
template <int W>
constexpr int kNormRows = kNormThreads<W> / (64 * W);  // rows of a workgroup

constexpr size_t kLongCols = 4 * kBlock;  // of a workgroup that passes over long rows by columns

constexpr size_t kMaxBlocks = size_t(1) << 21;  // a launch has fewer than 2^32 threads; more rows take turns

// Calls f(W, NV, LONG as constants) for a row of n columns: the fewest waves that
// hold it with four quads a lane, but for rows of 4097 to 8192 packed, whose f64
// products want the registers: two quads.  us, packed with the sum, four quads and
// two: 8192 x 4096 87, 92; 4096 x 8192 120, 107.  Forward and backward: 4096 x 8192
// 184, 187; 4096 x 6000 144, 157.  (Eight quads: 2048 x 16384 packed 129, four 109.)
// MAY_PACK: whether the caller's kernels pack at all.
template <bool MAY_PACK, class F>
void for_cols(size_t n, bool packed, F &&f) {
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    const integral_constant<int, 8> eight{};
    const integral_constant<int, 16> sixteen{};
    const integral_constant<bool, false> held{};
    if (n <= 256) f(one, one, held);
    else if (n <= 512) f(one, two, held);
    else if (n <= 1024) f(one, four, held);
    else if (n <= 2048) f(four, two, held);
    else if (n <= 4096) f(four, four, held);
    else if (n <= 8192) {
        if constexpr (MAY_PACK) {
            if (packed) return f(sixteen, two, held);
        }
        f(eight, four, held);
    }
    else if (n <= kMaxHeldCols) f(sixteen, four, held);
    else f(sixteen, four, integral_constant<bool, true>{});
}

inline size_t rows_per_block(size_t cols) { return cols <= 1024 ? 4 : 1; }

// Workgroups of the backward pass: as many as run at once (2048 threads a CU, at
// most 4 workgroups), so that each sums many rows before it writes dw.
inline size_t back_blocks(size_t rows, size_t cols) {
    const size_t need = (rows + rows_per_block(cols) - 1) / rows_per_block(cols);
    const size_t cap = static_cast<size_t>(device_cu_count()) * (cols > 4096 ? 1 : 2);
    return need < cap ? need : cap;
}

// Rows of a part of long_columns: as many as leave eight workgroups a CU, in no more parts than back_blocks
inline size_t long_run(size_t rows, size_t cols) {
    const size_t wide = (cols + kLongCols - 1) / kLongCols, most = back_blocks(rows, cols);
    const size_t want = (static_cast<size_t>(device_cu_count()) * 8 + wide - 1) / wide;
    const size_t parts = want < most ? want : most;
    return (rows + parts - 1) / parts;
}

constexpr size_t kMaxRows = size_t(1) << 31;
// Parts that one workgroup adds up sooner than another launch has started: 128 x 784
// (32 parts) forward and backward 26.8 us by two launches, 24.5 by one; 16384 x 64
// (512 parts) 27.1 by two, 69 by one.
constexpr size_t kTicketParts = 64, kTicketFloats = 32768;

}  // namespace tship
