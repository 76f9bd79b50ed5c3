// A layer's small products.
//
// A wave computes 32 x 32 of C in blocks of
// v_mfma_f32_16x16x4_f32, its operands straight from memory to registers: a
// lane takes four k of a row (k 4 q + s of 16 in step s, the same for both
// operands), so what lies along k comes in 16-byte loads.  Nothing is staged:
// such a call is a launch and a few waits for memory, and a stage's barrier
// would be one more.  The waves of a workgroup take equal parts of K and their
// sums are added in order through LDS: few tiles have a long way each.
#pragma once

#include <type_traits>

#include "ts_hip_linear.h"

namespace tship {

constexpr int kDirectTile = 32;
constexpr int kDirectK = 16;

// A small product and the layout of its grid.
struct DirectProduct {
    Operand A, B;
    float *C;
    LinearEpi epi;
    int M, N, K, tiles_n, tiles;
};

// KG waves share the tile (1: any wave by itself).
template <Src SA, Src SB, int KG>
__device__ __forceinline__ void direct_tile(const DirectProduct &p, int tile, float *lds) {
    const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
    const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int i0 = tile / p.tiles_n * kDirectTile, j0 = tile % p.tiles_n * kDirectTile;
    f4v_t acc[2][2] = {};
    int ra[2], rb[2];  // rows past an edge read the last one and are not stored
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        ra[x] = min(i0 + 16 * x + li, p.M - 1);
        rb[x] = min(j0 + 16 * x + li, p.N - 1);
    }
    const int steps = (p.K + kDirectK - 1) / kDirectK, per = (steps + KG - 1) / KG;
    const int from = group * per, to = min(from + per, steps);
    constexpr int U = 4;  // steps whose loads are issued before the first is used
    for (int s0 = from; s0 < to; s0 += U) {
        float a[U][2][4], b[U][2][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s0 + u) * kDirectK + 4 * lq, K = s0 + u < to ? p.K : 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                operand4<SA>(p.A, ra[x], k, K, a[u][x]);
                operand4<SB>(p.B, rb[x], k, K, b[u][x]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        acc[x][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][x][s], b[u][c][s], acc[x][c], 0, 0, 0);
    }
    // lane (li, lq), register r of block (x, c): row 16 x + 4 lq + r, column 16 c + li
    if constexpr (KG == 1) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int j = j0 + 16 * c + li;
            if (j >= p.N) continue;
            const float bias = p.epi.bias ? p.epi.bias[j] : 0.0f;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = i0 + 16 * x + 4 * lq + r;
                    if (i < p.M) epilogue_store(p.epi, p.C, static_cast<size_t>(i) * p.N + j, acc[x][c][r], bias);
                }
        }
    } else {
        // the groups' sums by LDS, [group][row][column]; the workgroup then adds
        // and stores whole rows
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    lds[(group * kDirectTile + 16 * x + 4 * lq + r) * kDirectTile + 16 * c + li] = acc[x][c][r];
        __syncthreads();
        for (int n = threadIdx.x; n < kDirectTile * kDirectTile; n += 64 * KG) {
            const int i = i0 + n / kDirectTile, j = j0 + n % kDirectTile;
            float v = lds[n];
#pragma unroll
            for (int g = 1; g < KG; ++g) v += lds[g * kDirectTile * kDirectTile + n];
            if (i < p.M && j < p.N)
                epilogue_store(p.epi, p.C, static_cast<size_t>(i) * p.N + j, v, p.epi.bias ? p.epi.bias[j] : 0.0f);
        }
    }
}

inline DirectProduct direct_product(const LinearProduct &p) {
    const int tm = (p.M + kDirectTile - 1) / kDirectTile, tn = (p.N + kDirectTile - 1) / kDirectTile;
    return {p.A, p.B, p.C, p.epi, p.M, p.N, p.K, tn, tm * tn};
}

// Calls f with a product's operand kinds as constants: the layouts that a layer's products have.
template <class F>
void with_sources(Src a, Src b, F &&f) {
    using K = std::integral_constant<Src, Src::kFloatK>;
    using R = std::integral_constant<Src, Src::kFloatR>;
    if (a == Src::kFloatK && b == Src::kFloatR) f(K{}, R{});       // x W
    else if (a == Src::kFloatK) f(K{}, K{});                       // dz W^T
    else if (a == Src::kFloatR) f(R{}, R{});                       // x^T dz
    else if (a == Src::kCodesK && b == Src::kCodesK)
        f(std::integral_constant<Src, Src::kCodesK>{}, std::integral_constant<Src, Src::kCodesK>{});
    else if (a == Src::kCodesK) f(std::integral_constant<Src, Src::kCodesK>{}, R{});
    else f(std::integral_constant<Src, Src::kCodesR>{}, R{});
}

}  // namespace tship
