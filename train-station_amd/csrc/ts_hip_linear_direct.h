// A layer's small products.
//
// A wave computes 32 x 32 of C in blocks of v_mfma_f32_16x16x4_f32, its operands
// straight from memory to registers: a lane takes four k of two neighbouring rows
// (k 4 q + s of 16 in step s, the same for both operands; row 2 i + x in block x),
// so what lies along k comes in 16-byte loads and what lies along the rows in
// 8-byte ones.  Nothing is staged: such a call is a launch and a few waits for
// memory, and a stage's barrier would be one more.
//
// Few tiles have a long way each: kg waves of a workgroup take parts of a tile's
// K, joined through LDS in their order, and past 2048 k several workgroups
// (slices), whose sums a second launch adds in their order.  Layer 300 -> 200,
// batch 8192: its weight's gradient, 70 tiles of 8192 k, 1050 us by a wave each.
#pragma once

#include <type_traits>

#include "ts_hip_linear.h"

namespace tship {

constexpr int kDirectTile = 32;
constexpr int kDirectK = 16;
constexpr int kDirectWaves = 8;  // of a workgroup, at most: the largest kg of its launch
constexpr int kDirectThreads = 64 * kDirectWaves;
constexpr unsigned kDirectLds = kDirectTile * kDirectTile * sizeof(float);  // a wave's, in bytes

// A small product and its share of a launch: blocks workgroups, of waves / kg
// units (a tile's slice) each.
struct DirectProduct {
    Operand A, B;
    float *C;
    LinearEpi epi;
    int M, N, K, tiles_n, tiles;
    int kg, slices, slice_steps, blocks;
    float *part;  // several slices: [slices][M][N]
};

inline DirectProduct direct_product(const LinearProduct &p) {
    const int tm = (p.M + kDirectTile - 1) / kDirectTile, tn = (p.N + kDirectTile - 1) / kDirectTile;
    const int steps = (p.K + kDirectK - 1) / kDirectK;
    return {p.A, p.B, p.C, p.epi, p.M, p.N, p.K, tn, tm * tn, 1, 1, steps, 0, nullptr};
}

// Steps from .. to of a tile, added to acc.  U steps' loads are issued at a time;
// AHEAD: a round's before the products of the one before.
template <Src SA, Src SB, int U, bool AHEAD>
__device__ __forceinline__ void direct_steps(const DirectProduct &p, int i0, int j0, int from, int to, int lane,
                                             f4v_t (&acc)[2][2]) {
    const int li = lane & 15, lq = lane >> 4;
    constexpr int R = AHEAD ? 2 : 1;
    float a[R][U][2][4], b[R][U][2][4];
    auto load = [&](int r, int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= to) break;  // uniform
            const int k = (s0 + u) * kDirectK + 4 * lq;
            operand_pair<SA>(p.A, i0 + 2 * li, k, p.K, a[r][u]);
            operand_pair<SB>(p.B, j0 + 2 * li, k, p.K, b[r][u]);
        }
    };
    auto multiply = [&](int r, int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= to) break;  // uniform
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        acc[x][c] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(a[r][u][x][s], b[r][u][c][s], acc[x][c], 0, 0, 0);
        }
    };
    if constexpr (AHEAD) {
        load(0, from);
        for (int s0 = from; s0 < to; s0 += 2 * U) {
            load(1, s0 + U);
            multiply(0, s0);
            load(0, s0 + 2 * U);
            multiply(1, s0 + U);
        }
    } else {
        for (int s0 = from; s0 < to; s0 += U) {
            load(0, s0);
            multiply(0, s0);
        }
    }
}
// lane (li, lq), register r of block (x, c): row 2 (4 lq + r) + x, column 2 li + c
template <class F>
__device__ __forceinline__ void direct_each(const f4v_t (&acc)[2][2], int lane, F &&f) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) f(2 * (4 * (lane >> 4) + r) + x, 2 * (lane & 15), acc[x][0][r], acc[x][1][r]);
}

// Steps from .. to of a tile by one wave, with the epilogue (in few registers:
// what the large products fall back to).
template <Src SA, Src SB>
__device__ __forceinline__ void direct_tile(const DirectProduct &p, int tile, int from, int to, int lane) {
    const int i0 = tile / p.tiles_n * kDirectTile, j0 = tile % p.tiles_n * kDirectTile;
    f4v_t acc[2][2] = {};
    direct_steps<SA, SB, 1, false>(p, i0, j0, from, to, lane, acc);
    direct_each(acc, lane, [&](int row, int col, float v0, float v1) {
        const int i = i0 + row, j = j0 + col;
        if (i >= p.M) return;
        const size_t at = static_cast<size_t>(i) * p.N + j;
        if (j < p.N) epilogue_store(p.epi, p.C, at, v0, p.epi.bias ? p.epi.bias[j] : 0.0f);
        if (j + 1 < p.N) epilogue_store(p.epi, p.C, at + 1, v1, p.epi.bias ? p.epi.bias[j + 1] : 0.0f);
    });
}

// Workgroup `block` of a product, of `waves` waves; lds: a tile per wave.
template <Src SA, Src SB>
__device__ __forceinline__ void direct_block(const DirectProduct &p, int block, int waves, float (*lds)[kDirectTile * kDirectTile]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = p.kg, group = wave % kg, unit = block * (waves / kg) + wave / kg;
    const bool live = unit < p.tiles * p.slices;  // uniform per wave; the others reach the barrier
    const int tile = unit / p.slices, slice = unit % p.slices;
    const int i0 = tile / p.tiles_n * kDirectTile, j0 = tile % p.tiles_n * kDirectTile;
    if (live) {
        const int steps = (p.K + kDirectK - 1) / kDirectK;
        const int first = slice * p.slice_steps, last = min(first + p.slice_steps, steps);
        const int per = (last - first + kg - 1) / kg, from = first + group * per;
        f4v_t acc[2][2] = {};
        direct_steps<SA, SB, 2, true>(p, i0, j0, from, min(from + per, last), lane, acc);
        direct_each(acc, lane, [&](int row, int col, float v0, float v1) {
            float *to = &lds[wave][row * kDirectTile + col];
            to[0] = v0;
            to[1] = v1;
        });
    }
    __syncthreads();
    if (!live) return;
    // the unit's waves add and store four columns a lane
    float *part = p.part + static_cast<size_t>(slice) * p.M * p.N;
    for (int n = group * 64 + lane; n < kDirectTile * kDirectTile / 4; n += 64 * kg) {
        const int i = i0 + n / (kDirectTile / 4), j = j0 + n % (kDirectTile / 4) * 4;
        f4v_t v = *reinterpret_cast<const f4v_t *>(&lds[wave - group][4 * n]);
        for (int g = 1; g < kg; ++g) v += *reinterpret_cast<const f4v_t *>(&lds[wave - group + g][4 * n]);
        if (i >= p.M) continue;
        const size_t at = static_cast<size_t>(i) * p.N + j;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e >= p.N) continue;
            if (p.slices > 1) part[at + e] = v[e];
            else epilogue_store(p.epi, p.C, at + e, v[e], p.epi.bias ? p.epi.bias[j + e] : 0.0f);
        }
    }
}

// A product's slices added in their order, with its epilogue (ts_hip_linear.hip).
void join_slices(const DirectProduct &p, hipStream_t s);

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
