// Values in 8 bits with a 32-bit scale for each block of 128 columns, of one row or
// of 128 rows (the layout and its rules: ts_hip.h, ts_hip_block8).
//
// A block's scale is its largest magnitude over 448, rounded to fp32; a code is the
// rounding of its value times 448 / largest, which is taken in f64: on its own side of
// every border, and off by at most 2^-4 + 2^-24 of itself.
#pragma once

#include "ts_hip_pack8.h"

namespace tship {

constexpr double kBlock8Least = 0x1p-100, kBlock8Most = 448.0 * 0x1p119;  // a block's largest, as its scale holds it

struct Block8Scale {
    float scale;
    double inv;
    bool beyond;  // larger values than the scale holds: those take 448
};
__device__ __forceinline__ Block8Scale block8_scale(double largest) {
    const double m = fmin(fmax(largest, kBlock8Least), kBlock8Most);
    return {static_cast<float>(m * (1.0 / 448.0)), 448.0 / m, largest > kBlock8Most};
}

// max of the 32 lanes of a half wave, in each of them
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
// with the neighbouring row of 16 lanes: one copy ends with the even rows, the other with the odd
__device__ __forceinline__ float other_row_max(float m) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ double other_row_max(double m) {
    const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(m), __double2hiint(m), false, false);
    const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(m), __double2loint(m), false, false);
    return fmax(__hiloint2double(hi[0], lo[0]), __hiloint2double(hi[1], lo[1]));
}
template <class F>
__device__ __forceinline__ F half_wave_max(F m) {
    m = larger(m, dpp<0xB1>(m));   // lanes 1 0 3 2
    m = larger(m, dpp<0x4E>(m));   // lanes 2 3 0 1
    m = larger(m, dpp<0x141>(m));  // eight lanes mirrored
    m = larger(m, dpp<0x140>(m));  // sixteen lanes mirrored
    return other_row_max(m);
}

template <class F>
__device__ __forceinline__ F largest4(const F (&v)[4]) {  // (NaN is left out)
    auto size = [](F x) { return x < 0 ? -x : x; };
    return larger(larger(size(v[0]), size(v[1])), larger(size(v[2]), size(v[3])));
}

// A code of a value's fp32 rounding is the value's own unless that rounding is a border:
// from 2^-6 on, one whose last 20 bits are 0x80000.  Those, one in 2^20, and what is below,
// but not 0, take the way by round_odd.
template <class F>
__device__ __forceinline__ unsigned block8_codes(const F (&v)[4], const Block8Scale &s) {
    constexpr unsigned kNormal = 0x3c800000;  // 2^-6
    float q[4];
    unsigned border = ~0u, least = ~0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        q[e] = static_cast<float>(v[e] * s.inv);
        border = min(border, (__float_as_uint(q[e]) << 12) + 0x80000000u);
        least = min(least, (__float_as_uint(q[e]) << 1) - 1);
    }
    if (border == 0 || least < 2 * kNormal - 1 || s.beyond) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = round_odd(v[e] * s.inv);
        return pack4(q, 1.0f);
    }
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true));
}

// Packs four columns c .. c + 3 of a row (past its end: zeros in v); the 32 lanes of a
// block call together.  codes: the row's; scales: the row's of block 0, scale_step apart.
template <class F>
__device__ __forceinline__ void block8_store(const F (&v)[4], size_t c, uint8_t *codes, float *scales, size_t scale_step) {
    const Block8Scale s = block8_scale(half_wave_max(largest4(v)));
    *reinterpret_cast<unsigned *>(codes + c) = block8_codes(v, s);
    if ((threadIdx.x & 31) == 0) scales[c / kPackGroup * scale_step] = s.scale;
}

}  // namespace tship
