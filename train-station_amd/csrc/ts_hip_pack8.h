// Values in 8 bits: e4m3 codes with one power-of-two scale per 32 columns of a
// row (the layout and its rules: ts_hip.h, ts_hip_pack8).
//
// A block's scale exponent k is the smallest that keeps its largest magnitude
// within 448 = 1.75 2^8, read from that value's bits; a value's code is the
// rounding of v 2^-k, exact in fp32 but for results far below the smallest
// code's half.
#pragma once

#include "ts_hip_internal.h"

namespace tship {

constexpr int kPackBlock = 32;   // columns of a scale
constexpr int kPackGroup = 128;  // columns whose scales stand together
constexpr int kPackMinExp = -117, kPackMaxExp = 119, kPackBias = 127;

// four floats at any 4-byte address (gfx950 loads them with one instruction)
typedef float pk4u_t __attribute__((ext_vector_type(4), aligned(4)));

__host__ __device__ inline size_t packed_pitch(size_t cols) { return (cols + kPackGroup - 1) / kPackGroup * kPackGroup; }

// the smallest k in the range with amax <= 448 2^k: past a mantissa of 1.75 the
// sum carries into the exponent
__device__ __forceinline__ int pack_exponent(float amax) {
    const int k = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return min(max(k, kPackMinExp), kPackMaxExp);
}

__device__ __forceinline__ float pow2f(int k) { return __uint_as_float(static_cast<unsigned>(k + 127) << 23); }

// d in fp32, the last bit set where it is not exact: comparisons with, and
// roundings at, every border of fewer bits come out as d's own
__device__ __forceinline__ float round_odd(double d) {
    const float f = static_cast<float>(d);
    const double back = f;
    if (back == d || !(back == back) || __builtin_isinf(back)) return f;
    const unsigned u = __float_as_uint(f);
    if (u & 1u) return f;
    // f is even and off: its odd neighbour on d's side (f = 0: the smallest of d's sign)
    if (f == 0.0f) return d < 0 ? __uint_as_float(0x80000001u) : __uint_as_float(1u);
    return __uint_as_float(fabs(d) > fabs(back) ? u + 1u : u - 1u);
}

// four values times inv (2^-k) as four codes, the first in the low byte
__device__ __forceinline__ unsigned pack4(const float (&v)[4], float inv) {
    float q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float s = v[c] * inv;
        q[c] = fabsf(s) > 448.0f ? copysignf(448.0f, s) : s;  // (a NaN stays)
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true);
    return static_cast<unsigned>(r);
}

// the values that four codes and their block's scale byte stand for
__device__ __forceinline__ void unpack4(unsigned code, uint8_t scale, float (&v)[4]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const float k = pow2f(static_cast<int>(scale) - kPackBias);
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), false);
    const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), true);
    v[0] = lo[0] * k;
    v[1] = lo[1] * k;
    v[2] = hi[0] * k;
    v[3] = hi[1] * k;
}

typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));

// eight codes (two words) and their scale as bf16
__device__ __forceinline__ bf8_t widen(unsigned lo, unsigned hi, float scale) {
    union {
        bf8_t v;
        bf2_t p[4];
    } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return u.v;
}

// Packs four columns c .. c + 3 of a row (past cols: zeros in v); the eight
// lanes of a block of 32 call together.  scales points at the row's entry of
// group 0, groups scale_step bytes apart.
__device__ __forceinline__ void pack_store(const float (&v)[4], size_t c, uint8_t *codes, uint8_t *scales,
                                           size_t scale_step) {
    float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const int k = pack_exponent(m);
    *reinterpret_cast<unsigned *>(codes + c) = pack4(v, pow2f(-k));
    if ((threadIdx.x & 7) == 0)
        scales[c / kPackGroup * scale_step + c / kPackBlock % 4] = static_cast<uint8_t>(k + kPackBias);
}

}  // namespace tship
