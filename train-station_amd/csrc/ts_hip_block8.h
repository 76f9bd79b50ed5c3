// Values in 8 bits with a 32-bit scale for each block of 128 columns, of one row or
// of 128 rows (the layout and its rules: ts_hip.h, ts_hip_block8).
//
// A block's scale is its largest magnitude over 448, a code the rounding of its value
// times 1 / scale: two fp32 roundings before the one to four bits, so a value is off by
// at most 2^-4 + 2^-22 of itself.
#pragma once

#include "ts_hip_pack8.h"

namespace tship {

constexpr float kBlock8Least = 0x1p-100f, kBlock8Most = 448.0f * 0x1p119f;  // a block's largest, as its scale holds it

struct Block8Scale {
    float scale, inv;
};
__device__ __forceinline__ Block8Scale block8_scale(float largest) {
    const float scale = fminf(fmaxf(largest, kBlock8Least), kBlock8Most) / 448.0f;
    return {scale, 1.0f / scale};
}

// max of the 32 lanes of a half wave, in each of them
__device__ __forceinline__ float half_wave_max(float m) {
#define TS_DPP_MAX(ctrl) \
    m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), ctrl, 0xf, 0xf, true)))
    TS_DPP_MAX(0xB1);   // lanes 1 0 3 2
    TS_DPP_MAX(0x4E);   // lanes 2 3 0 1
    TS_DPP_MAX(0x141);  // eight lanes mirrored
    TS_DPP_MAX(0x140);  // sixteen lanes mirrored
#undef TS_DPP_MAX
    return fmaxf(m, __shfl_xor(m, 16, 64));
}

__device__ __forceinline__ float largest4(const float (&v)[4]) {  // (NaN is left out)
    return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
}

// Packs four columns c .. c + 3 of a row (past its end: zeros in v); the 32 lanes of a
// block call together.  codes: the row's; scales: the row's of block 0, scale_step apart.
__device__ __forceinline__ void block8_store(const float (&v)[4], size_t c, uint8_t *codes, float *scales, size_t scale_step) {
    const Block8Scale s = block8_scale(half_wave_max(largest4(v)));
    *reinterpret_cast<unsigned *>(codes + c) = pack4(v, s.inv);
    if ((threadIdx.x & 31) == 0) scales[c / kPackGroup * scale_step] = s.scale;
}

}  // namespace tship
