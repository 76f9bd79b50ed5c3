// What a layer's kernels share (ts_hip_linear.hip: the entries and the small
// products; ts_hip_linear_planes.hip: the large ones): activations, the
// epilogues and the operands as their elements are read one by one.
#pragma once

#include "ts_hip_pack8.h"

namespace tship {

// ---- activations -----------------------------------------------------------------

// e^-|v|: 2^(i + f) with -|v| log2(e) = i + f, the product's rounding error in f
// (from 104 on the result is 0)
__device__ __forceinline__ float exp_neg_abs(float v) {
    const float a = fmaxf(-fabsf(v), -150.0f), t = a * 1.44269502f;  // log2(e) in two pieces
    const float i = __builtin_rintf(t);
    const float f = __builtin_fmaf(a, 1.92596303e-8f, __builtin_fmaf(a, 1.44269502f, -i));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(i));
}

constexpr float kGelu1 = 1.59576912f;  // 2 sqrt(2 / pi)
constexpr float kGelu2 = 0.044715f;

// s(v) = 1 / (1 + e^-v) from q = e^-|v|, and s (1 - s): no cancellation at either end
__device__ __forceinline__ float sigmoid_of(float v, float q) {
    const float inv = 1.0f / (1.0f + q);
    return v >= 0.0f ? inv : v < 0.0f ? q * inv : v;  // (a NaN stays)
}

__device__ __forceinline__ float activate(float z, int act) {
    if (act == TS_HIP_ACT_NONE) return z;
    if (act == TS_HIP_ACT_RELU) return z > 0.0f ? z : 0.0f;
    const float v = act == TS_HIP_ACT_SILU ? z : kGelu1 * (z + kGelu2 * z * z * z);
    return z * sigmoid_of(v, exp_neg_abs(v));
}

__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == TS_HIP_ACT_NONE) return 1.0f;
    if (act == TS_HIP_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    const bool silu = act == TS_HIP_ACT_SILU;
    const float v = silu ? z : kGelu1 * (z + kGelu2 * z * z * z);
    const float q = exp_neg_abs(v), s = sigmoid_of(v, q), inv = 1.0f / (1.0f + q);
    if (q == 0.0f) return s;  // far out the second term is nothing, whatever its factors
    return s + z * (q * inv * inv) * (silu ? 1.0f : kGelu1 * (1.0f + 3.0f * kGelu2 * z * z));
}

// ---- epilogues -------------------------------------------------------------------

// Of a product P [M, N] stored with ldc = N:
//   v = P + bias[j];  z[i][j] = v where z is set
//   go set:  c = go v's slope               (a layer's dz)
//   else:    c = act(v) + residual
struct LinearEpi {
    const float *bias, *residual, *go;
    float *z;
    int act;
};

__device__ __forceinline__ void epilogue_store(const LinearEpi &e, float *c, size_t at, float v, float bias) {
    if (e.bias) v += bias;
    if (e.z) e.z[at] = v;
    if (e.go) {
        v = e.go[at] * act_slope(v, e.act);
    } else {
        v = activate(v, e.act);
        if (e.residual) v += e.residual[at];
    }
    c[at] = v;
}

// ---- operands --------------------------------------------------------------------

// An operand's rows (its index in the product that is not k) and k: floats with
// k or the row contiguous, or codes [rows][pitch] with k or the row along the
// code rows.
enum class Src { kFloatK, kFloatR, kCodesK, kCodesR };

struct Operand {
    const float *p;
    const uint8_t *codes, *scales;
    int ld;         // floats: the leading dimension
    int rows;       // the product's rows
    size_t pitch;   // codes
    size_t code_rows;
};

template <Src S>
__device__ __forceinline__ float operand_at(const Operand &o, int row, int k) {
    if constexpr (S == Src::kFloatK) return o.p[static_cast<size_t>(row) * o.ld + k];
    else if constexpr (S == Src::kFloatR) return o.p[static_cast<size_t>(k) * o.ld + row];
    else {
        const size_t r = S == Src::kCodesK ? row : k, c = S == Src::kCodesK ? k : row;
        const int s = o.scales[(c / kPackGroup * o.code_rows + r) * 4 + c / kPackBlock % 4];
        return __builtin_amdgcn_cvt_f32_fp8(o.codes[r * o.pitch + c], 0) * pow2f(s - kPackBias);
    }
}

// k .. k + 3 of a row (k a multiple of 4), zeros from K on
template <Src S>
__device__ __forceinline__ void operand4(const Operand &o, int row, int k, int K, float (&v)[4]) {
    if constexpr (S == Src::kFloatK) {
        const float *p = o.p + static_cast<size_t>(row) * o.ld;
        if (k + 4 <= K) {
            const pk4u_t q = *reinterpret_cast<const pk4u_t *>(p + k);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = q[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = k + c < K ? p[k + c] : 0.0f;
        }
    } else if constexpr (S == Src::kCodesK) {  // (the padding's codes are zeros)
        if (k < K) {
            const int s = o.scales[(static_cast<size_t>(k / kPackGroup) * o.code_rows + row) * 4 + k / kPackBlock % 4];
            unpack4(*reinterpret_cast<const unsigned *>(o.codes + row * o.pitch + k), static_cast<uint8_t>(s), v);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = 0.0f;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = k + c < K ? operand_at<S>(o, row, k + c) : 0.0f;
    }
}

// ---- products ------------------------------------------------------------------------

// C [M, N] = A B with an epilogue; a: Src of A, b: of B.
struct LinearProduct {
    Operand A, B;
    Src a, b;
    int M, N, K;
    float *C;
    LinearEpi epi;
};

// ---- the large products (ts_hip_linear_planes.hip) ---------------------------------

// What the pass over an operand does beside its planes.
struct PlanesExtra {
    // A along k: its values in 8 bits as well
    uint8_t *codes = nullptr, *scales = nullptr;
    // B along its rows: its rows' sums over k into `sums`, by planes_sum_floats(N, K) of `sum_parts`
    float *sums = nullptr, *sum_parts = nullptr;
};

bool planes_take(size_t M, size_t N, size_t K);
size_t planes_workspace_floats(size_t M, size_t N, size_t K, Src a, Src b);
size_t planes_sum_floats(size_t N, size_t K);
int planes_product(const LinearProduct &p, const PlanesExtra &extra, float *workspace, hipStream_t s);

}  // namespace tship
