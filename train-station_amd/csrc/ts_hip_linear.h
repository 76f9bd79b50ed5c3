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

// act(z) and, where SLOPE, act'(z); relu's zero is -0, which the other two do not give (s + d, s >= 0)
template <bool SLOPE>
__device__ __forceinline__ float activate(float z, int act, float &slope) {
    if (act == TS_HIP_ACT_NONE) {
        slope = 1.0f;
        return z;
    }
    if (act == TS_HIP_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : -0.0f;
        return z > 0.0f ? z : 0.0f;
    }
    const bool silu = act == TS_HIP_ACT_SILU;
    const float v = silu ? z : kGelu1 * (z + kGelu2 * z * z * z);
    const float q = exp_neg_abs(v), inv = 1.0f / (1.0f + q);
    const float s = v >= 0.0f ? inv : v < 0.0f ? q * inv : v;  // 1 / (1 + e^-v); a NaN stays
    if (SLOPE) {
        // s + z s (1 - s) v', s (1 - s) = q / (1 + q)^2: no cancellation at either end; far out the second
        // term is nothing, whatever its factors
        const float d = z * (q * inv * inv) * (silu ? 1.0f : kGelu1 * (1.0f + 3.0f * kGelu2 * z * z));
        slope = q == 0.0f ? s : s + d;
    }
    return z * s;
}

// dz = go act'(z), but nothing where relu holds go back (a slope of -0), whatever go is
__device__ __forceinline__ float through_slope(float go, float slope) {
    return __float_as_uint(slope) == 0x80000000u ? 0.0f : go * slope;
}

// ---- epilogues -------------------------------------------------------------------

// Of a product P [M, N] stored with ldc = N:
//   v = P + bias[j];  slope[i][j] = act'(v) where slope is set
//   go set:  c = go act'(v)                 (a layer's dz)
//   else:    c = act(v) + residual
struct LinearEpi {
    const float *bias, *residual, *go;
    float *slope;
    int act;
};

// c from v = P and the value of go or residual at its place (extra)
__device__ __forceinline__ void epilogue_store(const LinearEpi &e, float *c, size_t at, float v, float bias, float extra) {
    if (e.bias) v += bias;
    float slope;
    if (e.go) {
        activate<true>(v, e.act, slope);
        c[at] = through_slope(extra, slope);
        return;
    }
    if (e.slope) {
        v = activate<true>(v, e.act, slope);
        e.slope[at] = slope;
    } else {
        v = activate<false>(v, e.act, slope);
    }
    if (e.residual) v += extra;
    c[at] = v;
}
__device__ __forceinline__ void epilogue_store(const LinearEpi &e, float *c, size_t at, float v, float bias) {
    const float *extra = e.go ? e.go : e.residual;
    epilogue_store(e, c, at, v, bias, extra ? extra[at] : 0.0f);
}

// ---- operands --------------------------------------------------------------------

// An operand's rows (its index in the product that is not k) and k: floats with
// k or the row contiguous (through what stands at the same place of `times`,
// where set: go and a layer's slopes), or codes [rows][pitch] with k or the row
// along the code rows.
enum class Src { kFloatK, kFloatR, kCodesK, kCodesR };

struct Operand {
    const float *p, *times;
    const uint8_t *codes, *scales;
    int ld;         // floats: the leading dimension
    int rows;       // the product's rows
    size_t pitch;   // codes
    size_t code_rows;
};

template <Src S>
__device__ __forceinline__ float operand_at(const Operand &o, int row, int k) {
    if constexpr (S == Src::kFloatK || S == Src::kFloatR) {
        const size_t at = S == Src::kFloatK ? static_cast<size_t>(row) * o.ld + k : static_cast<size_t>(k) * o.ld + row;
        return o.times ? through_slope(o.p[at], o.times[at]) : o.p[at];
    } else {
        const size_t r = S == Src::kCodesK ? row : k, c = S == Src::kCodesK ? k : row;
        const int s = o.scales[(c / kPackGroup * o.code_rows + r) * 4 + c / kPackBlock % 4];
        return __builtin_amdgcn_cvt_f32_fp8(o.codes[r * o.pitch + c], 0) * pow2f(s - kPackBias);
    }
}

// k .. k + 3 (k a multiple of 4; zeros from K on) of rows row and row + 1 (row
// even; past the last one: its values, or zeros)
template <Src S>
__device__ __forceinline__ void operand_pair(const Operand &o, int row, int k, int K, float (&v)[2][4]) {
    typedef float pk2u_t __attribute__((ext_vector_type(2), aligned(4)));
    if constexpr (S == Src::kFloatK) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = min(row + x, o.rows - 1);
            const size_t at = static_cast<size_t>(r) * o.ld + k;
            if (k + 4 <= K) {
                const pk4u_t q = *reinterpret_cast<const pk4u_t *>(o.p + at);
#pragma unroll
                for (int c = 0; c < 4; ++c) v[x][c] = q[c];
                if (o.times) {  // uniform
                    const pk4u_t t = *reinterpret_cast<const pk4u_t *>(o.times + at);
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[x][c] = through_slope(q[c], t[c]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) v[x][c] = k + c < K ? operand_at<S>(o, r, k + c) : 0.0f;
            }
        }
    } else if constexpr (S == Src::kFloatR) {
        const bool two = row + 1 < o.rows;
        const int r = min(row, o.rows - 1);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            pk2u_t q = {0.0f, 0.0f};
            if (k + c < K) {
                const size_t at = static_cast<size_t>(k + c) * o.ld + r;
                if (two) {
                    q = *reinterpret_cast<const pk2u_t *>(o.p + at);
                    if (o.times) {
                        const pk2u_t t = *reinterpret_cast<const pk2u_t *>(o.times + at);
                        q = pk2u_t{through_slope(q[0], t[0]), through_slope(q[1], t[1])};
                    }
                } else {
                    q[0] = operand_at<S>(o, r, k + c);
                }
            }
            v[0][c] = q[0];
            v[1][c] = q[1];
        }
    } else if constexpr (S == Src::kCodesK) {  // (the padding's codes are zeros)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const size_t r = min(row + x, o.rows - 1);
            unsigned code = 0;
            uint8_t scale = 0;
            if (k < K) {
                code = *reinterpret_cast<const unsigned *>(o.codes + r * o.pitch + k);
                scale = o.scales[(static_cast<size_t>(k / kPackGroup) * o.code_rows + r) * 4 + k / kPackBlock % 4];
            }
            unpack4(code, scale, v[x]);
        }
    } else {  // two codes of a code row and its scale (a row's pitch holds the whole tile)
        const size_t col = row, group = (col / kPackGroup * o.code_rows) * 4 + col / kPackBlock % 4;
        unsigned code[4];
        int scale[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const size_t r = min(k + c, K - 1);
            code[c] = *reinterpret_cast<const uint16_t *>(o.codes + r * o.pitch + col);
            scale[c] = o.scales[group + 4 * r];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            const f2 q = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code[c]), false);
            const float by = k + c < K ? pow2f(scale[c] - kPackBias) : 0.0f;
            v[0][c] = k + c < K ? q[0] * by : 0.0f;
            v[1][c] = k + c < K ? q[1] * by : 0.0f;
        }
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
    bool streams = false;  // B is read as it lies (streams_take)
};

// ---- the large products (ts_hip_linear_planes.hip) ---------------------------------

bool planes_take(size_t M, size_t N, size_t K);
// whether floats B of rows of ld go to the product as they lie, if they begin at 16 bytes
bool streams_take(size_t M, size_t N, size_t K, size_t ld);
size_t streams_workspace_floats(size_t M, size_t N, size_t K, Src a);
// a product's planes (none where both operands are codes along k) and slices
size_t planes_workspace_floats(size_t M, size_t N, size_t K, Src a, Src b);
size_t planes_sum_floats(size_t N, size_t K);

// One operand's way into planes, at planes_of_a / _b of its product's workspace,
// and what the pass over it does beside.
struct PlaneTask {
    const LinearProduct *p;
    bool b;  // B, else A
    char *out;
    uint8_t *codes, *scales;  // A of floats along k: its values in 8 bits as well
    float *sum_parts;         // B of floats along its rows: parts of their sums over k
};
constexpr int kMaxPlaneTasks = 4;
char *planes_of_a(const LinearProduct &p, float *workspace);
char *planes_of_b(const LinearProduct &p, float *workspace);
void planes_write(const PlaneTask *tasks, int count, hipStream_t s);
// the product from its planes; sums: B's rows' sums from their parts
void planes_multiply(const LinearProduct &p, float *workspace, const float *sum_parts, float *sums, hipStream_t s);

}  // namespace tship
