// A layer over values in 8 bits (ts_hip.h, ts_hip_linear_packed).
//
//   y[i][j] = act(sum over k of x[i][k] W[j][k] + bias[j]) + residual[i][j]
//
// The codes are widened to bf16 with their scales applied, which is exact (four
// significant bits, and every exponent of code and scale together is one of
// bf16's), multiplied exactly and summed in fp32 by the bf16 instructions.  The
// 8-bit instructions run twice as fast but do not keep fp32 sums: of each eight
// neighbouring products they drop what is 2^-13 below the largest, and 4096
// normal values come out 1.5e-5 off their root mean square (bf16: 2e-7).
//
// Few rows (packed_direct): the weights' bytes are all there is to do.  A wave
// holds 16 columns of y for 16 rows of x, W's rows as the instruction's A
// operand, so a lane ends with four neighbouring columns of a row; the waves of
// a workgroup take every second, fourth, ... group of 128 k, each lane the 32
// codes of one scale (two 16-byte loads), and are joined through LDS.  One row, us:
// 4096 x 4096 6.1 (17 MB, from the cache), 8192 x 8192 13 (69 MB, 5.2 TB/s); 32 rows,
// 4096 x 4096 12.7 (two blocks of rows and columns a wave).
#include "ts_hip_linear.h"

namespace tship {

namespace {

typedef unsigned u4_t __attribute__((ext_vector_type(4)));

struct PackedProduct {
    const uint8_t *xc, *xs, *wc, *ws;
    const float *bias, *residual;
    float *y;
    int M, N, groups, act;  // groups of 128 k
    int tiles_n;
};

// FN blocks of 16 columns, FM of 16 rows a wave; KG waves share K.
template <int FN, int FM, int KG>
__global__ __launch_bounds__(64 * KG) void packed_direct(PackedProduct p) {
    const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j0 = static_cast<int>(blockIdx.x) % p.tiles_n * 16 * FN, i0 = static_cast<int>(blockIdx.x) / p.tiles_n * 16 * FM;
    const size_t pitch = static_cast<size_t>(p.groups) * kPackGroup;
    f4v_t acc[FN][FM] = {};
    const uint8_t *wp[FN], *xp[FM];
    const unsigned *wsp[FN], *xsp[FM];
#pragma unroll
    for (int a = 0; a < FN; ++a) {  // rows past an edge: the last one's, not stored
        const int j = min(j0 + 16 * a + li, p.N - 1);
        wp[a] = p.wc + j * pitch + 32 * lq;
        wsp[a] = reinterpret_cast<const unsigned *>(p.ws) + j;
    }
#pragma unroll
    for (int b = 0; b < FM; ++b) {
        const int i = min(i0 + 16 * b + li, p.M - 1);
        xp[b] = p.xc + i * pitch + 32 * lq;
        xsp[b] = reinterpret_cast<const unsigned *>(p.xs) + i;
    }
    auto scale = [&](unsigned four) { return pow2f(static_cast<int>(four >> (8 * lq) & 255u) - kPackBias); };
    constexpr int U = FN * FM == 1 ? 4 : 2;  // groups whose loads are issued before the first is used
    for (int g0 = group; g0 < p.groups; g0 += KG * U) {
        u4_t w[U][FN][2], x[U][FM][2];
        unsigned wk[U][FN], xk[U][FM];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int g = min(g0 + u * KG, p.groups - 1);  // (past the last: read again, not used)
            const size_t at = static_cast<size_t>(g) * kPackGroup;
#pragma unroll
            for (int a = 0; a < FN; ++a) {
                const u4_t *q = reinterpret_cast<const u4_t *>(wp[a] + at);
                w[u][a][0] = q[0];
                w[u][a][1] = q[1];
                wk[u][a] = wsp[a][static_cast<size_t>(g) * p.N];
            }
#pragma unroll
            for (int b = 0; b < FM; ++b) {
                const u4_t *q = reinterpret_cast<const u4_t *>(xp[b] + at);
                x[u][b][0] = q[0];
                x[u][b][1] = q[1];
                xk[u][b] = xsp[b][static_cast<size_t>(g) * p.M];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (g0 + u * KG >= p.groups) break;  // uniform
#pragma unroll
            for (int h = 0; h < 4; ++h) {  // eight of the lane's 32 k at a time
                bf8_t fw[FN], fx[FM];
#pragma unroll
                for (int a = 0; a < FN; ++a)
                    fw[a] = widen(w[u][a][h >> 1][2 * (h & 1)], w[u][a][h >> 1][2 * (h & 1) + 1], scale(wk[u][a]));
#pragma unroll
                for (int b = 0; b < FM; ++b)
                    fx[b] = widen(x[u][b][h >> 1][2 * (h & 1)], x[u][b][h >> 1][2 * (h & 1) + 1], scale(xk[u][b]));
#pragma unroll
                for (int a = 0; a < FN; ++a)
#pragma unroll
                    for (int b = 0; b < FM; ++b)
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[a], fx[b], acc[a][b], 0, 0, 0);
            }
        }
    }
    // lane (li, lq), register r of block (a, b): column 16 a + 4 lq + r of row 16 b + li
    if constexpr (KG > 1) {
        __shared__ f4v_t sums[KG - 1][FN * FM][64];
        if (group > 0) {
#pragma unroll
            for (int n = 0; n < FN * FM; ++n) sums[group - 1][n][lane] = acc[n / FM][n % FM];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; ++g)
#pragma unroll
            for (int n = 0; n < FN * FM; ++n) acc[n / FM][n % FM] += sums[g][n][lane];
    }
#pragma unroll
    for (int a = 0; a < FN; ++a) {
        const int j = j0 + 16 * a + 4 * lq;
#pragma unroll
        for (int b = 0; b < FM; ++b) {
            const int i = i0 + 16 * b + li;
            if (i >= p.M || j >= p.N) continue;
            const size_t at = static_cast<size_t>(i) * p.N + j;
            float bias[4] = {}, res[4] = {};
            const bool whole = j + 4 <= p.N;
            if (whole) {
                if (p.bias) *reinterpret_cast<pk4u_t *>(bias) = *reinterpret_cast<const pk4u_t *>(p.bias + j);
                if (p.residual) *reinterpret_cast<pk4u_t *>(res) = *reinterpret_cast<const pk4u_t *>(p.residual + at);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (j + r >= p.N) continue;
                    if (p.bias) bias[r] = p.bias[j + r];
                    if (p.residual) res[r] = p.residual[at + r];
                }
            }
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = acc[a][b][r];
                if (p.bias) v += bias[r];
                float slope;
                v = activate<false>(v, p.act, slope);
                if (p.residual) v += res[r];
                o[r] = v;
            }
            if (whole) {
                *reinterpret_cast<pk4u_t *>(p.y + at) = pk4u_t{o[0], o[1], o[2], o[3]};
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (j + r < p.N) p.y[at + r] = o[r];
            }
        }
    }
}

template <int FN, int FM, int KG>
void launch_packed(PackedProduct p, hipStream_t s) {
    p.tiles_n = (p.N + 16 * FN - 1) / (16 * FN);
    const size_t tiles = static_cast<size_t>(p.tiles_n) * ((p.M + 16 * FM - 1) / (16 * FM));
    launch((packed_direct<FN, FM, KG>), dim3(static_cast<unsigned>(tiles)), dim3(64 * KG), 0, s, p);
}

template <int FN, int FM>
void launch_packed(const PackedProduct &p, hipStream_t s) {
    const size_t tiles = static_cast<size_t>((p.N + 16 * FN - 1) / (16 * FN)) * ((p.M + 16 * FM - 1) / (16 * FM));
    const size_t waves = static_cast<size_t>(device_cu_count()) * 16;
    int kg = 1;
    while (kg < 8 && tiles * kg * 2 <= waves && kg * 2 <= p.groups) kg *= 2;
    if (kg == 8) launch_packed<FN, FM, 8>(p, s);
    else if (kg == 4) launch_packed<FN, FM, 4>(p, s);
    else if (kg == 2) launch_packed<FN, FM, 2>(p, s);
    else launch_packed<FN, FM, 1>(p, s);
}

}  // namespace

}  // namespace tship

using namespace tship;

extern "C" {

size_t ts_hip_linear_packed_workspace_floats(size_t batch, size_t fan_in, size_t fan_out) {
    return planes_take(batch, fan_out, fan_in)
               ? planes_workspace_floats(batch, fan_out, fan_in, Src::kCodesK, Src::kCodesK)
               : 0;
}

int ts_hip_linear_packed(const uint8_t *x_codes, const uint8_t *x_scales, const uint8_t *w_codes,
                         const uint8_t *w_scales, size_t batch, size_t fan_in, size_t fan_out, const float *bias,
                         int act, const float *residual, float *y, float *workspace, size_t workspace_floats,
                         void *stream) {
    const size_t lim = size_t(1) << 24;
    if (batch >= lim || fan_in >= lim || fan_out >= lim || batch * fan_out >= size_t(1) << 34 || act < TS_HIP_ACT_NONE || act > TS_HIP_ACT_GELU_TANH)
        return TS_HIP_EINVAL;
    if (batch == 0 || fan_out == 0) return TS_HIP_OK;
    if (!y || (fan_in && (!x_codes || !x_scales || !w_codes || !w_scales))) return TS_HIP_EINVAL;
    if (workspace_floats < ts_hip_linear_packed_workspace_floats(batch, fan_in, fan_out)) return TS_HIP_EWORKSPACE;
    if (planes_take(batch, fan_out, fan_in)) {
        if (!workspace && ts_hip_linear_packed_workspace_floats(batch, fan_in, fan_out)) return TS_HIP_EINVAL;
        LinearProduct q{};
        q.A = {nullptr, nullptr, x_codes, x_scales, 0, static_cast<int>(batch), packed_pitch(fan_in), batch};
        q.B = {nullptr, nullptr, w_codes, w_scales, 0, static_cast<int>(fan_out), packed_pitch(fan_in), fan_out};
        q.a = q.b = Src::kCodesK;
        q.M = static_cast<int>(batch);
        q.N = static_cast<int>(fan_out);
        q.K = static_cast<int>(fan_in);
        q.C = y;
        q.epi = {bias, residual, nullptr, nullptr, act};
        planes_multiply(q, workspace, nullptr, nullptr, as_stream(stream));
        return launch_status();
    }
    const PackedProduct p = {x_codes, x_scales, w_codes, w_scales, bias, residual, y, static_cast<int>(batch),
                             static_cast<int>(fan_out), static_cast<int>(packed_pitch(fan_in) / kPackGroup), act, 0};
    if (batch <= 16) launch_packed<1, 1>(p, as_stream(stream));
    else launch_packed<2, 2>(p, as_stream(stream));
    return launch_status();
}

}  // extern "C"
