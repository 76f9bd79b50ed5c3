// Layer norm with the residual's addition (ts_hip.h, ts_hip_layer_norm and the entries
// after it), its form in 8 bits with a scale per 128 columns, and its backward.
//
//   h = x + residual,  m = mean(h),  r = 1 / sqrt(mean((h - m)^2) + eps),  u = (h - m) r
//   y = u w + b
//   g = go w:  dh = r (g - mean(g) - u mean(g u)),  dw = sum over rows of go u,  db = of go
//
// A row is held in registers and memory passed over once, as in ts_hip_norm.h.  The
// sums are of d = h - K with K the row's first value, in f64: sum d, sum d^2, and
// backward sum g and sum g d, so that one exchange between a row's waves is enough.
// K being one of the n values, (m - K)^2 <= n var, and var = mean(d^2) - mean(d)^2 loses
// no more than a factor n of f64's 2^-53 however far the row is from zero.
// m is kept as two fp32, and h - m taken in fp32, exactly where h is near m.
#include "ts_hip_block8.h"
#include "ts_hip_norm.h"

namespace tship {

namespace {

// What a row's sums of d say of its values: u = ((h pre - mh) - ml) post rf, pre and post
// being r's power of two: before the differences, so that tiny rows' means keep their
// bits, but after them where a far row's values would leave fp32.
struct RowNorm {
    float pre, post, rf, mh, ml;
    __device__ __forceinline__ float unit(float h) const { return ((h * pre - mh) - ml) * post * rf; }
};
__device__ __forceinline__ RowNorm row_norm(double shift, double mean_d, double r) {
    const RowScale s = row_scale(r);
    const double far = fabs(shift + mean_d) * s.up;  // (the values are within sqrt(cols) of it)
    const float pre = s.up <= 1.0f || far < 0x1p100 ? s.up : 1.0f;
    const double mean = (shift + mean_d) * pre;
    const float hi = static_cast<float>(mean);
    return {pre, pre == s.up ? 1.0f : s.up, static_cast<float>(s.f), hi, static_cast<float>(mean - hi)};
}
__device__ __forceinline__ double row_r(double mean_d, double mean_dd, double eps) {
    const double var = mean_dd - mean_d * mean_d;
    return 1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps);  // (a NaN stays)
}

// columns past the row: its first value, so that d is 0
__device__ __forceinline__ void fill_past(float (&v)[4], size_t c, size_t cols, float first) {
    if (c + 4 <= cols) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e >= cols) v[e] = first;
}

struct LayerNormArgs {
    const float *x, *residual, *weight, *bias;
    float *h, *y;  // h: with a residual
    uint8_t *codes;
    float *scales;  // packed
    size_t rows, cols, pitch;
    double eps;
};

// A row per W waves; LONG: more columns than the waves hold, passed over twice.
template <int W, int NV, bool RES, bool PACK, bool LONG>
__global__ __launch_bounds__(kNormThreads<W>) void layer_norm_rows(LayerNormArgs a) {
    constexpr int RPB = kNormRows<W>;
    __shared__ double lds[RPB * 2 * W];
    const int slot = threadIdx.x / (64 * W), t = threadIdx.x % (64 * W);
    const size_t span = static_cast<size_t>(256) * W * NV, end = PACK ? a.pitch : a.cols;
    float w[NV][4], b[NV][4];
    auto weights = [&](size_t from) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t c = from + 4 * (t + 64 * W * i);
            load4(a.weight, c, a.cols, w[i]);
            if (a.bias) {  // uniform
                load4(a.bias, c, a.cols, b[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) b[i][e] = 0.0f;
            }
        }
    };
    if (!LONG) weights(0);
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    for (size_t row = static_cast<size_t>(blockIdx.x) * RPB + slot; row < a.rows; row += step) {  // (W > 1: uniform)
        const size_t base = row * a.cols;
        const float *x = a.x + base, *res = RES ? a.residual + base : nullptr;
        const float first = RES ? x[0] + res[0] : x[0];
        const double shift = first;
        float v[NV][4];
        auto fetch = [&](size_t c0) {  // h of the columns from c0 on
            float r[NV][4];
#pragma unroll
            for (int i = 0; i < NV; ++i) load4(x, c0 + 4 * (t + 64 * W * i), a.cols, v[i]);
            if (RES) {
#pragma unroll
                for (int i = 0; i < NV; ++i) load4(res, c0 + 4 * (t + 64 * W * i), a.cols, r[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][e] += r[i][e];
            }
        };
        double s[2] = {0.0, 0.0};
        size_t c0 = 0;
        do {
            fetch(c0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                fill_past(v[i], c0 + 4 * (t + 64 * W * i), a.cols, first);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double d = v[i][e] - shift;
                    s[0] += d;
                    s[1] += d * d;
                }
            }
            c0 += span;
        } while (LONG && c0 < a.cols);
        row_sum<W, 2>(s, lds + slot * 2 * W);
        const double cols = static_cast<double>(a.cols), mean_d = s[0] / cols;
        const double r = row_r(mean_d, s[1] / cols, a.eps), mean = shift + mean_d;
        const RowNorm n = row_norm(shift, mean_d, r);
        c0 = 0;
        do {
            if (LONG) {
                fetch(c0);
                weights(c0);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t c = c0 + 4 * (t + 64 * W * i);
                if (c >= end) continue;
                if (RES) store4(a.h + base, c, a.cols, v[i]);
                if constexpr (PACK) {  // in f64: a code takes the side of its border that y itself is on
                    double o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[e] = c + e < a.cols ? __builtin_fma((v[i][e] - mean) * r, static_cast<double>(w[i][e]), static_cast<double>(b[i][e])) : 0.0;
                    block8_store(o, c, a.codes + row * a.pitch, a.scales + row, a.rows);
                } else {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(n.unit(v[i][e]), w[i][e], b[i][e]);
                    store4(a.y + base, c, a.cols, o);
                }
            }
            c0 += span;
        } while (LONG && c0 < end);
    }
}

struct LayerNormBackArgs {
    const float *h, *weight, *go;
    float *dh, *dw_part, *db_part;  // parts: [gridDim.x][cols]; db_part may be null beside dw_part
    RowNorm *norms;                 // LONG with parts: each row's
    float2 *means;                  // and its mean(g) and mean(g u)
    size_t rows, cols;
    double eps;
    float *dw, *db;    // with a ticket: the last workgroup adds the parts up
    unsigned *ticket;  // zero, and zero again when the launch has run; null: none
};

// Rows blockIdx.x * RPB + slot, and on by the grid's; a thread keeps the sums of its
// columns for dw and db (f64), the workgroup's go to the parts.  LONG with DP: no thread
// has columns of its own; what a row's values need is left for long_layer_columns.
template <int W, int NV, bool DH, bool DP, bool LONG>
__global__ __launch_bounds__(kNormThreads<W>) void layer_norm_back(LayerNormBackArgs a) {
    constexpr int RPB = kNormRows<W>;
    __shared__ double lds[RPB * 4 * W];
    const int slot = threadIdx.x / (64 * W), t = threadIdx.x % (64 * W);
    const size_t span = static_cast<size_t>(256) * W * NV;
    // dw's sums stand in registers; where 16 waves of four quads leave none, in shared
    // memory, each thread its own, and db's alone in registers
    constexpr bool SHARED = DP && !LONG && W * NV >= 64;
    __shared__ double held[SHARED ? NV * 4 * 64 * W : 1];
    double own[SHARED ? 1 : NV][4] = {}, db[NV][4] = {};
    auto dw = [&](int i, int e) -> double & {
        if constexpr (SHARED) return held[(i * 4 + e) * 64 * W + t];
        else return own[i][e];
    };
    if constexpr (SHARED) {
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) dw(i / 4, i % 4) = 0.0;
    }
    float w[NV][4];
    auto weights = [&](size_t c0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load4(a.weight, c0 + 4 * (t + 64 * W * i), a.cols, w[i]);
    };
    if (!LONG) weights(0);
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    // every wave of the workgroup takes every round (the barriers)
    for (size_t r0 = static_cast<size_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += step) {
        const size_t row = r0 + slot;
        const bool live = row < a.rows;
        const size_t base = live ? row * a.cols : 0, n = live ? a.cols : 0;
        float h[NV][4], g[NV][4];
        const float first = a.h[base];
        const double shift = first;
        auto fetch = [&](size_t c0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load4(a.h + base, c0 + 4 * (t + 64 * W * i), n, h[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i) load4(a.go + base, c0 + 4 * (t + 64 * W * i), n, g[i]);
        };
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        size_t c0 = 0;
        do {
            fetch(c0);
            if (LONG) weights(c0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                fill_past(h[i], c0 + 4 * (t + 64 * W * i), n, first);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double d = h[i][e] - shift, gw = static_cast<double>(g[i][e]) * w[i][e];
                    s[0] += d;
                    s[1] += d * d;
                    s[2] += gw;
                    s[3] += gw * d;
                }
            }
            c0 += span;
        } while (LONG && c0 < a.cols);
        row_sum<W, 4>(s, lds + slot * 4 * W);
        const double cols = static_cast<double>(a.cols), mean_d = s[0] / cols;
        const double r = row_r(mean_d, s[1] / cols, a.eps);
        const RowNorm norm = row_norm(shift, mean_d, r);
        const float mean_g = static_cast<float>(s[2] / cols), mean_gu = static_cast<float>(r * ((s[3] - mean_d * s[2]) / cols));
        if (DP && LONG) {
            if (t == 0) {
                a.norms[row] = norm;
                a.means[row] = make_float2(mean_g, mean_gu);
            }
            continue;
        }
        c0 = 0;
        do {
            if (LONG) {
                fetch(c0);
                weights(c0);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t c = c0 + 4 * (t + 64 * W * i);
                float u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = norm.unit(h[i][e]);
                if (DH && c < n) {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[e] = norm.post * (norm.pre * (norm.rf * (g[i][e] * w[i][e] - mean_g - u[e] * mean_gu)));
                    store4(a.dh + base, c, a.cols, o);
                }
                if (DP && !LONG && live) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        dw(i, e) += static_cast<double>(g[i][e]) * u[e];
                        db[i][e] += g[i][e];
                    }
                }
            }
            c0 += span;
        } while (LONG && c0 < a.cols);
    }
    if (DP && !LONG) {
        if constexpr (RPB > 1) {  // the workgroup's rows together, in their order
            __shared__ double sum[(RPB - 1) * 64 * W * NV * 4];
            auto join = [&](double (&v)[NV][4]) {
                __syncthreads();
                if (slot > 0) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[((slot - 1) * NV * 4 + i * 4 + e) * 64 * W + t] = v[i][e];
                }
                __syncthreads();
                if (slot == 0) {
#pragma unroll
                    for (int k = 0; k < RPB - 1; ++k)
#pragma unroll
                        for (int i = 0; i < NV; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[i][e] += sum[(k * NV * 4 + i * 4 + e) * 64 * W + t];
                }
            };
            join(own);
            join(db);
        }
        if (slot == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t c = 4 * (t + 64 * W * i), at = static_cast<size_t>(blockIdx.x) * a.cols;
                float o[4];
                if (c >= a.cols) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(dw(i, e));
                if (a.dw_part) store4(a.dw_part + at, c, a.cols, o);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(db[i][e]);
                if (a.db_part) store4(a.db_part + at, c, a.cols, o);
            }
        }
    }
    if (DP && a.ticket) {  // uniform: the last workgroup to get here adds the parts up
        __shared__ bool last;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        for (size_t c = threadIdx.x; c < 2 * a.cols; c += kNormThreads<W>) {
            const bool second = c >= a.cols;
            const size_t at = second ? c - a.cols : c;
            const float *part = second ? a.db_part : a.dw_part;
            if (!part) continue;
            double s = 0.0;
#pragma unroll 16
            for (size_t g = 0; g < gridDim.x; ++g) s += part[g * a.cols + at];
            (second ? a.db : a.dw)[at] = static_cast<float>(s);
        }
        if (threadIdx.x == 0) *a.ticket = 0;
    }
}

// dw, db and dh of rows longer than a workgroup holds, by columns: a thread has four of
// them, of `run` rows (sums: f64).  The first pass by rows takes their sums alone.
template <bool DH>
__global__ __launch_bounds__(kBlock) void long_layer_columns(LayerNormBackArgs a, size_t run) {
    const size_t c = blockIdx.x * kLongCols + 4 * threadIdx.x, first = blockIdx.y * run;
    if (c >= a.cols) return;
    const size_t last = first + run < a.rows ? first + run : a.rows;
    float w[4];
    if (DH) load4(a.weight, c, a.cols, w);
    double s[4] = {}, sb[4] = {};
#pragma unroll 4
    for (size_t row = first; row < last; ++row) {
        const RowNorm norm = a.norms[row];
        const float2 mean = a.means[row];
        const size_t base = row * a.cols;
        float h[4], g[4], u[4];
        load4(a.h + base, c, a.cols, h);
        load4(a.go + base, c, a.cols, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u[e] = norm.unit(h[e]);
            s[e] += static_cast<double>(g[e]) * u[e];
            sb[e] += g[e];
        }
        if (DH) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = norm.post * (norm.pre * (norm.rf * (g[e] * w[e] - mean.x - u[e] * mean.y)));
            store4(a.dh + base, c, a.cols, o);
        }
    }
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(s[e]);
    if (a.dw_part) store4(a.dw_part + blockIdx.y * a.cols, c, a.cols, o);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(sb[e]);
    if (a.db_part) store4(a.db_part + blockIdx.y * a.cols, c, a.cols, o);
}

// two sums' parts by one launch
__global__ __launch_bounds__(kBlock) void sum_two_parts(PartSums first, PartSums second) {
    __shared__ double lds[kPartSumsLds];
    const int block = static_cast<int>(blockIdx.x);
    if (block < first.blocks) part_sums_block(first, block, lds);  // (uniform)
    else part_sums_block(second, block - first.blocks, lds);
}

template <int W, int NV, bool LONG>
void launch_layer_norm(const LayerNormArgs &a, bool pack, hipStream_t s) {
    const size_t need = (a.rows + kNormRows<W> - 1) / kNormRows<W>;
    const dim3 grid(static_cast<unsigned>(need < kMaxBlocks ? need : kMaxBlocks)), block(kNormThreads<W>);
    if (a.residual && pack) launch((layer_norm_rows<W, NV, true, true, LONG>), grid, block, 0, s, a);
    else if (a.residual) launch((layer_norm_rows<W, NV, true, false, LONG>), grid, block, 0, s, a);
    else if (pack) launch((layer_norm_rows<W, NV, false, true, LONG>), grid, block, 0, s, a);
    else launch((layer_norm_rows<W, NV, false, false, LONG>), grid, block, 0, s, a);
}

template <int W, int NV, bool LONG>
void launch_layer_back(const LayerNormBackArgs &a, unsigned grid, hipStream_t s) {
    const dim3 block(kNormThreads<W>);
    const bool parts = a.dw_part || a.db_part;
    if (a.dh && parts) launch((layer_norm_back<W, NV, true, true, LONG>), dim3(grid), block, 0, s, a);
    else if (a.dh) launch((layer_norm_back<W, NV, true, false, LONG>), dim3(grid), block, 0, s, a);
    else launch((layer_norm_back<W, NV, false, true, LONG>), dim3(grid), block, 0, s, a);
}

int layer_norm_forward(const float *x, const float *residual, const float *weight, const float *bias, size_t rows, size_t cols,
                       float eps, float *h, float *y, uint8_t *codes, float *scales, void *stream) {
    if (rows == 0 || cols == 0) return TS_HIP_OK;
    if (!x || !weight || (residual != nullptr) != (h != nullptr) || rows >= kMaxRows) return TS_HIP_EINVAL;
    const LayerNormArgs a = {x, residual, weight, bias, h, y, codes, scales, rows, cols, packed_pitch(cols), eps};
    for_cols(codes ? a.pitch : cols, false, [&](auto w, auto nv, auto long_rows) {
        launch_layer_norm<w.value, nv.value, long_rows.value>(a, codes != nullptr, as_stream(stream));
    });
    return launch_status();
}

constexpr size_t kRowFloats = (sizeof(RowNorm) + sizeof(float2)) / sizeof(float);  // LONG: a row's in the workspace

}  // namespace

}  // namespace tship

using namespace tship;

extern "C" {

int ts_hip_layer_norm(const float *x, const float *residual, const float *weight, const float *bias, size_t rows, size_t cols,
                      float eps, float *h, float *y, void *stream) {
    if (rows && cols && !y) return TS_HIP_EINVAL;
    return layer_norm_forward(x, residual, weight, bias, rows, cols, eps, h, y, nullptr, nullptr, stream);
}

int ts_hip_layer_norm_block8(const float *x, const float *residual, const float *weight, const float *bias, size_t rows,
                             size_t cols, float eps, float *h, uint8_t *codes, float *scales, void *stream) {
    if (rows && cols && (!codes || !scales)) return TS_HIP_EINVAL;
    return layer_norm_forward(x, residual, weight, bias, rows, cols, eps, h, nullptr, codes, scales, stream);
}

size_t ts_hip_layer_norm_backward_workspace_floats(size_t rows, size_t cols) {
    return 2 * back_blocks(rows, cols) * cols + (cols > kMaxHeldCols ? kRowFloats * rows : 0);
}

int ts_hip_layer_norm_backward(const float *h, const float *weight, const float *go, size_t rows, size_t cols, float eps,
                               float *dh, float *dweight, float *dbias, float *workspace, size_t workspace_floats,
                               unsigned *ticket, void *stream) {
    const bool parts = dweight || dbias;
    if (cols == 0 || (!dh && !parts)) return TS_HIP_OK;
    if (rows == 0) {
        int status = dweight ? ts_hip_fill(dweight, 0.0f, cols, stream) : TS_HIP_OK;
        if (status == TS_HIP_OK && dbias) status = ts_hip_fill(dbias, 0.0f, cols, stream);
        return status;
    }
    if (!h || !weight || !go || rows >= kMaxRows) return TS_HIP_EINVAL;
    if (parts && (!workspace || workspace_floats < ts_hip_layer_norm_backward_workspace_floats(rows, cols)))
        return TS_HIP_EWORKSPACE;
    const unsigned grid = static_cast<unsigned>(back_blocks(rows, cols));
    const bool long_rows = cols > kMaxHeldCols;
    if (!parts || long_rows || grid > kTicketParts || grid * cols > kTicketFloats) ticket = nullptr;
    // workspace: a long row's means and norms, then the parts
    float2 *const means = reinterpret_cast<float2 *>(workspace);
    RowNorm *const norms = reinterpret_cast<RowNorm *>(workspace + 2 * rows);
    float *const sums = parts ? workspace + (long_rows ? kRowFloats * rows : 0) : nullptr;
    const LayerNormBackArgs a = {h, weight, go, dh, dweight ? sums : nullptr, dbias ? sums + grid * cols : nullptr,
                                 norms, means, rows, cols, eps, dweight, dbias, ticket};
    const hipStream_t s = as_stream(stream);
    for_cols(cols, false, [&](auto w, auto nv, auto lng) { launch_layer_back<w.value, nv.value, lng.value>(a, grid, s); });
    size_t count = grid;
    if (parts && long_rows) {
        const size_t run = long_run(rows, cols);
        count = (rows + run - 1) / run;
        const dim3 columns(static_cast<unsigned>((cols + kLongCols - 1) / kLongCols), static_cast<unsigned>(count));
        if (dh) launch(long_layer_columns<true>, columns, dim3(kBlock), 0, s, a, run);
        else launch(long_layer_columns<false>, columns, dim3(kBlock), 0, s, a, run);
    }
    if (parts && !ticket) {
        const PartSums none{}, w = dweight ? part_sums(a.dw_part, count, cols, dweight) : none,
                       b = dbias ? part_sums(a.db_part, count, cols, dbias) : none;
        launch(sum_two_parts, dim3(static_cast<unsigned>(w.blocks + b.blocks)), dim3(kBlock), 0, s, w, b);
    }
    return launch_status();
}

}  // extern "C"
