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
//
// What bounds it is memory.  8192 x 4096 with the residual: forward 90 us (537 MB, 6.0 TB/s),
// packed 82 (437 MB, 5.3), backward 86 (403 MB, 4.7) and 6.5 for the parts' sums; a copy of
// 2 GB reaches 4.9, one that the last cache holds 8.7.  3000 x 1003 without it: 7.2,
// 12.4 and 4.0.  128 x 784: 4.6 and 12; 1 x 4096 packed 4.8 (a launch alone is 2 to 3).
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
    const double v = (var < 0.0 ? 0.0 : var) + eps;  // (a NaN stays)
    // 1 / sqrt(v): the instruction's 24 bits and one step of third order; 0, infinity and NaN: the instruction's
    const double r = __builtin_amdgcn_rsq(v), e = __builtin_fma(-v * r, r, 1.0);
    return v > 0.0 && v < __builtin_inf() ? __builtin_fma(r * e, __builtin_fma(0.375, e, 0.5), r) : r;
}

// columns past the row: its first value, so that d is 0
__device__ __forceinline__ void fill_past(float (&v)[4], size_t c, size_t cols, float first) {
    if (c + 4 <= cols) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e >= cols) v[e] = first;
}

// A row has W waves, or half a wave (W 0): its lanes, the rows of a wave and of a workgroup.
// us, 16384 x 64 by half waves and by waves: forward 8.6, 13; backward 10.5, 15.
template <int W>
constexpr int kRowLanes = W ? 64 * W : 32;
template <int W>
constexpr int kWaveRows = W ? 1 : 2;
template <int W>
constexpr int kLayerRows = kNormThreads<W> / kRowLanes<W>;

// The sum over a row's lanes, in every one, joined within a wave by DPP.  lds: N * W doubles
// of this row, others than the last row's (a barrier stands between the two).
constexpr int kBcast15 = 0x142, kBcast31 = 0x143;
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_0(double v) {  // 0 in the other rows of 16
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false));
}
template <int W, int N>
__device__ __forceinline__ void row_sums(double (&s)[N], double *lds) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        double v = s[n];
        v += dpp<0xB1>(v);   // lanes 1 0 3 2
        v += dpp<0x4E>(v);   // lanes 2 3 0 1
        v += dpp<0x141>(v);  // eight lanes mirrored
        v += dpp<0x140>(v);  // sixteen lanes mirrored
        if (W == 0) {  // the neighbouring row of 16: one copy ends with the even rows, the other with the odd
            const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
            const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
            s[n] = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
            continue;
        }
        v += dpp_or_0<kBcast15, 0xa>(v);
        v += dpp_or_0<kBcast31, 0xc>(v);  // lane 63: all
        s[n] = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
    }
    if constexpr (W > 1) {
        const int wave = (threadIdx.x >> 6) % W;
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
}

// The rows that a wave has of a round's from r0 on: the first of them and how many there are
// (uniform), the lane's own.
template <int W>
struct WaveRows {
    size_t first, row;
    unsigned there;
    bool live;
    __device__ __forceinline__ WaveRows(size_t r0, int wave_row, int slot, size_t rows) : first(r0 + wave_row), row(r0 + slot) {
        there = first < rows ? static_cast<unsigned>(min(rows - first, static_cast<size_t>(kWaveRows<W>))) : 0;
        live = row < rows;
        if (!there) first = 0;
    }
    __device__ __forceinline__ size_t at(size_t cols) const { return W || !live ? first * cols : row * cols; }  // (a row that exists)
};

// A lane's quads c = 4 (t + lanes i) of rows of `cols` columns, by the buffer instructions,
// for which a lane past the row is one past the buffer: 0 comes back, nothing is written.
// The quad that a row ends in is read from the row's last four columns and moved into place.
template <int W, int NV>
struct RowQuads {
    unsigned t, cols;
    int wave, parts;  // the wave's place in the row, the row's parts of 256 columns
    unsigned skip;    // bytes from the wave's first row to the lane's
    static constexpr int L = kRowLanes<W>;
    __device__ __forceinline__ RowQuads(unsigned t, size_t cols)
        : t(t), cols(static_cast<unsigned>(cols)), wave(__builtin_amdgcn_readfirstlane(t / 64)), parts(static_cast<int>((cols + 255) / 256)),
          skip(W ? 0 : threadIdx.x % 64 / L * 4 * static_cast<unsigned>(cols)) {}
    __device__ __forceinline__ unsigned col(int i) const { return 4 * (t + L * i); }
    // whether any lane of the wave has columns of quad i (uniform): what is past the row is not
    // computed (backward, us: 3400 x 4100 46, 51 with it computed; 1700 x 8200 53, 67)
    __device__ __forceinline__ bool some(int i) const { return i == 0 || W * i + wave < parts; }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const float *p, unsigned rows) const {  // p, rows: uniform
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p), 0, static_cast<int>(4 * cols * rows), 0x00020000);
    }
    // the lane's quads of the row at p, or of its own of the rows there (by: its skip)
    __device__ __forceinline__ void load(const float *p, unsigned rows, float (&v)[NV][4], unsigned by = 0) const {
        const __amdgpu_buffer_rsrc_t r = buffer(p, rows);
        if (W == 0 && cols < 4) {  // uniform
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[i][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, col(i) + e < cols ? by + 4 * (col(i) + e) : kPast, 0, 0));
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned off = col(i) < cols ? by + 4 * min(col(i), cols - 4) : kPast;
            const f4v_t q = __builtin_bit_cast(f4v_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = q[e];
        }
    }
    // what was loaded into place, and `past` in the columns past the row
    __device__ __forceinline__ void fill(float (&v)[NV][4], float past) const {
        if (cols == 4 * L * NV) return;  // uniform
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned c = col(i);
            const bool ends = c < cols && c + 4 > cols && cols >= 4;
            if (cols & 1) {  // uniform: by 4 - cols % 4
#pragma unroll
                for (int e = 0; e < 3; ++e) v[i][e] = ends ? v[i][e + 1] : v[i][e];
            }
            if ((cols & 3) == 1 || (cols & 3) == 2) {
#pragma unroll
                for (int e = 0; e < 2; ++e) v[i][e] = ends ? v[i][e + 2] : v[i][e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = c + e < cols ? v[i][e] : past;
        }
    }
    // quad i of the lane's row, of the rows at p (a lane whose row is not there does not call)
    __device__ __forceinline__ void store(float *p, unsigned rows, int i, const float (&v)[4]) const {
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        const unsigned c = col(i), off = c + 4 <= cols ? skip + 4 * c : kPast;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, f4v_t{v[0], v[1], v[2], v[3]}), buffer(p, rows), off, 0, 0);
        if (cols & 3) {  // uniform
            if (c < cols && c + 4 > cols) {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (c + e < cols) p[skip / 4 + c + e] = v[e];
            }
        }
    }
    static constexpr unsigned kPast = 0x80000000u;
};

struct LayerNormArgs {
    const float *x, *residual, *weight, *bias;
    float *h, *y;  // h: with a residual
    uint8_t *codes;
    float *scales;  // packed
    size_t rows, cols, pitch;
    double eps, per_col;  // 1 / cols
};

// s += a quad's part of sum d and sum d^2
__device__ __forceinline__ void norm_sums(const float (&h)[4], double shift, double (&s)[2]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double d = h[e] - shift;
        s[0] += d;
        s[1] += d * d;
    }
}

// What a row's sums say of its output; packed in f64: a code takes the side of its border
// that y itself is on
struct RowOut {
    RowNorm norm;
    double mean, r;
    __device__ __forceinline__ RowOut(const double (&s)[2], double per_col, double shift, double eps) {
        const double mean_d = s[0] * per_col;
        r = row_r(mean_d, s[1] * per_col, eps);
        mean = shift + mean_d;
        norm = row_norm(shift, mean_d, r);
    }
    __device__ __forceinline__ float y(float h, float w, float b) const { return __builtin_fmaf(norm.unit(h), w, b); }
    __device__ __forceinline__ double wide_y(float h, float w, float b) const {
        return __builtin_fma((h - mean) * r, static_cast<double>(w), static_cast<double>(b));
    }
};

// A row per W waves (or half a wave), and on by the grid's where there are more rows than workgroups.
template <int W, int NV, bool RES, bool PACK>
__global__ __launch_bounds__(kNormThreads<W>, 4) void layer_norm_rows(LayerNormArgs a) {
    constexpr int RPB = kLayerRows<W>, L = kRowLanes<W>;
    __shared__ double lds[W > 1 ? RPB * 2 * 2 * W : 1];
    const int wave_row = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 / L, t = threadIdx.x % L;
    const int slot = W ? wave_row : threadIdx.x / L;
    const RowQuads<W, NV> at(t, a.cols);
    float w[NV][4], b[NV][4];
    at.load(a.weight, 1, w);
    at.load(a.bias, a.bias ? 1 : 0, b);
    at.fill(w, 0.0f);
    at.fill(b, 0.0f);
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    int turn = 0;
    // every wave of the workgroup takes every round (the barriers)
    for (size_t r0 = static_cast<size_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += step) {
        const WaveRows<W> rows(r0, wave_row, slot, a.rows);
        const size_t base = rows.first * a.cols, own = rows.at(a.cols);
        float v[NV][4], first = a.x[own];
        at.load(a.x + base, rows.there, v, at.skip);
        if constexpr (RES) {
            float r[NV][4];
            at.load(a.residual + base, rows.there, r, at.skip);
            first += a.residual[own];
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] += r[i][e];
        }
        at.fill(v, first);
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (int i = 0; i < NV; ++i) norm_sums(v[i], first, s);
        row_sums<W, 2>(s, W > 1 ? lds + (slot * 2 + turn) * 2 * W : lds);
        turn ^= 1;
        if (!rows.live) continue;  // (uniform in a wave, past the round's barrier)
        const RowOut out(s, a.per_col, first, a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (RES) at.store(a.h + base, rows.there, i, v[i]);
            if constexpr (PACK) {
                const size_t c = at.col(i);
                if (c >= a.pitch) continue;  // (whole blocks)
                // a quad after the other, and nothing in f64 kept for it: registers
#pragma unroll
                for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(v[i][e]), "+v"(w[i][e]), "+v"(b[i][e])::"memory");
                double o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = c + e < a.cols ? out.wide_y(v[i][e], w[i][e], b[i][e]) : 0.0;
                block8_store(o, c, a.codes + rows.row * a.pitch, a.scales + rows.row, a.rows);
            } else {
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = out.y(v[i][e], w[i][e], b[i][e]);
                at.store(a.y + base, rows.there, i, o);
            }
        }
    }
}

// A row longer than a workgroup holds, passed over twice.
template <bool RES, bool PACK>
__global__ __launch_bounds__(1024) void long_layer_norm(LayerNormArgs a) {
    constexpr int W = 16, NV = 4;
    __shared__ double lds[2 * 2 * W];
    const size_t cols = a.cols, span = static_cast<size_t>(256) * W * NV, end = PACK ? a.pitch : cols;
    int turn = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {  // uniform
        const size_t base = row * cols;
        const float first = RES ? a.x[base] + a.residual[base] : a.x[base];
        auto pass = [&](size_t end, auto &&f) {
            for (size_t c0 = 4 * threadIdx.x; c0 < end; c0 += span) {
                float v[NV][4], r[NV][4];
#pragma unroll
                for (int i = 0; i < NV; ++i) load4(a.x + base, c0 + 256 * W * i, cols, v[i]);
                if (RES) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) load4(a.residual + base, c0 + 256 * W * i, cols, r[i]);
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[i][e] += r[i][e];
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) f(c0 + 256 * W * i, v[i]);
            }
        };
        double s[2] = {0.0, 0.0};
        pass(cols, [&](size_t c, float (&v)[4]) {
            fill_past(v, c, cols, first);
            norm_sums(v, first, s);
        });
        row_sums<W, 2>(s, lds + turn * 2 * W);
        turn ^= 1;
        const RowOut out(s, a.per_col, first, a.eps);
        pass(end, [&](size_t c, const float (&v)[4]) {
            if (c >= end) return;  // (packed: whole blocks)
            float w[4], b[4] = {};
            load4(a.weight, c, cols, w);
            if (a.bias) load4(a.bias, c, cols, b);
            if (RES && c < cols) store4(a.h + base, c, cols, v);
            if constexpr (PACK) {
                double o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = c + e < cols ? out.wide_y(v[e], w[e], b[e]) : 0.0;
                block8_store(o, c, a.codes + row * a.pitch, a.scales + row, a.rows);
            } else {
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = out.y(v[e], w[e], b[e]);
                store4(a.y + base, c, cols, o);
            }
        });
    }
}

struct LayerNormBackArgs {
    const float *h, *weight, *go;
    float *dh, *dw_part, *db_part;  // parts: [gridDim.x][cols]; db_part may be null beside dw_part
    RowNorm *norms;                 // long rows with parts: each row's
    float2 *means;                  // and its mean(g) and mean(g u)
    size_t rows, cols;
    double eps, per_col;  // 1 / cols
    float *dw, *db;    // with a ticket: the last workgroup adds the parts up
    unsigned *ticket;  // zero, and zero again when the launch has run; null: none
};

// s += a quad's part of sum d, sum d^2, sum g and sum g d, with g = go w
__device__ __forceinline__ void back_sums(const float (&h)[4], const float (&go)[4], const float (&w)[4], double shift,
                                          double (&s)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double d = h[e] - shift, g = static_cast<double>(go[e]) * w[e];
        s[0] += d;
        s[1] += d * d;
        s[2] += g;
        s[3] += g * d;
    }
}

// What a row's sums say of its gradients
struct RowBack {
    RowNorm norm;
    float mean_g, mean_gu;
    __device__ __forceinline__ float dh(float go, float w, float u) const {
        return norm.post * (norm.pre * (norm.rf * (go * w - mean_g - u * mean_gu)));
    }
};
__device__ __forceinline__ RowBack row_back(const double (&s)[4], double per_col, double shift, double eps) {
    const double mean_d = s[0] * per_col, r = row_r(mean_d, s[1] * per_col, eps);
    return {row_norm(shift, mean_d, r), static_cast<float>(s[2] * per_col),
            static_cast<float>(r * ((s[3] - mean_d * s[2]) * per_col))};
}

// A lane's quads of a row of h and of go, and its first value
template <int NV>
struct BackRow {
    float h[NV][4], g[NV][4], first;
};

// Rows blockIdx.x * RPB + slot, and on by the grid's, the next one's values on their way
// while one is computed; a thread keeps the sums of its columns for dw and db (f64), the
// workgroup's go to the parts.
template <int W, int NV, bool DH, bool DP>
__global__ __launch_bounds__(kNormThreads<W>, 2) void layer_norm_back(LayerNormBackArgs a) {
    constexpr int RPB = kLayerRows<W>, L = kRowLanes<W>;
    __shared__ double lds[W > 1 ? RPB * 2 * 4 * W : 1];
    const int wave_row = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 / L, t = threadIdx.x % L;
    const int slot = W ? wave_row : threadIdx.x / L;
    // dw's sums stand in registers; where eight quads a lane leave none, in shared memory,
    // each thread its own, and db's alone in registers
    constexpr bool SHARED = DP && NV == 8;
    __shared__ double held[SHARED ? NV * 4 * L : 1];
    double own[SHARED ? 1 : NV][4] = {}, db[NV][4] = {};
    auto dw = [&](int i, int e) -> double & {
        if constexpr (SHARED) return held[(i * 4 + e) * L + t];
        else return own[i][e];
    };
    if constexpr (SHARED) {
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) dw(i / 4, i % 4) = 0.0;
    }
    const RowQuads<W, NV> at(t, a.cols);
    constexpr bool AHEAD = NV < 8;  // (there no registers are left for the next row)
    float w[NV][4];
    at.load(a.weight, 1, w);
    at.fill(w, 0.0f);
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    auto fetch = [&](size_t r0, BackRow<NV> &v) {  // a row past the last: zeros
        const WaveRows<W> rows(r0, wave_row, slot, a.rows);
        const size_t base = rows.first * a.cols;
        v.first = a.h[rows.at(a.cols)];
        at.load(a.h + base, rows.there, v.h, at.skip);
        at.load(a.go + base, rows.there, v.g, at.skip);
    };
    BackRow<NV> v, next;
    if (AHEAD) fetch(static_cast<size_t>(blockIdx.x) * RPB, next);
    int turn = 0;
    // every wave of the workgroup takes every round (the barriers)
    for (size_t r0 = static_cast<size_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += step) {
        const WaveRows<W> rows(r0, wave_row, slot, a.rows);
        if constexpr (AHEAD) {
            v = next;
            if (r0 + step < a.rows) fetch(r0 + step, next);
        } else {
            fetch(r0, v);
        }
        at.fill(v.h, v.first);
        at.fill(v.g, 0.0f);
        const double shift = v.first;
        double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!at.some(i)) continue;
            if (!AHEAD) {  // (or the weights' f64 stand in registers through the loop)
#pragma unroll
                for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(w[i][e]));
            }
            back_sums(v.h[i], v.g[i], w[i], shift, s);
        }
        row_sums<W, 4>(s, W > 1 ? lds + (slot * 2 + turn) * 4 * W : lds);
        turn ^= 1;
        if (!rows.live) continue;  // (uniform in a wave, past the round's barrier)
        const RowBack back = row_back(s, a.per_col, shift, a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!at.some(i)) continue;
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float go = v.g[i][e];
                asm volatile("" : "+v"(go));  // (or the first pass's f64 of it stands in a register until here)
                const float u = back.norm.unit(v.h[i][e]);
                if (DH) o[e] = back.dh(go, w[i][e], u);
                if (DP) {
                    dw(i, e) += static_cast<double>(go) * u;
                    db[i][e] += go;
                }
            }
            if (DH) at.store(a.dh + rows.first * a.cols, rows.there, i, o);
            if (SHARED) asm volatile("" ::: "memory");  // (or every quad's sums of dw are read first)
        }
    }
    if constexpr (!DP) return;
    if constexpr (RPB > 1) {  // the workgroup's rows together, in their order
        __shared__ double sum[(RPB - 1) * L * NV * 4];
        auto join = [&](double (&v)[NV][4]) {
            __syncthreads();
            if (slot > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[((slot - 1) * NV * 4 + i * 4 + e) * L + t] = v[i][e];
            }
            __syncthreads();
            if (slot == 0) {
#pragma unroll
                for (int k = 0; k < RPB - 1; ++k)
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[i][e] += sum[(k * NV * 4 + i * 4 + e) * L + t];
            }
        };
        join(own);
        join(db);
    }
    // The parts.  With a ticket they go past the caches of the chip's dies, and are there
    // before the ticket counts them (a fence would write back all that the die holds).
    if (slot == 0) {
        auto put = [&](float *part, auto &&value) {
            if (!part) return;  // uniform
            part += static_cast<size_t>(blockIdx.x) * a.cols;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t c = at.col(i);
                if (a.ticket) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < a.cols)
                            __hip_atomic_store(part + c + e, value(i, e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                } else {
                    const float o[4] = {value(i, 0), value(i, 1), value(i, 2), value(i, 3)};
                    if (c < a.cols) store4(part, c, a.cols, o);
                }
            }
        };
        put(a.dw_part, [&](int i, int e) { return static_cast<float>(dw(i, e)); });
        put(a.db_part, [&](int i, int e) { return static_cast<float>(db[i][e]); });
    }
    if (a.ticket) {  // uniform: the last workgroup to get here adds the parts up
        __shared__ bool last;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0)
            last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        __syncthreads();
        if (!last) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        // a thread a quad (a row's last one: its last four columns), or a column where there are fewer
        auto add_up = [&](auto value, size_t count, auto &&column) {
            using Value = decltype(value);
            for (size_t q = threadIdx.x; q < 2 * count; q += kNormThreads<W>) {
                const bool second = q >= count;
                const size_t c = column(second ? q - count : q);
                const float *part = (second ? a.db_part : a.dw_part);
                if (!part) continue;
                constexpr int n = sizeof(Value) / 4, batch = 32;
                double s[n] = {};
                for (unsigned g0 = 0; g0 < gridDim.x; g0 += batch) {
                    float v[batch][n];
#pragma unroll
                    for (int u = 0; u < batch; ++u)  // (past the last: it again, not added)
                        __builtin_memcpy(v[u], part + static_cast<size_t>(min(g0 + u, gridDim.x - 1)) * a.cols + c, sizeof(Value));
#pragma unroll
                    for (int u = 0; u < batch; ++u)
#pragma unroll
                        for (int e = 0; e < n; ++e) s[e] += g0 + u < gridDim.x ? v[u][e] : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < n; ++e) (second ? a.db : a.dw)[c + e] = static_cast<float>(s[e]);
            }
        };
        if (a.cols < 4) add_up(0.0f, a.cols, [](size_t q) { return q; });
        else add_up(pk4u_t{}, (a.cols + 3) / 4, [&](size_t q) { return q * 4 + 4 <= a.cols ? q * 4 : a.cols - 4; });
        if (threadIdx.x == 0) __hip_atomic_store(a.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// A row longer than a workgroup holds, passed over twice; with parts (DP) once, what its
// values need left for long_layer_columns.
template <bool DP>
__global__ __launch_bounds__(1024) void long_layer_rows(LayerNormBackArgs a) {
    constexpr int W = 16, NV = 4;
    __shared__ double lds[2 * 4 * W];
    const size_t cols = a.cols, span = static_cast<size_t>(256) * W * NV;
    int turn = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {  // uniform
        const size_t base = row * cols;
        const float first = a.h[base];
        auto pass = [&](auto &&f) {
            for (size_t c0 = 4 * threadIdx.x; c0 < cols; c0 += span) {
                float h[NV][4], g[NV][4], w[NV][4];
#pragma unroll
                for (int i = 0; i < NV; ++i) load4(a.h + base, c0 + 256 * W * i, cols, h[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i) load4(a.go + base, c0 + 256 * W * i, cols, g[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i) load4(a.weight, c0 + 256 * W * i, cols, w[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i) f(c0 + 256 * W * i, h[i], g[i], w[i]);
            }
        };
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        pass([&](size_t c, float (&h)[4], const float (&g)[4], const float (&w)[4]) {
            fill_past(h, c, cols, first);
            back_sums(h, g, w, first, s);
        });
        row_sums<W, 4>(s, lds + turn * 4 * W);
        turn ^= 1;
        const RowBack back = row_back(s, a.per_col, first, a.eps);
        if constexpr (DP) {
            if (threadIdx.x == 0) {
                a.norms[row] = back.norm;
                a.means[row] = make_float2(back.mean_g, back.mean_gu);
            }
        } else {
            pass([&](size_t c, const float (&h)[4], const float (&g)[4], const float (&w)[4]) {
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = back.dh(g[e], w[e], back.norm.unit(h[e]));
                if (c < cols) store4(a.dh + base, c, cols, o);
            });
        }
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
        const float2 mean = a.means[row];
        const RowBack back = {a.norms[row], mean.x, mean.y};
        const size_t base = row * a.cols;
        float h[4], g[4], u[4];
        load4(a.h + base, c, a.cols, h);
        load4(a.go + base, c, a.cols, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u[e] = back.norm.unit(h[e]);
            s[e] += static_cast<double>(g[e]) * u[e];
            sb[e] += g[e];
        }
        if (DH) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = back.dh(g[e], w[e], u[e]);
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

template <bool LONG, int W, int NV, bool RES, bool PACK>
void launch_layer_norm(const LayerNormArgs &a, hipStream_t s) {
    // a row each; of 16 waves as many workgroups as run at once, which keep the weights.  us, a
    // row each and as many as run at once: 8192 x 4096 89, 96, packed 82, 86; 4096 x 8192 98,
    // 97; 2048 x 16384 113, 100
    const size_t need = (a.rows + kLayerRows<W> - 1) / kLayerRows<W>, cap = W == 16 ? device_cu_count() : kMaxBlocks;
    const dim3 grid(static_cast<unsigned>(need < cap ? need : cap)), block(kNormThreads<W>);
    if constexpr (LONG) launch((long_layer_norm<RES, PACK>), grid, block, 0, s, a);
    else launch((layer_norm_rows<W, NV, RES, PACK>), grid, block, 0, s, a);
}
template <int W, int NV, bool LONG>
void launch_layer_norm(const LayerNormArgs &a, hipStream_t s) {
    if (a.residual && a.codes) launch_layer_norm<LONG, W, NV, true, true>(a, s);
    else if (a.residual) launch_layer_norm<LONG, W, NV, true, false>(a, s);
    else if (a.codes) launch_layer_norm<LONG, W, NV, false, true>(a, s);
    else launch_layer_norm<LONG, W, NV, false, false>(a, s);
}

template <int W, int NV, bool LONG>
void launch_layer_back(const LayerNormBackArgs &a, unsigned grid, hipStream_t s) {
    const dim3 block(kNormThreads<W>);
    const bool parts = a.dw_part || a.db_part;
    if constexpr (LONG) {
        if (parts) launch(long_layer_rows<true>, dim3(grid), block, 0, s, a);
        else launch(long_layer_rows<false>, dim3(grid), block, 0, s, a);
    } else {
        if (a.dh && parts) launch((layer_norm_back<W, NV, true, true>), dim3(grid), block, 0, s, a);
        else if (a.dh) launch((layer_norm_back<W, NV, true, false>), dim3(grid), block, 0, s, a);
        else launch((layer_norm_back<W, NV, false, true>), dim3(grid), block, 0, s, a);
    }
}

// for_cols, with half a wave for rows of 128 at most
template <class F>
void for_layer_cols(size_t n, F &&f) {
    using std::integral_constant;
    if (n <= 128) f(integral_constant<int, 0>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
    else for_cols<false>(n, false, f);
}
// The backward pass's: for rows of 1025 to 2048 two waves of four quads in place of four of
// two, since what a wave does for its row beside its quads is as much as a quad and a
// half.  us: 13000 x 1100 41, 58; 7000 x 2048 32, 33.  For longer ones than 8192 eight waves
// of eight quads in place of 16 of four, with twice the registers: 2048 x 16384 105, 124; 1200
// x 12000 51, 56; 1700 x 8200 53, 53.
template <class F>
void for_back_cols(size_t n, F &&f) {
    using std::integral_constant;
    if (n > 1024 && n <= 2048) f(integral_constant<int, 2>{}, integral_constant<int, 4>{}, integral_constant<bool, false>{});
    else if (n > 8192 && n <= kMaxHeldCols) f(integral_constant<int, 8>{}, integral_constant<int, 8>{}, integral_constant<bool, false>{});
    else for_layer_cols(n, [&](auto w, auto nv, auto lng) {
        if constexpr (!(w.value == 4 && nv.value == 2) && !(w.value == 16 && nv.value == 4 && !lng.value)) f(w, nv, lng);
    });
}
size_t layer_back_blocks(size_t rows, size_t cols) {  // (twice back_blocks's rows a workgroup there)
    return cols <= 128 || (cols > 1024 && cols <= 2048) ? back_blocks((rows + 1) / 2, cols) : back_blocks(rows, cols);
}

int layer_norm_forward(const float *x, const float *residual, const float *weight, const float *bias, size_t rows, size_t cols,
                       float eps, float *h, float *y, uint8_t *codes, float *scales, void *stream) {
    if (rows == 0 || cols == 0) return TS_HIP_OK;
    if (!x || !weight || (residual != nullptr) != (h != nullptr) || rows >= kMaxRows) return TS_HIP_EINVAL;
    const LayerNormArgs a = {x, residual, weight, bias, h, y, codes, scales, rows, cols, packed_pitch(cols), eps, 1.0 / static_cast<double>(cols)};
    for_layer_cols(codes ? a.pitch : cols, [&](auto w, auto nv, auto long_rows) {
        launch_layer_norm<w.value, nv.value, long_rows.value>(a, as_stream(stream));
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
    return 2 * layer_back_blocks(rows, cols) * cols + (cols > kMaxHeldCols ? kRowFloats * rows : 0);
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
    const unsigned grid = static_cast<unsigned>(layer_back_blocks(rows, cols));
    const bool long_rows = cols > kMaxHeldCols;
    if (!parts || long_rows || grid > kTicketParts || grid * cols > kTicketFloats) ticket = nullptr;
    // workspace: a long row's means and norms, then the parts
    float2 *const means = reinterpret_cast<float2 *>(workspace);
    RowNorm *const norms = reinterpret_cast<RowNorm *>(workspace + 2 * rows);
    float *const sums = parts ? workspace + (long_rows ? kRowFloats * rows : 0) : nullptr;
    const LayerNormBackArgs a = {h, weight, go, dh, dweight ? sums : nullptr, dbias ? sums + grid * cols : nullptr,
                                 norms, means, rows, cols, eps, 1.0 / static_cast<double>(cols), dweight, dbias, ticket};
    const hipStream_t s = as_stream(stream);
    for_back_cols(cols, [&](auto w, auto nv, auto lng) { launch_layer_back<w.value, nv.value, lng.value>(a, grid, s); });
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
