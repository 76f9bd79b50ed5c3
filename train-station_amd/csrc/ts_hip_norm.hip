// Root-mean-square norm with the residual's addition (ts_hip.h, ts_hip_rms_norm
// and the entries after it), its packed form, its backward, and the packing of
// plain rows.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   g = go w:  dh = r g - h r^3 mean(g h),  dw = sum over rows of go h r
//
// A row is held in registers by W waves, four neighbouring columns a lane and
// NV such quads, so memory is passed over once; sums are f64.  Backward needs
// h^2's and g h's row sums only, and takes both in the same pass: nothing but h
// is kept from the forward.  r is held as a power of two and a factor near one
// (row_scale): with u the power and f the factor, dh = u (f g - (u h) b) and
// b = f^2 r mean(g h), whose parts are of g's size however long a row is, where
// r and r^3 mean(g h) themselves leave fp32 long before dh does.
//
// Bound by memory from a few thousand rows on, below by the launch and by what a
// row's waves wait for in turn: loads, sums, stores (3000 x 1003 packed 8.6 us for 15 MB).
// us, 8192 x 4096 with the sum: forward 85 for 537 MB, packed 87 for 437 MB, backward 85
// for 403 MB (h partly from the last-level cache); 16384 x 2048 the same; 1 x 4096 packed 5.
// The f64 sums and the packed form's f64 products are under that: a wave has four
// loads of 16 bytes in flight per operand, and four waves a row leave two rows a SIMD.
#include "ts_hip_pack8.h"
#include "ts_hip_parts.h"

namespace tship {

namespace {

constexpr size_t kMaxHeldCols = 16384;  // 16 waves of 64 lanes of four quads

__device__ __forceinline__ void load4(const float *p, size_t c, size_t cols, float (&v)[4]) {
    if (c + 4 <= cols) {
        const pk4u_t q = *reinterpret_cast<const pk4u_t *>(p + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? p[c + e] : 0.0f;
    }
}

__device__ __forceinline__ void store4(float *p, size_t c, size_t cols, const float (&v)[4]) {
    if (c + 4 <= cols) {
        *reinterpret_cast<pk4u_t *>(p + c) = pk4u_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) p[c + e] = v[e];
    }
}

// The sum over the W waves of a row, in every lane; lds: N * W doubles of this row.
template <int W, int N>
__device__ __forceinline__ void row_sum(double (&s)[N], double *lds) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = wave_sum(s[n]);
    if (W == 1) return;
    const int wave = (threadIdx.x >> 6) % W;
    __syncthreads();  // the last row's reads
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

// r = up * f with up a power of two (as fp32 has them) and f in [1, 2) where r is
// one of fp32's range, within a few binades of it for what rows can give beyond.
struct RowScale {
    float up;
    double f;
};
__device__ __forceinline__ RowScale row_scale(double r) {
    const int e = min(max(static_cast<int>(__double_as_longlong(r) >> 52 & 0x7ff) - 1023, -126), 127);  // (inf, NaN: 127)
    const double down = __longlong_as_double(static_cast<long long>(1023 - e) << 52);
    return {__uint_as_float(static_cast<unsigned>(e + 127) << 23), r * down};
}

template <int W>
constexpr int kNormThreads = W < 4 ? 256 : 64 * W;
template <int W>
constexpr int kNormRows = kNormThreads<W> / (64 * W);  // rows of a workgroup

struct NormArgs {
    const float *x, *residual, *weight;
    float *h, *y;             // h: with a residual
    uint8_t *codes, *scales;  // packed
    size_t rows, cols, pitch;
    double eps;
};

// A row per W waves; LONG: more columns than the waves hold, passed over twice.
template <int W, int NV, bool RES, bool PACK, bool LONG>
__global__ __launch_bounds__(kNormThreads<W>) void rms_norm_rows(NormArgs a) {
    constexpr int RPB = kNormRows<W>;
    __shared__ double lds[RPB * W];
    const int slot = threadIdx.x / (64 * W), t = threadIdx.x % (64 * W);
    const size_t span = static_cast<size_t>(256) * W * NV, end = PACK ? a.pitch : a.cols;
    float w[NV][4];
    auto weights = [&](size_t from) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load4(a.weight, from + 4 * (t + 64 * W * i), a.cols, w[i]);
    };
    if (!LONG) weights(0);
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    for (size_t row = static_cast<size_t>(blockIdx.x) * RPB + slot; row < a.rows; row += step) {  // (W > 1: uniform)
        const size_t base = row * a.cols;
        const float *x = a.x + base, *res = RES ? a.residual + base : nullptr;
        float v[NV][4];
        auto fetch = [&](size_t c0) {  // h of the columns from c0 on (past the row: zeros)
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
        double s[1] = {0.0};
        size_t c0 = 0;
        do {
            fetch(c0);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[0] += static_cast<double>(v[i][e]) * v[i][e];
            c0 += span;
        } while (LONG && c0 < a.cols);
        row_sum<W, 1>(s, lds + slot * W);
        const double r = 1.0 / sqrt(s[0] / static_cast<double>(a.cols) + a.eps);
        const RowScale scale = row_scale(r);
        const float up = scale.up, rf = static_cast<float>(scale.f);
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
                float o[4];
                if (PACK) {  // in f64: a code takes the side of its border that y itself is on
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[e] = c + e < a.cols ? round_odd(static_cast<double>(v[i][e]) * r * w[i][e]) : 0.0f;
                    pack_store(o, c, a.codes + row * a.pitch, a.scales + 4 * row, 4 * a.rows);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = up * v[i][e] * rf * w[i][e];
                    store4(a.y + base, c, a.cols, o);
                }
            }
            c0 += span;
        } while (LONG && c0 < end);
    }
}

struct NormBackArgs {
    const float *h, *weight, *go;
    float *dh, *dw_part;  // dw_part: [gridDim.x][cols]
    float *scales;        // LONG with dw_part: each row's up, f and back
    size_t rows, cols;
    double eps;
    float *dw;         // with a ticket: the last workgroup adds the parts up
    unsigned *ticket;  // zero, and zero again when the launch has run; null: none
};

// Rows blockIdx.x * RPB + slot, and on by the grid's; a thread keeps dw's sums
// of its columns (f64), the workgroup's go to dw_part.  LONG with dw: no thread has
// columns of its own; the rows' scales are left for long_columns.
template <int W, int NV, bool DH, bool DW, bool LONG>
__global__ __launch_bounds__(kNormThreads<W>) void rms_norm_back(NormBackArgs a) {
    constexpr int RPB = kNormRows<W>;
    __shared__ double lds[RPB * 2 * W];
    const int slot = threadIdx.x / (64 * W), t = threadIdx.x % (64 * W);
    const size_t span = static_cast<size_t>(256) * W * NV;
    // The sums stand in registers; where 16 waves of four quads leave none, in shared
    // memory, each thread its own (2048 x 16384 forward and backward: registers, 60 of
    // them spilled, 227 us, shared memory 195; 300 x 12000 47, 34).
    constexpr bool SHARED = DW && !LONG && W * NV >= 64;
    __shared__ double held[SHARED ? NV * 4 * 64 * W : 1];
    double own[SHARED ? 1 : NV][4] = {};
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
    float *part = DW ? a.dw_part + static_cast<size_t>(blockIdx.x) * a.cols : nullptr;
    const size_t step = static_cast<size_t>(gridDim.x) * RPB;
    // every wave of the workgroup takes every round (the barriers)
    for (size_t r0 = static_cast<size_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += step) {
        const size_t row = r0 + slot;
        const bool live = row < a.rows;
        const size_t base = live ? row * a.cols : 0, n = live ? a.cols : 0;
        float h[NV][4], g[NV][4];
        auto fetch = [&](size_t c0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load4(a.h + base, c0 + 4 * (t + 64 * W * i), n, h[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i) load4(a.go + base, c0 + 4 * (t + 64 * W * i), n, g[i]);
        };
        double s[2] = {0.0, 0.0};
        size_t c0 = 0;
        do {
            fetch(c0);
            if (LONG) weights(c0);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double hv = h[i][e];
                    s[0] += hv * hv;
                    s[1] += hv * (static_cast<double>(g[i][e]) * w[i][e]);
                }
            c0 += span;
        } while (LONG && c0 < a.cols);
        row_sum<W, 2>(s, lds + slot * 2 * W);
        const double cols = static_cast<double>(a.cols);
        const double r = 1.0 / sqrt(s[0] / cols + a.eps);
        const RowScale scale = row_scale(r);
        const float up = scale.up, rf = static_cast<float>(scale.f);
        const float back = static_cast<float>(scale.f * scale.f * (r * (s[1] / cols)));
        if (DW && LONG) {
            if (t == 0) {
                a.scales[3 * row] = up;
                a.scales[3 * row + 1] = rf;
                a.scales[3 * row + 2] = back;
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
                if (DH && c < n) {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = up * (rf * (g[i][e] * w[i][e]) - up * h[i][e] * back);
                    store4(a.dh + base, c, a.cols, o);
                }
                if (DW && !LONG && live) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) dw(i, e) += static_cast<double>(g[i][e]) * (up * h[i][e] * rf);
                }
            }
            c0 += span;
        } while (LONG && c0 < a.cols);
    }
    if (DW && !LONG) {
        if constexpr (RPB > 1) {  // the workgroup's rows together, in their order
            __shared__ double sum[(RPB - 1) * 64 * W * NV * 4];
            __syncthreads();
            if (slot > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[((slot - 1) * NV * 4 + i * 4 + e) * 64 * W + t] = dw(i, e);
            }
            __syncthreads();
            if (slot == 0) {
#pragma unroll
                for (int k = 0; k < RPB - 1; ++k)
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) dw(i, e) += sum[(k * NV * 4 + i * 4 + e) * 64 * W + t];
            }
        }
        if (slot == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t c = 4 * (t + 64 * W * i);
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(dw(i, e));
                if (c < a.cols) store4(part, c, a.cols, o);
            }
        }
    }
    if (DW && a.ticket) {  // uniform: the last workgroup to get here adds the parts up
        __shared__ bool last;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        for (size_t c = threadIdx.x; c < a.cols; c += kNormThreads<W>) {
            double s = 0.0;
#pragma unroll 16
            for (size_t g = 0; g < gridDim.x; ++g) s += a.dw_part[g * a.cols + c];
            a.dw[c] = static_cast<float>(s);
        }
        if (threadIdx.x == 0) *a.ticket = 0;
    }
}

// dw, and dh, of rows longer than a workgroup holds, by columns: a thread has four of
// them, of `run` rows (dw: f64).  Rows are read twice either way: the first pass by rows
// takes their sums alone.  Forward and backward, us: 2048 x 20000 277, 512 x 65536 197
// (dh by rows, and dw row by row on a line of each workgroup's in fp32: 293, 242).
constexpr size_t kLongCols = 4 * kBlock;  // of a workgroup
template <bool DH>
__global__ __launch_bounds__(kBlock) void long_columns(NormBackArgs a, size_t run) {
    const size_t c = blockIdx.x * kLongCols + 4 * threadIdx.x, first = blockIdx.y * run;
    if (c >= a.cols) return;
    const size_t last = first + run < a.rows ? first + run : a.rows;
    float w[4];
    if (DH) load4(a.weight, c, a.cols, w);
    double s[4] = {};
#pragma unroll 4
    for (size_t row = first; row < last; ++row) {
        const float up = a.scales[3 * row], rf = a.scales[3 * row + 1], back = a.scales[3 * row + 2];
        const size_t base = row * a.cols;
        float h[4], g[4];
        load4(a.h + base, c, a.cols, h);
        load4(a.go + base, c, a.cols, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += static_cast<double>(g[e]) * (up * h[e] * rf);
        if (DH) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = up * (rf * (g[e] * w[e]) - up * h[e] * back);
            store4(a.dh + base, c, a.cols, o);
        }
    }
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(s[e]);
    store4(a.dw_part + blockIdx.y * a.cols, c, a.cols, o);
}

__global__ __launch_bounds__(kBlock) void sum_parts(PartSums p) {
    __shared__ double lds[kPartSumsLds];
    part_sums_block(p, blockIdx.x, lds);
}

// Rows of plain values to 8 bits: a thread packs a quad, a grid stride over all quads.
__global__ __launch_bounds__(kBlock) void pack_rows(const float *__restrict__ x, size_t rows, size_t cols, size_t pitch,
                                                    uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    const size_t quads = pitch / 4, total = rows * quads;  // a multiple of 32: blocks of eight lanes stay together
    const size_t stride = static_cast<size_t>(gridDim.x) * kBlock;
    for (size_t q = static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x; q < total; q += stride) {
        const size_t row = q / quads, c = 4 * (q % quads);
        float v[4];
        load4(x + row * cols, c, cols, v);
        pack_store(v, c, codes + row * pitch, scales + 4 * row, 4 * rows);
    }
}

__global__ __launch_bounds__(kBlock) void unpack_rows(const uint8_t *__restrict__ codes,
                                                      const uint8_t *__restrict__ scales, size_t rows, size_t cols,
                                                      size_t pitch, float *__restrict__ out) {
    const size_t quads = (cols + 3) / 4, total = rows * quads;
    const size_t stride = static_cast<size_t>(gridDim.x) * kBlock;
    for (size_t q = static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x; q < total; q += stride) {
        const size_t row = q / quads, c = 4 * (q % quads);
        const unsigned code = *reinterpret_cast<const unsigned *>(codes + row * pitch + c);
        const uint8_t k = scales[(c / kPackGroup * rows + row) * 4 + c / kPackBlock % 4];
        float v[4];
        unpack4(code, k, v);
        store4(out + row * cols, c, cols, v);
    }
}

constexpr size_t kMaxBlocks = size_t(1) << 21;  // a launch has fewer than 2^32 threads; more rows take turns

template <int W, int NV, bool LONG>
void launch_norm(const NormArgs &a, bool pack, hipStream_t s) {
    const size_t need = (a.rows + kNormRows<W> - 1) / kNormRows<W>;
    const dim3 grid(static_cast<unsigned>(need < kMaxBlocks ? need : kMaxBlocks)), block(kNormThreads<W>);
    if (a.residual && pack) launch((rms_norm_rows<W, NV, true, true, LONG>), grid, block, 0, s, a);
    else if (a.residual) launch((rms_norm_rows<W, NV, true, false, LONG>), grid, block, 0, s, a);
    else if (pack) launch((rms_norm_rows<W, NV, false, true, LONG>), grid, block, 0, s, a);
    else launch((rms_norm_rows<W, NV, false, false, LONG>), grid, block, 0, s, a);
}

template <int W, int NV, bool LONG>
void launch_back(const NormBackArgs &a, unsigned grid, hipStream_t s) {
    const dim3 block(kNormThreads<W>);
    if (a.dh && a.dw_part) launch((rms_norm_back<W, NV, true, true, LONG>), dim3(grid), block, 0, s, a);
    else if (a.dh) launch((rms_norm_back<W, NV, true, false, LONG>), dim3(grid), block, 0, s, a);
    else launch((rms_norm_back<W, NV, false, true, LONG>), dim3(grid), block, 0, s, a);
}

// Calls f(W, NV, LONG as constants) for a row of n columns: the fewest waves that
// hold it with four quads a lane, but for rows of 4097 to 8192 packed, whose f64
// products want the registers: two quads.  us, packed with the sum, four quads and
// two: 8192 x 4096 87, 92; 4096 x 8192 120, 107.  Forward and backward: 4096 x 8192
// 184, 187; 4096 x 6000 144, 157.  (Eight quads: 2048 x 16384 packed 129, four 109.)
template <class F>
void for_cols(size_t n, bool packed, F &&f) {
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    const integral_constant<int, 8> eight{};
    const integral_constant<int, 16> sixteen{};
    const integral_constant<bool, false> held{};
    if (n <= 256) f(one, one, held);
    else if (n <= 512) f(one, two, held);
    else if (n <= 1024) f(one, four, held);
    else if (n <= 2048) f(four, two, held);
    else if (n <= 4096) f(four, four, held);
    else if (n <= 8192) packed ? f(sixteen, two, held) : f(eight, four, held);
    else if (n <= kMaxHeldCols) f(sixteen, four, held);
    else f(sixteen, four, integral_constant<bool, true>{});
}

size_t rows_per_block(size_t cols) { return cols <= 1024 ? 4 : 1; }

// Workgroups of the backward pass: as many as run at once (2048 threads a CU, at
// most 4 workgroups), so that each sums many rows before it writes dw.
size_t back_blocks(size_t rows, size_t cols) {
    const size_t need = (rows + rows_per_block(cols) - 1) / rows_per_block(cols);
    const size_t cap = static_cast<size_t>(device_cu_count()) * (cols > 4096 ? 1 : 2);
    return need < cap ? need : cap;
}

// Rows of a part of long_columns: as many as leave eight workgroups a CU, in no more parts than back_blocks
size_t long_run(size_t rows, size_t cols) {
    const size_t wide = (cols + kLongCols - 1) / kLongCols, most = back_blocks(rows, cols);
    const size_t want = (static_cast<size_t>(device_cu_count()) * 8 + wide - 1) / wide;
    const size_t parts = want < most ? want : most;
    return (rows + parts - 1) / parts;
}

constexpr size_t kMaxRows = size_t(1) << 31;
// Parts that one workgroup adds up sooner than another launch has started: 128 x 784
// (32 parts) forward and backward 26.8 us by two launches, 24.5 by one; 16384 x 64
// (512 parts) 27.1 by two, 69 by one.
constexpr size_t kTicketParts = 64, kTicketFloats = 32768;

}  // namespace

}  // namespace tship

using namespace tship;

extern "C" {

size_t ts_hip_packed_pitch(size_t cols) { return packed_pitch(cols); }

int ts_hip_pack8(const float *x, size_t rows, size_t cols, uint8_t *codes, uint8_t *scales, void *stream) {
    if (rows == 0 || cols == 0) return TS_HIP_OK;
    if (!x || !codes || !scales) return TS_HIP_EINVAL;
    const size_t pitch = packed_pitch(cols);
    launch(pack_rows, dim3(grid_for(rows * pitch / 4)), dim3(kBlock), 0, as_stream(stream), x, rows, cols, pitch, codes,
           scales);
    return launch_status();
}

int ts_hip_unpack8(const uint8_t *codes, const uint8_t *scales, size_t rows, size_t cols, float *out, void *stream) {
    if (rows == 0 || cols == 0) return TS_HIP_OK;
    if (!codes || !scales || !out) return TS_HIP_EINVAL;
    launch(unpack_rows, dim3(grid_for(rows * ((cols + 3) / 4))), dim3(kBlock), 0, as_stream(stream), codes, scales, rows,
           cols, packed_pitch(cols), out);
    return launch_status();
}

static int norm_forward(const float *x, const float *residual, const float *weight, size_t rows, size_t cols, float eps,
                        float *h, float *y, uint8_t *codes, uint8_t *scales, void *stream) {
    if (rows == 0 || cols == 0) return TS_HIP_OK;
    if (!x || !weight || (residual != nullptr) != (h != nullptr) || rows >= kMaxRows) return TS_HIP_EINVAL;
    const NormArgs a = {x, residual, weight, h, y, codes, scales, rows, cols, packed_pitch(cols), eps};
    for_cols(codes ? a.pitch : cols, codes != nullptr, [&](auto w, auto nv, auto long_rows) {
        launch_norm<w.value, nv.value, long_rows.value>(a, codes != nullptr, as_stream(stream));
    });
    return launch_status();
}

int ts_hip_rms_norm(const float *x, const float *residual, const float *weight, size_t rows, size_t cols, float eps,
                    float *h, float *y, void *stream) {
    if (rows && cols && !y) return TS_HIP_EINVAL;
    return norm_forward(x, residual, weight, rows, cols, eps, h, y, nullptr, nullptr, stream);
}

int ts_hip_rms_norm_packed(const float *x, const float *residual, const float *weight, size_t rows, size_t cols,
                           float eps, float *h, uint8_t *codes, uint8_t *scales, void *stream) {
    if (rows && cols && (!codes || !scales)) return TS_HIP_EINVAL;
    return norm_forward(x, residual, weight, rows, cols, eps, h, nullptr, codes, scales, stream);
}

size_t ts_hip_rms_norm_backward_workspace_floats(size_t rows, size_t cols) {
    return back_blocks(rows, cols) * cols + (cols > kMaxHeldCols ? 3 * rows : 0);
}

int ts_hip_rms_norm_backward(const float *h, const float *weight, const float *go, size_t rows, size_t cols, float eps,
                             float *dh, float *dweight, float *workspace, size_t workspace_floats, unsigned *ticket,
                             void *stream) {
    if (cols == 0 || (!dh && !dweight)) return TS_HIP_OK;
    if (rows == 0) return dweight ? ts_hip_fill(dweight, 0.0f, cols, stream) : TS_HIP_OK;
    if (!h || !weight || !go || rows >= kMaxRows) return TS_HIP_EINVAL;
    if (dweight && (!workspace || workspace_floats < ts_hip_rms_norm_backward_workspace_floats(rows, cols)))
        return TS_HIP_EWORKSPACE;
    const unsigned grid = static_cast<unsigned>(back_blocks(rows, cols));
    const bool long_rows = cols > kMaxHeldCols;
    if (!dweight || long_rows || grid > kTicketParts || grid * cols > kTicketFloats) ticket = nullptr;
    float *const parts = dweight ? workspace : nullptr, *const scales = parts ? parts + grid * cols : nullptr;
    const NormBackArgs a = {h, weight, go, dh, parts, scales, rows, cols, eps, dweight, ticket};
    const hipStream_t s = as_stream(stream);
    for_cols(cols, false, [&](auto w, auto nv, auto lng) { launch_back<w.value, nv.value, lng.value>(a, grid, s); });
    size_t count = grid;
    if (dweight && long_rows) {
        const size_t run = long_run(rows, cols);
        count = (rows + run - 1) / run;
        const dim3 columns(static_cast<unsigned>((cols + kLongCols - 1) / kLongCols), static_cast<unsigned>(count));
        if (dh) launch(long_columns<true>, columns, dim3(kBlock), 0, s, a, run);
        else launch(long_columns<false>, columns, dim3(kBlock), 0, s, a, run);
    }
    if (dweight && !ticket)
        launch(sum_parts, dim3(static_cast<unsigned>((cols + 15) / 16)), dim3(kBlock), 0, s,
               part_sums(parts, count, cols, dweight));
    return launch_status();
}

}  // extern "C"
