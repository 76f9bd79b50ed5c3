// A layer's forward and backward (ts_hip.h, ts_hip_linear and the entries after
// it) and the launches of its small products.
#include <algorithm>

#include "ts_hip_linear_direct.h"

namespace tship {

namespace {

// Work beside a product in its launch: the packing of x (forward)...
struct PackJob {
    const float *x;
    uint8_t *codes, *scales;
    size_t rows, cols, pitch;
    int blocks;
};
// ... or dz's column sums (backward): f64, a workgroup per 16 columns and slice of rows
struct SumJob {
    const float *x, *times;
    float *out, *part;  // part: several slices, [slices][cols]
    int rows, cols, slices, slice_rows, blocks;
};

__device__ __forceinline__ void pack_job(const PackJob &j, int block) {
    const size_t quads = j.pitch / 4, total = j.rows * quads, stride = static_cast<size_t>(j.blocks) * blockDim.x;
    for (size_t q = static_cast<size_t>(block) * blockDim.x + threadIdx.x; q < total; q += stride) {
        const size_t row = q / quads, c = 4 * (q % quads);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < j.cols ? j.x[row * j.cols + c + e] : 0.0f;
        pack_store(v, c, j.codes + row * j.pitch, j.scales + 4 * row, 4 * j.rows);
    }
}

__device__ __forceinline__ void sum_job(const SumJob &j, int block, double *lds) {
    const int lanes = blockDim.x / 16;  // rows side by side
    const int slice = block % j.slices, c = threadIdx.x & 15, q = threadIdx.x >> 4, col = block / j.slices * 16 + c;
    const int from = slice * j.slice_rows, to = min(from + j.slice_rows, j.rows);
    double s = 0.0;
    if (col < j.cols) {
#pragma unroll 8
        for (int r = from + q; r < to; r += lanes) {
            const size_t at = static_cast<size_t>(r) * j.cols + col;
            s += j.times ? through_slope(j.x[at], j.times[at]) : j.x[at];
        }
    }
    lds[q * 16 + c] = s;
    __syncthreads();
    if (q == 0 && col < j.cols) {
#pragma unroll 4
        for (int k = 1; k < lanes; ++k) s += lds[k * 16 + c];
        (j.slices > 1 ? j.part + static_cast<size_t>(slice) * j.cols : j.out)[col] = static_cast<float>(s);
    }
}

template <Src SA, Src SB>
__global__ __launch_bounds__(kDirectThreads) void linear_direct(DirectProduct p, PackJob pack) {
    extern __shared__ __attribute__((aligned(16))) float direct_lds[];
    auto lds = reinterpret_cast<float(*)[kDirectTile * kDirectTile]>(direct_lds);
    const int waves = blockDim.x / 64;
    const int b = blockIdx.x;
    if (b < p.blocks) direct_block<SA, SB>(p, b, waves, lds);  // uniform
    else pack_job(pack, b - p.blocks);
}

// dx = dz W^T, dweight = X^T dz and dz's column sums as one launch: none reads another's.
template <Src SX>
__global__ __launch_bounds__(kDirectThreads) void linear_direct_back(DirectProduct dx, DirectProduct dw, SumJob sum) {
    extern __shared__ __attribute__((aligned(16))) float direct_lds[];
    auto lds = reinterpret_cast<float(*)[kDirectTile * kDirectTile]>(direct_lds);
    const int waves = blockDim.x / 64;
    const int b = blockIdx.x;
    if (b < dw.blocks) direct_block<SX, Src::kFloatR>(dw, b, waves, lds);  // uniform
    else if (b < dw.blocks + dx.blocks) direct_block<Src::kFloatK, Src::kFloatK>(dx, b - dw.blocks, waves, lds);
    else sum_job(sum, b - dw.blocks - dx.blocks, reinterpret_cast<double *>(direct_lds));
}

// The slices' sums added in their order, with the products' epilogues; dz's column sums in f64, as each slice took its own.
__global__ __launch_bounds__(kBlock) void linear_join(DirectProduct p, DirectProduct q, SumJob sum) {
    const size_t np = p.slices > 1 ? static_cast<size_t>(p.M) * p.N : 0;
    const size_t nq = q.slices > 1 ? static_cast<size_t>(q.M) * q.N : 0;
    const size_t all = np + nq + (sum.slices > 1 ? sum.cols : 0), stride = static_cast<size_t>(gridDim.x) * kBlock;
    for (size_t n = static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x; n < all; n += stride) {
        auto total = [&](const float *part, size_t at, size_t size, int slices) {
            float v = part[at];
#pragma unroll 4
            for (int s = 1; s < slices; ++s) v += part[s * size + at];
            return v;
        };
        if (n < np) epilogue_store(p.epi, p.C, n, total(p.part, n, np, p.slices), p.epi.bias ? p.epi.bias[n % p.N] : 0.0f);
        else if (n < np + nq)
            epilogue_store(q.epi, q.C, n - np, total(q.part, n - np, nq, q.slices),
                           q.epi.bias ? q.epi.bias[(n - np) % q.N] : 0.0f);
        else {
            const size_t at = n - np - nq;
            double v = 0.0;
#pragma unroll 4
            for (int s = 0; s < sum.slices; ++s) v += sum.part[s * static_cast<size_t>(sum.cols) + at];
            sum.out[at] = static_cast<float>(v);
        }
    }
}

// How a product's tiles share the chip: up to eight waves a tile while there are
// fewer than four a SIMD and each has two steps of its own (one round of loads);
// then slices of eight steps a wave, up to as many.
struct DirectPlan {
    int kg, slices, slice_steps;
};
DirectPlan direct_plan(size_t M, size_t N, size_t K) {
    const size_t tiles = ((M + kDirectTile - 1) / kDirectTile) * ((N + kDirectTile - 1) / kDirectTile);
    const size_t waves = static_cast<size_t>(device_cu_count()) * 16, steps = (K + kDirectK - 1) / kDirectK;
    DirectPlan p = {1, 1, static_cast<int>(steps)};
    if (tiles == 0) return p;  // (no rows or no columns: asked for its workspace all the same)
    while (p.kg < kDirectWaves && tiles * p.kg * 2 <= waves && steps >= static_cast<size_t>(p.kg) * 2 * 2) p.kg *= 2;
    if (p.kg == kDirectWaves && steps > 16 * kDirectWaves) {
        const size_t want = steps / (8 * kDirectWaves), room = waves / (tiles * kDirectWaves);
        const size_t n = want < room ? want : room;
        if (n > 1) {
            p.slice_steps = static_cast<int>((steps + n - 1) / n);
            p.slices = static_cast<int>((steps + p.slice_steps - 1) / p.slice_steps);
        }
    }
    return p;
}
size_t round64(size_t n) { return (n + 63) / 64 * 64; }
size_t direct_floats(size_t M, size_t N, size_t K) {
    const int slices = direct_plan(M, N, K).slices;
    return slices > 1 ? round64(slices * M * N) : 0;
}

// p with its plan, its parts at `part`.  Its workgroups follow from the launch's
// waves (direct_blocks).
DirectProduct planned(const LinearProduct &p, float *part) {
    DirectProduct d = direct_product(p);
    const DirectPlan plan = direct_plan(p.M, p.N, p.K);
    d.kg = plan.kg;
    d.slices = plan.slices;
    d.slice_steps = plan.slice_steps;
    d.part = part;
    return d;
}
void direct_blocks(DirectProduct &d, int waves) {
    const int per = waves / d.kg;
    d.blocks = (d.tiles * d.slices + per - 1) / per;
}

void join(const DirectProduct &p, const DirectProduct &q, const SumJob &sum, hipStream_t s) {
    const size_t n = (p.slices > 1 ? static_cast<size_t>(p.M) * p.N : 0) + (q.slices > 1 ? static_cast<size_t>(q.M) * q.N : 0) +
                     (sum.slices > 1 ? sum.cols : 0);
    if (n) launch(linear_join, dim3(grid_for(n)), dim3(kBlock), 0, s, p, q, sum);
}

// One product by itself (with x packed beside it).
template <Src SA>
void run_direct(const LinearProduct &p, PackJob pack, float *part, hipStream_t s) {
    DirectProduct d = planned(p, part);
    direct_blocks(d, d.kg);
    launch((linear_direct<SA, Src::kFloatR>), dim3(d.blocks + pack.blocks), dim3(64 * d.kg), d.kg * kDirectLds, s, d, pack);
    join(d, DirectProduct{}, SumJob{}, s);
}

PackJob pack_work(const float *x, uint8_t *codes, uint8_t *scales, size_t rows, size_t cols) {
    PackJob j = {x, codes, scales, rows, cols, packed_pitch(cols), 0};
    if (codes) {
        const size_t need = (rows * j.pitch / 4 + kBlock - 1) / kBlock;
        const size_t cap = static_cast<size_t>(device_cu_count()) * 4;
        j.blocks = static_cast<int>(need < cap ? need : cap);
    }
    return j;
}

// dz's column sums: slices of 512 rows past 1024
SumJob sum_work(const float *x, const float *times, float *out, size_t rows, size_t cols, float *part) {
    SumJob j = {x, times, out, part, static_cast<int>(rows), static_cast<int>(cols), 1, static_cast<int>(rows), 0};
    if (rows > 1024) {
        j.slice_rows = 512;
        j.slices = static_cast<int>((rows + 511) / 512);
    }
    j.blocks = static_cast<int>((cols + 15) / 16) * j.slices;
    return j;
}
size_t sum_floats(size_t rows, size_t cols) { return rows > 1024 ? round64((rows + 511) / 512 * cols) : 0; }

Operand floats(const float *p, size_t ld, size_t rows, const float *times = nullptr) {
    return {p, times, nullptr, nullptr, static_cast<int>(ld), static_cast<int>(rows), 0, 0};
}
Operand packed(const uint8_t *codes, const uint8_t *scales, size_t code_rows, size_t cols, size_t rows) {
    return {nullptr, nullptr, codes, scales, 0, static_cast<int>(rows), packed_pitch(cols), code_rows};
}

// x W (of floats, or the codes of x)
LinearProduct forward_product(const ts_hip_linear_shape &s, const float *x, const uint8_t *codes, const uint8_t *scales,
                              const float *w, float *C, const LinearEpi &e) {
    LinearProduct p;
    p.A = codes ? packed(codes, scales, s.batch, s.fan_in, s.batch) : floats(x, s.fan_in, s.batch);
    p.a = codes ? Src::kCodesK : Src::kFloatK;
    p.B = floats(w, s.fan_out, s.fan_out);
    p.b = Src::kFloatR;
    p.M = static_cast<int>(s.batch);
    p.N = static_cast<int>(s.fan_out);
    p.K = static_cast<int>(s.fan_in);
    p.C = C;
    p.epi = e;
    return p;
}
LinearProduct dx_product(const ts_hip_linear_shape &s, const float *dz, const float *slope, const float *w, float *dx) {
    LinearProduct p{};
    p.A = floats(dz, s.fan_out, s.batch, slope);
    p.a = Src::kFloatK;
    p.B = floats(w, s.fan_out, s.fan_in);
    p.b = Src::kFloatK;
    p.M = static_cast<int>(s.batch);
    p.N = static_cast<int>(s.fan_in);
    p.K = static_cast<int>(s.fan_out);
    p.C = dx;
    return p;
}
LinearProduct dw_product(const ts_hip_linear_shape &s, const float *x, const uint8_t *codes, const uint8_t *scales,
                         const float *dz, const float *slope, float *dw) {
    LinearProduct p{};
    p.A = codes ? packed(codes, scales, s.batch, s.fan_in, s.fan_in) : floats(x, s.fan_in, s.fan_in);
    p.a = codes ? Src::kCodesR : Src::kFloatR;
    p.B = floats(dz, s.fan_out, s.fan_out, slope);
    p.b = Src::kFloatR;
    p.M = static_cast<int>(s.fan_in);
    p.N = static_cast<int>(s.fan_out);
    p.K = static_cast<int>(s.batch);
    p.C = dw;
    return p;
}

// A product with a layer's weight goes by planes (true) or directly: floats that
// stream by planes of the other side, where they begin at 16 bytes.
bool weight_planes(LinearProduct &p) {
    if (!streams_take(p.M, p.N, p.K, p.B.ld)) return planes_take(p.M, p.N, p.K);
    p.streams = reinterpret_cast<uintptr_t>(p.B.p) % 16 == 0;
    return p.streams;
}
size_t weight_floats(size_t M, size_t N, size_t K, Src a, Src b, size_t ld) {
    if (streams_take(M, N, K, ld)) return std::max(streams_workspace_floats(M, N, K, a), direct_floats(M, N, K));
    return planes_take(M, N, K) ? planes_workspace_floats(M, N, K, a, b) : direct_floats(M, N, K);
}

// The backward pass's workspace, in floats: dz, the parts of its column sums, then
// each product's planes or slices: the layer's computed again, dx's, dweight's.
struct BackLayout {
    size_t sums, again, dx, dw, total;
};
BackLayout back_layout(const ts_hip_linear_shape &s) {
    BackLayout l{};
    l.sums = round64(s.batch * s.fan_out);
    l.again = l.sums + (planes_take(s.fan_in, s.fan_out, s.batch) ? round64(planes_sum_floats(s.fan_out, s.batch))
                                                                  : sum_floats(s.batch, s.fan_out));
    l.dx = l.again + round64(weight_floats(s.batch, s.fan_out, s.fan_in, Src::kCodesK, Src::kFloatR, s.fan_out));
    l.dw = l.dx + round64(weight_floats(s.batch, s.fan_in, s.fan_out, Src::kFloatK, Src::kFloatK, s.fan_out));
    l.total = l.dw + (planes_take(s.fan_in, s.fan_out, s.batch)
                          ? round64(planes_workspace_floats(s.fan_in, s.fan_out, s.batch, Src::kFloatR, Src::kFloatR))
                          : direct_floats(s.fan_in, s.fan_out, s.batch));
    return l;
}

// Operands of products in planes, written by one launch.
struct PlaneWrites {
    PlaneTask tasks[kMaxPlaneTasks];
    int count = 0;
    void a(const LinearProduct &p, float *workspace, uint8_t *codes = nullptr, uint8_t *scales = nullptr) {
        tasks[count++] = {&p, false, planes_of_a(p, workspace), codes, scales, nullptr};
    }
    void b(const LinearProduct &p, float *workspace, float *sum_parts = nullptr) {
        tasks[count++] = {&p, true, planes_of_b(p, workspace), nullptr, nullptr, sum_parts};
    }
    void run(hipStream_t s) {
        if (count) planes_write(tasks, count, s);
        count = 0;
    }
};

bool shape_ok(const ts_hip_linear_shape *s) {
    const size_t lim = size_t(1) << 24;  // row and column numbers stay far inside 32 bits
    if (!s || s->batch >= lim || s->fan_in >= lim || s->fan_out >= lim) return false;
    const size_t most = size_t(1) << 34;  // elements of a matrix: a launch has fewer than 2^32 threads
    return s->batch * s->fan_in < most && s->batch * s->fan_out < most && s->fan_in * s->fan_out < most;
}
bool act_ok(int act) { return act >= TS_HIP_ACT_NONE && act <= TS_HIP_ACT_GELU_TANH; }

}  // namespace

void join_slices(const DirectProduct &p, hipStream_t s) { join(p, DirectProduct{}, SumJob{}, s); }

}  // namespace tship

using namespace tship;

extern "C" {

size_t ts_hip_linear_workspace_floats(const ts_hip_linear_shape *shape) {
    if (!shape_ok(shape)) return 0;
    const ts_hip_linear_shape &d = *shape;
    return weight_floats(d.batch, d.fan_out, d.fan_in, Src::kFloatK, Src::kFloatR, d.fan_out);
}

int ts_hip_linear(const ts_hip_linear_shape *shape, const float *x, const float *weight, const float *bias, int act,
                  const float *residual, float *y, float *slope, uint8_t *codes, uint8_t *scales, float *workspace,
                  size_t workspace_floats, void *stream) {
    if (!shape_ok(shape) || !act_ok(act) || (codes != nullptr) != (scales != nullptr)) return TS_HIP_EINVAL;
    if (workspace_floats < ts_hip_linear_workspace_floats(shape)) return TS_HIP_EWORKSPACE;
    const ts_hip_linear_shape &d = *shape;
    if (d.batch == 0) return TS_HIP_OK;
    if (codes && d.fan_in == 0) codes = scales = nullptr;
    if (d.fan_out == 0) return codes ? ts_hip_pack8(x, d.batch, d.fan_in, codes, scales, stream) : TS_HIP_OK;
    if (!y || (d.fan_in && (!x || !weight))) return TS_HIP_EINVAL;
    const hipStream_t s = as_stream(stream);
    LinearProduct p = forward_product(d, x, nullptr, nullptr, weight, y, {bias, residual, nullptr, slope, act});
    if (!workspace && ts_hip_linear_workspace_floats(shape)) return TS_HIP_EINVAL;
    if (weight_planes(p)) {
        PlaneWrites writes;
        writes.a(p, workspace, codes, scales);
        if (!p.streams) writes.b(p, workspace);
        writes.run(s);
        planes_multiply(p, workspace, nullptr, nullptr, s);
        return launch_status();
    }
    run_direct<Src::kFloatK>(p, pack_work(x, codes, scales, d.batch, d.fan_in), workspace, s);
    return launch_status();
}

size_t ts_hip_linear_backward_workspace_floats(const ts_hip_linear_shape *shape) {
    return shape_ok(shape) ? back_layout(*shape).total : 0;
}

int ts_hip_linear_backward(const ts_hip_linear_shape *shape, const float *x, const uint8_t *codes,
                           const uint8_t *scales, const float *weight, const float *bias, int act, const float *slope,
                           const float *go, float *dx, float *dweight, float *dbias, float *workspace,
                           size_t workspace_floats, void *stream) {
    if (!shape_ok(shape) || !act_ok(act) || (codes != nullptr) != (scales != nullptr)) return TS_HIP_EINVAL;
    if (workspace_floats < ts_hip_linear_backward_workspace_floats(shape)) return TS_HIP_EWORKSPACE;
    const ts_hip_linear_shape &d = *shape;
    const hipStream_t s = as_stream(stream);
    int st = TS_HIP_OK;
    // with no batch, or nothing to sum over, the sums are zeros
    if (d.batch == 0 || d.fan_in == 0 || d.fan_out == 0) {
        const bool has_go = d.batch && d.fan_out;
        if (dx && d.batch && d.fan_in) st = ts_hip_fill(dx, 0.0f, d.batch * d.fan_in, stream);
        if (!st && dweight && d.fan_in && d.fan_out) st = ts_hip_fill(dweight, 0.0f, d.fan_in * d.fan_out, stream);
        if (!st && dbias && d.fan_out && !has_go) st = ts_hip_fill(dbias, 0.0f, d.fan_out, stream);
        if (st || !has_go || !dbias) return st;
        dx = dweight = nullptr;
    }
    if (!dx && !dweight && !dbias) return TS_HIP_OK;
    if (!go || !workspace) return TS_HIP_EINVAL;
    const BackLayout at = back_layout(d);
    float *const sums = workspace + at.sums, *const w_again = workspace + at.again, *const w_dx = workspace + at.dx,
                *const w_dw = workspace + at.dw;
    // dz: go times the forward's slopes as the products read them, or go times the
    // slopes of the layer computed again from its checkpoint, stored
    const bool again = act != TS_HIP_ACT_NONE && !slope;
    if (act == TS_HIP_ACT_NONE) slope = nullptr;
    if ((again && (!codes || !weight)) || (dx && !weight) || (dweight && !codes && !x)) return TS_HIP_EINVAL;
    const float *dz = again ? workspace : go;
    LinearProduct pz = forward_product(d, nullptr, codes, scales, weight, workspace, {bias, nullptr, go, nullptr, act});
    LinearProduct px = dx_product(d, dz, slope, weight, dx);
    const LinearProduct pw = dw_product(d, x, codes, scales, dz, slope, dweight);
    const bool planes_x = dx && weight_planes(px), planes_w = dweight && planes_take(pw.M, pw.N, pw.K);
    // what does not wait for dz goes into planes first, with the layer's own operands
    PlaneWrites writes;
    if (planes_x && !px.streams) writes.b(px, w_dx);
    if (planes_w) writes.a(pw, w_dw);
    if (again) {
        if (weight_planes(pz)) {
            writes.a(pz, w_again);
            if (!pz.streams) writes.b(pz, w_again);
            writes.run(s);
            planes_multiply(pz, w_again, nullptr, nullptr, s);
        } else {
            run_direct<Src::kCodesK>(pz, PackJob{}, w_again, s);
        }
    }
    if (planes_x) writes.a(px, w_dx);
    if (planes_w) writes.b(pw, w_dw, dbias ? sums : nullptr);  // dz is passed over for its planes anyway
    writes.run(s);
    if (planes_x) planes_multiply(px, w_dx, nullptr, nullptr, s);
    if (planes_w) planes_multiply(pw, w_dw, sums, dbias, s);
    if (planes_w) dbias = nullptr;
    // the others as one launch
    const bool later_x = dx && !planes_x, later_w = dweight && !planes_w;
    if (!later_x && !later_w && !dbias) return launch_status();
    DirectProduct gx{}, gw{};
    if (later_x) gx = planned(px, w_dx);
    if (later_w) gw = planned(pw, w_dw);
    const SumJob sum = dbias ? sum_work(dz, slope, dbias, d.batch, d.fan_out, sums) : SumJob{};
    int waves = sum.blocks ? 4 : 1;  // (the sums: 16 rows side by side at least)
    if (later_x) waves = gx.kg > waves ? gx.kg : waves;
    if (later_w) waves = gw.kg > waves ? gw.kg : waves;
    if (later_x) direct_blocks(gx, waves);
    if (later_w) direct_blocks(gw, waves);
    const dim3 grid(gx.blocks + gw.blocks + sum.blocks), block(64 * waves);
    const unsigned lds = waves * kDirectLds;
    if (codes) launch((linear_direct_back<Src::kCodesR>), grid, block, lds, s, gx, gw, sum);
    else launch((linear_direct_back<Src::kFloatR>), grid, block, lds, s, gx, gw, sum);
    join(gx, gw, sum, s);
    return launch_status();
}

}  // extern "C"
