// A layer's forward and backward (ts_hip.h, ts_hip_linear and the entries after
// it) and the launches of its small products.
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
// ... or dz's column sums (backward): f64, a workgroup per 16 columns
struct SumJob {
    const float *x;
    float *out;
    int rows, cols, blocks;
};

template <int KG>
__device__ __forceinline__ void pack_job(const PackJob &j, int block) {
    const size_t quads = j.pitch / 4, total = j.rows * quads, stride = static_cast<size_t>(j.blocks) * 64 * KG;
    for (size_t q = static_cast<size_t>(block) * 64 * KG + threadIdx.x; q < total; q += stride) {
        const size_t row = q / quads, c = 4 * (q % quads);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < j.cols ? j.x[row * j.cols + c + e] : 0.0f;
        pack_store(v, c, j.codes + row * j.pitch, j.scales + 4 * row, 4 * j.rows);
    }
}

template <int KG>
__device__ __forceinline__ void sum_job(const SumJob &j, int block, float *lds) {
    constexpr int Q = 4 * KG;  // rows side by side
    double *part = reinterpret_cast<double *>(lds);
    const int c = threadIdx.x & 15, q = threadIdx.x >> 4, col = block * 16 + c;
    double s = 0.0;
    if (col < j.cols) {
#pragma unroll 4
        for (int r = q; r < j.rows; r += Q) s += j.x[static_cast<size_t>(r) * j.cols + col];
    }
    part[q * 16 + c] = s;
    __syncthreads();
    if (q == 0 && col < j.cols) {
#pragma unroll 4
        for (int k = 1; k < Q; ++k) s += part[k * 16 + c];
        j.out[col] = static_cast<float>(s);
    }
}

template <int KG>
constexpr int kDirectLds = KG * kDirectTile * kDirectTile;

template <Src SA, Src SB, int KG>
__global__ __launch_bounds__(64 * KG) void linear_direct(DirectProduct p, PackJob pack) {
    __shared__ float lds[kDirectLds<KG>];
    const int b = blockIdx.x;
    if (b < p.tiles) direct_tile<SA, SB, KG>(p, b, lds);  // uniform
    else pack_job<KG>(pack, b - p.tiles);
}

// dx = dz W^T, dweight = X^T dz and dz's column sums as one launch: none reads another's.
template <Src SX, int KG>
__global__ __launch_bounds__(64 * KG) void linear_direct_back(DirectProduct dx, DirectProduct dw, SumJob sum) {
    __shared__ __attribute__((aligned(8))) float lds[kDirectLds<KG>];
    const int b = blockIdx.x;
    if (b < dw.tiles) direct_tile<SX, Src::kFloatR, KG>(dw, b, lds);  // uniform
    else if (b < dw.tiles + dx.tiles) direct_tile<Src::kFloatK, Src::kFloatK, KG>(dx, b - dw.tiles, lds);
    else sum_job<KG>(sum, b - dw.tiles - dx.tiles, lds);
}

// dz = go act'(z)
__global__ __launch_bounds__(kBlock) void linear_dz(const float *__restrict__ z, const float *__restrict__ go, int act,
                                                    size_t n, float *__restrict__ dz) {
    const size_t stride = static_cast<size_t>(gridDim.x) * kBlock * 4;
    for (size_t i = (static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x) * 4; i < n; i += stride) {
        if (i + 4 <= n) {
            const pk4u_t zq = *reinterpret_cast<const pk4u_t *>(z + i), gq = *reinterpret_cast<const pk4u_t *>(go + i);
            pk4u_t o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = gq[e] * act_slope(zq[e], act);
            *reinterpret_cast<pk4u_t *>(dz + i) = o;
        } else {
            for (size_t k = i; k < n; ++k) dz[k] = go[k] * act_slope(z[k], act);
        }
    }
}

// Waves that share a tile's K: as many as bring the launch to four waves a
// SIMD, while each has two rounds of loads of its own.
int direct_groups(size_t tiles, size_t K) {
    const size_t waves = static_cast<size_t>(device_cu_count()) * 16;
    int kg = 1;
    while (kg < 8 && tiles * kg * 2 <= waves && K >= static_cast<size_t>(kg) * 2 * 64) kg *= 2;
    return kg;
}

template <class F>
void with_groups(int kg, F &&f) {
    using std::integral_constant;
    switch (kg) {
        case 1: return f(integral_constant<int, 1>{});
        case 2: return f(integral_constant<int, 2>{});
        case 4: return f(integral_constant<int, 4>{});
        default: return f(integral_constant<int, 8>{});
    }
}

PackJob pack_work(const float *x, uint8_t *codes, uint8_t *scales, size_t rows, size_t cols, int threads) {
    PackJob j = {x, codes, scales, rows, cols, packed_pitch(cols), 0};
    if (codes) {
        const size_t need = (rows * j.pitch / 4 + threads - 1) / threads, cap = static_cast<size_t>(device_cu_count()) * 4;
        j.blocks = static_cast<int>(need < cap ? need : cap);
    }
    return j;
}

Operand floats(const float *p, size_t ld, size_t rows) {
    return {p, nullptr, nullptr, static_cast<int>(ld), static_cast<int>(rows), 0, 0};
}
Operand packed(const uint8_t *codes, const uint8_t *scales, size_t code_rows, size_t cols, size_t rows) {
    return {nullptr, codes, scales, 0, static_cast<int>(rows), packed_pitch(cols), code_rows};
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
LinearProduct dx_product(const ts_hip_linear_shape &s, const float *dz, const float *w, float *dx) {
    LinearProduct p{};
    p.A = floats(dz, s.fan_out, s.batch);
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
                         const float *dz, float *dw) {
    LinearProduct p{};
    p.A = codes ? packed(codes, scales, s.batch, s.fan_in, s.fan_in) : floats(x, s.fan_in, s.fan_in);
    p.a = codes ? Src::kCodesR : Src::kFloatR;
    p.B = floats(dz, s.fan_out, s.fan_out);
    p.b = Src::kFloatR;
    p.M = static_cast<int>(s.fan_in);
    p.N = static_cast<int>(s.fan_out);
    p.K = static_cast<int>(s.batch);
    p.C = dw;
    return p;
}

// The backward pass's workspace, in floats: dz, the parts of its column sums and
// the planes of one product after another.
struct BackLayout {
    size_t parts, planes, total;
};
BackLayout back_layout(const ts_hip_linear_shape &s) {
    BackLayout l{};
    auto round = [](size_t n) { return (n + 63) / 64 * 64; };
    l.parts = round(s.batch * s.fan_out);
    l.planes = l.parts;
    size_t most = 0;
    auto product = [&](size_t M, size_t N, size_t K, Src a, Src b) {
        if (!planes_take(M, N, K)) return;
        const size_t n = planes_workspace_floats(M, N, K, a, b);
        most = n > most ? n : most;
    };
    product(s.batch, s.fan_out, s.fan_in, Src::kCodesK, Src::kFloatR);
    product(s.batch, s.fan_in, s.fan_out, Src::kFloatK, Src::kFloatK);
    product(s.fan_in, s.fan_out, s.batch, Src::kFloatR, Src::kFloatR);
    if (planes_take(s.fan_in, s.fan_out, s.batch)) l.planes += round(planes_sum_floats(s.fan_out, s.batch));
    l.total = l.planes + most;
    return l;
}

bool shape_ok(const ts_hip_linear_shape *s) {
    const size_t lim = size_t(1) << 24;  // row and column numbers stay far inside 32 bits
    if (!s || s->batch >= lim || s->fan_in >= lim || s->fan_out >= lim) return false;
    const size_t most = size_t(1) << 40;  // elements of a matrix: tile numbers inside 32 bits
    return s->batch * s->fan_in < most && s->batch * s->fan_out < most && s->fan_in * s->fan_out < most;
}
bool act_ok(int act) { return act >= TS_HIP_ACT_NONE && act <= TS_HIP_ACT_GELU_TANH; }

}  // namespace

}  // namespace tship

using namespace tship;

extern "C" {

size_t ts_hip_linear_workspace_floats(const ts_hip_linear_shape *shape) {
    if (!shape_ok(shape)) return 0;
    const ts_hip_linear_shape &d = *shape;
    return planes_take(d.batch, d.fan_out, d.fan_in)
               ? planes_workspace_floats(d.batch, d.fan_out, d.fan_in, Src::kFloatK, Src::kFloatR)
               : 0;
}

int ts_hip_linear(const ts_hip_linear_shape *shape, const float *x, const float *weight, const float *bias, int act,
                  const float *residual, float *y, float *z, uint8_t *codes, uint8_t *scales, float *workspace,
                  size_t workspace_floats, void *stream) {
    if (!shape_ok(shape) || !act_ok(act) || (codes != nullptr) != (scales != nullptr)) return TS_HIP_EINVAL;
    if (workspace_floats < ts_hip_linear_workspace_floats(shape)) return TS_HIP_EWORKSPACE;
    const ts_hip_linear_shape &d = *shape;
    if (d.batch == 0) return TS_HIP_OK;
    if (codes && d.fan_in == 0) codes = scales = nullptr;
    if (d.fan_out == 0) return codes ? ts_hip_pack8(x, d.batch, d.fan_in, codes, scales, stream) : TS_HIP_OK;
    if (!y || (d.fan_in && (!x || !weight))) return TS_HIP_EINVAL;
    const hipStream_t s = as_stream(stream);
    const LinearProduct p = forward_product(d, x, nullptr, nullptr, weight, y, {bias, residual, nullptr, z, act});
    if (planes_take(d.batch, d.fan_out, d.fan_in)) {
        if (!workspace) return TS_HIP_EINVAL;
        PlanesExtra extra;
        extra.codes = codes;
        extra.scales = scales;
        return planes_product(p, extra, workspace, s);
    }
    const DirectProduct g = direct_product(p);
    with_groups(direct_groups(g.tiles, p.K), [&](auto kg) {
        const PackJob pack = pack_work(x, codes, scales, d.batch, d.fan_in, 64 * kg.value);
        launch((linear_direct<Src::kFloatK, Src::kFloatR, kg.value>), dim3(g.tiles + pack.blocks), dim3(64 * kg.value), 0,
               s, g, pack);
    });
    return launch_status();
}

size_t ts_hip_linear_backward_workspace_floats(const ts_hip_linear_shape *shape) {
    return shape_ok(shape) ? back_layout(*shape).total : 0;
}

int ts_hip_linear_backward(const ts_hip_linear_shape *shape, const float *x, const uint8_t *codes,
                           const uint8_t *scales, const float *weight, const float *bias, int act, const float *z,
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
    float *const planes = workspace + at.planes;
    const float *dz = go;
    if (act != TS_HIP_ACT_NONE) {
        if (z || d.fan_in == 0) {
            if (!z) return TS_HIP_EINVAL;
            const size_t n = d.batch * d.fan_out;
            launch(linear_dz, dim3(grid_for(n, 4)), dim3(kBlock), 0, s, z, go, act, n, workspace);
        } else {
            if (!codes || !weight) return TS_HIP_EINVAL;
            const LinearProduct p =
                forward_product(d, nullptr, codes, scales, weight, workspace, {bias, nullptr, go, nullptr, act});
            if (planes_take(d.batch, d.fan_out, d.fan_in)) {
                st = planes_product(p, {}, planes, s);
                if (st) return st;
            } else {
                const DirectProduct g = direct_product(p);
                with_groups(direct_groups(g.tiles, p.K), [&](auto kg) {
                    launch((linear_direct<Src::kCodesK, Src::kFloatR, kg.value>), dim3(g.tiles), dim3(64 * kg.value), 0, s,
                           g, PackJob{});
                });
            }
        }
        dz = workspace;
    }
    if ((dx && !weight) || (dweight && !codes && !x)) return TS_HIP_EINVAL;
    DirectProduct gx{}, gw{};
    if (dx) {
        const LinearProduct p = dx_product(d, dz, weight, dx);
        if (planes_take(p.M, p.N, p.K)) st = planes_product(p, {}, planes, s);
        else gx = direct_product(p);
    }
    if (dweight && !st) {
        const LinearProduct p = dw_product(d, x, codes, scales, dz, dweight);
        if (planes_take(p.M, p.N, p.K)) {
            PlanesExtra extra;
            extra.sums = dbias;  // dz is passed over for its planes anyway
            extra.sum_parts = workspace + at.parts;
            st = planes_product(p, extra, planes, s);
            dbias = nullptr;
        } else {
            gw = direct_product(p);
        }
    }
    if (st || (!gx.tiles && !gw.tiles && !dbias)) return st ? st : launch_status();
    SumJob sum = {dz, dbias, static_cast<int>(d.batch), static_cast<int>(d.fan_out),
                  dbias ? static_cast<int>((d.fan_out + 15) / 16) : 0};
    const size_t K = gw.tiles ? d.batch : d.fan_out;
    with_groups(direct_groups(static_cast<size_t>(gx.tiles) + gw.tiles, K), [&](auto kg) {
        const dim3 grid(gx.tiles + gw.tiles + sum.blocks), block(64 * kg.value);
        if (codes) launch((linear_direct_back<Src::kCodesR, kg.value>), grid, block, 0, s, gx, gw, sum);
        else launch((linear_direct_back<Src::kFloatR, kg.value>), grid, block, 0, s, gx, gw, sum);
    });
    return launch_status();
}

}  // extern "C"
