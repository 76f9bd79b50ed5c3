// A layer's large products on the bf16 matrix cores (the kernel; the passes that
// lay its operands out and the launches: ts_hip_linear_planes.hip).
//
// Planes.  An operand is first rewritten into what the instruction reads: its
// values as bf16 pieces (P = 3: the exact pieces h, m, l of ts_hip_gemm_split.h,
// times 2^16; P = 1: values of 8 bits, which are bf16 numbers as they are), in
// fragments of 32 rows and 16 k:
//   planes [row blocks][k blocks][P] x 1024 bytes, a fragment 64 lanes x 16 bytes,
//   lane 32 h + i holding k 8 h .. 8 h + 7 of row i,
// padded with zeros to whole row blocks and to an even number of k blocks.  The
// product's loop is then nothing but 16-byte DMA from memory to LDS, fragment
// reads in lane order (no bank conflict, no address but the lane's) and matrix
// instructions: no edge, no transpose, no splitting, whatever the layout of the
// operands was.  The rewriting costs a pass over each operand (10 % of a product
// of 8192 x 4096 x 4096).
//
// Products.  With pieces on both sides the six of ts_hip_gemm_split.h, summed from
// zero per 16 k and joined by the vector units, every second k block of A
// negated; with pieces on one side their three products and with none the one,
// summed in the accumulators.
//
// Finite.  A sum that is not finite comes from an operand that is not, a value past
// 2^111 or a sum past 2^95; its tile is marked and computed again on the fp32
// instructions by a launch that otherwise finds nothing to do.
#pragma once

#include "ts_hip_gemm_split.h"
#include "ts_hip_linear.h"

namespace tship {

constexpr int kPlaneRows = 32, kPlaneK = 16, kFragBytes = 1024;

struct PlanesArgs {
    const char *A, *B;  // planes
    float *C;
    LinearEpi epi;
    int M, N;
    int kb;              // k blocks (even)
    int rows_a, rows_b;  // row blocks
    int tiles_m, tiles_n;
    int *marks;  // per tile: computed again; null: none is
};

// BM x BN by WM x WN waves; stages of SK k blocks, NST of them in LDS.
template <int BM, int BN, int WM, int WN, int PA, int PB, int SK, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_planes(PlanesArgs g) {
    constexpr int NW = WM * WN, FM = BM / WM / kPlaneRows, FN = BN / WN / kPlaneRows;
    constexpr int NA = BM / kPlaneRows * SK * PA, NB = BN / kPlaneRows * SK * PB;  // fragments of a stage
    constexpr int PER = (NA + NB) / NW;
    static_assert((NA + NB) % NW == 0, "every wave moves as many fragments");
    constexpr int kStage = (NA + NB) * kFragBytes;
    __shared__ __attribute__((aligned(16))) char lds[NST * kStage];

    int tm, tn;
    tile_coords(g.tiles_m, g.tiles_n, blockIdx.x, tm, tn);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // this wave's fragments of a stage: consecutive ones of A's, then of B's
    const char *src[PER];
    unsigned dst[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int f = wave * PER + i;
        const bool a = f < NA;
        const int per_row = a ? SK * PA : SK * PB, n = a ? f : f - NA;
        const int row = min((a ? tm * (BM / kPlaneRows) : tn * (BN / kPlaneRows)) + n / per_row, (a ? g.rows_a : g.rows_b) - 1);
        src[i] = (a ? g.A : g.B) + (static_cast<size_t>(row) * g.kb * (a ? PA : PB) + n % per_row) * kFragBytes;
        dst[i] = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) char *)(lds + f * kFragBytes)));
    }
    const unsigned voff = lane * 16;
    const int stages = g.kb / SK;
    auto dma = [&](int stage, int slot) {
        const size_t at = static_cast<size_t>(min(stage, stages - 1)) * SK * kFragBytes;  // past the end: the last again
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const char *p = src[i] + at * (wave * PER + i < NA ? PA : PB);
            const unsigned to = dst[i] + slot * kStage;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
            asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(p), "s"(to) : "memory", "m0");
#pragma clang diagnostic pop
        }
    };
    auto frag = [&](const char *stage, int n) {
        return *reinterpret_cast<const b8v_t *>(stage + n * kFragBytes + lane * 16);
    };

    floatx16 acc[FM][FN];
#pragma unroll
    for (int x = 0; x < FM; ++x)
#pragma unroll
        for (int c = 0; c < FN; ++c) acc[x][c] = floatx16{};

#pragma unroll
    for (int s = 0; s < NST - 1; ++s) dma(s, s);
    int slot = 0;
    for (int s = 0; s < stages; ++s) {
        // this stage has landed, and every wave is done with the one before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PER *(NST - 2)) : "memory");
        dma(s + NST - 1, slot == 0 ? NST - 1 : slot - 1);
        const char *at = lds + slot * kStage;
#pragma unroll
        for (int k = 0; k < SK; ++k) {
            b8v_t fb[FN][PB];
#pragma unroll
            for (int c = 0; c < FN; ++c)
#pragma unroll
                for (int p = 0; p < PB; ++p) fb[c][p] = frag(at, NA + ((wn * FN + c) * SK + k) * PB + p);
            const float sign = (s * SK + k) & 1 ? -1.0f : 1.0f;
#pragma unroll
            for (int x = 0; x < FM; ++x) {
                b8v_t fa[PA];
#pragma unroll
                for (int p = 0; p < PA; ++p) fa[p] = frag(at, ((wm * FM + x) * SK + k) * PA + p);
#pragma unroll
                for (int c = 0; c < FN; ++c) {
                    auto mm = [&](floatx16 v, int pa, int pb) {
                        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[pa], fb[c][pb], v, 0, 0, 0);
                    };
                    if constexpr (PA == 3) {
                        floatx16 v = {};
                        v = mm(v, 0, 2);
                        v = mm(v, 1, 1);
                        v = mm(v, 2, 0);
                        v = mm(v, 0, 1);
                        v = mm(v, 1, 0);
                        v = mm(v, 0, 0);
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[x][c][r] = __builtin_fmaf(v[r], sign, acc[x][c][r]);
                    } else {
#pragma unroll
                        for (int p = PB - 1; p >= 0; --p) acc[x][c] = mm(acc[x][c], 0, p);
                    }
                }
            }
        }
        slot = slot + 1 == NST ? 0 : slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outstanding at exit

    if (PB == 3 && g.marks) {
        float worst = 0.0f;  // NaN * 0 and inf * 0 stay NaN
#pragma unroll
        for (int x = 0; x < FM; ++x)
#pragma unroll
            for (int c = 0; c < FN; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) worst = __builtin_fmaf(acc[x][c][r], 0.0f, worst);
        if (worst != worst) g.marks[tm * g.tiles_n + tn] = 1;
    }

    // lane (i, h), register r of block (x, c): row 8 (r / 4) + 4 h + r % 4, column i
    const int li = lane & 31, lh = lane >> 5;
    const int i0 = tm * BM + wm * FM * kPlaneRows, j0 = tn * BN + wn * FN * kPlaneRows;
    constexpr int kScale = (PA == 3 ? 16 : 0) + (PB == 3 ? 16 : 0);
    const float *extra = g.epi.go ? g.epi.go : g.epi.residual;
    const bool inside = i0 + FM * kPlaneRows <= g.M && j0 + FN * kPlaneRows <= g.N;  // uniform
    auto store = [&](auto edge) {
#pragma unroll
        for (int c = 0; c < FN; ++c) {
            const int j = j0 + c * kPlaneRows + li;
            const int jc = edge ? min(j, g.N - 1) : j;
            const float bias = g.epi.bias ? g.epi.bias[jc] : 0.0f;
#pragma unroll
            for (int x = 0; x < FM; ++x) {
                float ev[16];
                auto row_of = [&](int r) { return i0 + x * kPlaneRows + 8 * (r >> 2) + 4 * lh + (r & 3); };
                if (extra) {  // all of a block's before the first is used
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = edge ? min(row_of(r), g.M - 1) : row_of(r);
                        ev[r] = extra[static_cast<size_t>(i) * g.N + jc];
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = row_of(r);
                    if (edge && (i >= g.M || j >= g.N)) continue;
                    const size_t to = static_cast<size_t>(i) * g.N + j;
                    float v = kScale ? __builtin_ldexpf(acc[x][c][r], -kScale) : acc[x][c][r];
                    if (g.epi.bias) v += bias;
                    if (g.epi.z) g.epi.z[to] = v;
                    if (g.epi.go) {
                        v = ev[r] * act_slope(v, g.epi.act);
                    } else {
                        v = activate(v, g.epi.act);
                        if (extra) v += ev[r];
                    }
                    g.C[to] = v;
                }
            }
        }
    };
    if (inside) store(std::false_type{});
    else store(std::true_type{});
}

}  // namespace tship
