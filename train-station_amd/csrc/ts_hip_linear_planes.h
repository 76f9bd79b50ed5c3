// A layer's large products on the bf16 matrix cores (the kernel; the passes that
// lay its operands out and the launches: ts_hip_linear_planes.hip).
//
// Planes.  An operand is first rewritten into what the instruction reads: its
// values as the exact bf16 pieces h, m, l of ts_hip_gemm_split.h, times 2^16 (or,
// where they are 8-bit values, as the one bf16 number they are), in fragments of
// 32 rows and 16 k:
//   planes [row blocks][k blocks][pieces] x 1024 bytes, a fragment 64 lanes x 16
//   bytes, lane 32 h + i holding k 8 h .. 8 h + 7 of row i,
// padded with zeros to whole row blocks and to an even number of k blocks.  The
// product's loop is then nothing but 16-byte DMA from memory to LDS, fragment
// reads in lane order (no bank conflict, no address but the lane's) and matrix
// instructions: no edge, no transpose, no splitting, whatever the layout of the
// operands was.  The rewriting costs a pass over each operand (7 % of a layer of
// 4096 -> 4096 at batch 8192).  8192 x 4096 x 4096: 1242 us (1330 TFLOP/s of
// instructions), matrix cores busy 73 % of a clock that the power limit sets.
//
// Codes along k on both sides need no pass: they go to LDS as they are, half the
// bytes of bf16, and a fragment's eight are widened with their scale as they are
// read, an instruction for two.  8192 x 4096 x 4096: 253 us, against 261 and 38 for
// the passes from planes, whose LDS reads, 128 bytes a clock, are the bound.  Beside
// three pieces on the other side codes are widened by a pass all the same: 598 and
// 27 us, against 766 with the widening between the matrix instructions.
//
// Streams.  Few rows beside a large weight read each of its values once or a few
// times, and planes of it would cost more than the product.  Its floats then go to LDS
// as they lie, a wave has 32 columns of all the tile's rows, and splits its fragments as
// it reads them (a fifth of the time of their products of 128 rows); the waves are in
// two groups that share a stage's k.  128 x 4096 x 4096: 36 us, against 43 to 53 and 32
// for the weight's planes; 64 x 4096 x 4096: 22, 45 directly (67 MB at 4.8 TB/s: 14).
// Bound by the two in turn: without the products 128 rows take 22 us.
//
// Products.  With pieces on both sides the six of ts_hip_gemm_split.h, summed from
// zero per 16 k and joined by the vector units, every second k block of A
// negated; with pieces on one side their three products and with none the one,
// summed in the accumulators.
//
// Finite.  A sum that is not finite comes from an operand that is not, a value past
// 2^111 or a sum past 2^95; its tile is computed again from the operands
// themselves on the fp32 instructions (direct_tile).
#pragma once

#include "ts_hip_gemm_split.h"
#include "ts_hip_linear_direct.h"
#include "ts_hip_parts.h"

namespace tship {

constexpr bool of_codes(Src s) { return s == Src::kCodesK || s == Src::kCodesR; }
constexpr int pieces_of(Src s) { return of_codes(s) ? 1 : 3; }
constexpr bool as_codes(Src a, Src b) { return a == Src::kCodesK && b == Src::kCodesK; }  // read as codes, not from planes

constexpr int kPlaneRows = 32, kPlaneK = 16, kFragBytes = 1024;

struct PlanesArgs {
    const char *A, *B;  // planes
    DirectProduct p;     // the product itself (its tiles: 32 x 32)
    int kb;              // k blocks of the planes (even)
    int rows_a, rows_b;  // row blocks
    int stages;
    int tiles_m, tiles_n;
    int slice_stages;    // p.slices > 1: a workgroup's stages, its sums to p.part
    PartSums sums;       // a weight's gradient: dz's column sums, by workgroups past the tiles'
};

// One side's part of a stage of SK k blocks: R rows.
template <Src S, int R, int SK, bool CODES>
struct PlaneSide {
    static constexpr bool kCodes = CODES;
    static constexpr int P = pieces_of(S), kBlocks = R / kPlaneRows;
    static_assert(!kCodes || SK * kPlaneK == kPackGroup, "codes: a group of 128 a stage");
    // DMA instructions of 1 KB: fragments, or 8 rows of 128 codes (a row's chunk c
    // of 16 stands at c ^ row / 2 % 8: two rows fill the banks once, so the reads of
    // one chunk of 16 rows fall on all sixteen places)
    static constexpr int kUnits = kCodes ? kBlocks * 4 : kBlocks * SK * P;
    static constexpr int kBytes = kUnits * kFragBytes;
    static constexpr int kScaleUnits = kCodes ? R / 64 : 0;  // of 64 words: a row's four scales each
    static constexpr size_t kStep = kCodes ? kPackGroup : static_cast<size_t>(SK) * P * kFragBytes;  // bytes, a stage

    // unit u of the tile of row block b0: where it starts, and the lane's offset from there
    static __device__ __forceinline__ const char *start(const char *planes, const Operand &o, int b0, int u, int kb,
                                                        int row_blocks) {
        if constexpr (kCodes) {
            return reinterpret_cast<const char *>(o.codes) + static_cast<size_t>(b0) * kPlaneRows * o.pitch;
        } else {
            const int row = min(b0 + u / (SK * P), row_blocks - 1);
            return planes + (static_cast<size_t>(row) * kb * P + u % (SK * P)) * kFragBytes;
        }
    }
    static __device__ __forceinline__ unsigned offset(const Operand &o, int b0, int u, int lane) {
        if constexpr (kCodes) {
            const int last = o.rows - 1 - b0 * kPlaneRows;  // rows past an edge: the last one's
            return static_cast<unsigned>(min(u * 8 + (lane >> 3), last)) * static_cast<unsigned>(o.pitch) +
                   16u * ((lane & 7) ^ (4 * u + (lane >> 4) & 7));
        } else {
            return 16u * lane;
        }
    }
    // the codes of k blocks 2 k and 2 k + 1 of row block b: lane 32 h + i has 16 h .. 16 h + 15
    // of row i's 32, its first eight for the one fragment and the others for the next (the
    // same order of k on both sides)
    static __device__ __forceinline__ u4v_t codes16(const char *at, int b, int k, int lane) {
        const int i = lane & 31, h = lane >> 5;
        return *reinterpret_cast<const u4v_t *>(at + b * 4096 + i * 128 + 16 * ((2 * k + h) ^ (i >> 1 & 7)));
    }
};

// A side of floats as they lie in memory (16-byte rows: ld a multiple of 4 and the
// base aligned), split as its fragments are read; R columns of C, stages of 32 k.
//   along k: 8 rows of 32 k a unit, a row's chunk c of 16 bytes at c ^ row / 2 % 8
//   along the rows: 2 k of 128 rows a unit, a k's row at row ^ 32 (k / 8 % 2)
template <Src S, int R, int SK>
struct StreamSide {
    static constexpr bool kCodes = false;
    static constexpr int P = 3, kBlocks = R / kPlaneRows, kUnits = R / 8;
    static_assert(SK * kPlaneK == 32 && R == 128, "units");
    static constexpr int kBytes = kUnits * kFragBytes, kScaleUnits = 0;

    static __device__ __forceinline__ const char *start(const Operand &o, int b0) {
        const size_t j0 = static_cast<size_t>(b0) * kPlaneRows;
        return reinterpret_cast<const char *>(o.p + (S == Src::kFloatK ? j0 * o.ld : j0));
    }
    static __device__ __forceinline__ size_t step(const Operand &o) {
        return S == Src::kFloatK ? 128 : static_cast<size_t>(128) * o.ld;
    }
    // unit u's lane: from a stage of `left` k (what lies past an edge: the last there
    // is, beside zeros of the other side or sums that are not stored)
    static __device__ __forceinline__ unsigned offset(const Operand &o, int b0, int u, int left, int lane) {
        const int j0 = b0 * kPlaneRows;
        if constexpr (S == Src::kFloatK) {
            const int row = u * 8 + (lane >> 3), k = 4 * ((lane & 7) ^ (row >> 1 & 7));
            return 4u * (static_cast<unsigned>(min(row, o.rows - 1 - j0)) * static_cast<unsigned>(o.ld) + min(k, left - 4));
        } else {
            const int k = u * 2 + (lane >> 5), row = 4 * (lane & 31) ^ 32 * (k >> 3 & 1);
            return 4u * (static_cast<unsigned>(min(k, left - 1)) * static_cast<unsigned>(o.ld) + min(row, o.rows - 4 - j0));
        }
    }
    // a lane's eight values of block b's fragment of k block k
    static __device__ __forceinline__ void values(const char *at, int b, int k, int lane, float (&v)[8]) {
        const int i = lane & 31, h = lane >> 5;
        if constexpr (S == Src::kFloatK) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const f4v_t four = *reinterpret_cast<const f4v_t *>(at + (b * kPlaneRows + i) * 128 +
                                                                    16 * ((4 * k + 2 * h + q) ^ (i >> 1 & 7)));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * q + e] = four[e];
            }
        } else {
            const float *from = reinterpret_cast<const float *>(at) + (16 * k + 8 * h) * R + ((b * kPlaneRows + i) ^ 32 * h);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = from[e * R];
        }
    }
    // ... and its three pieces
    static __device__ __forceinline__ void split(const float (&v)[8], b8v_t (&f)[3]) {
        u4v_t h4, m4, l4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const Pieces p = split2(v[2 * e], v[2 * e + 1], kSplitScale);
            h4[e] = p.h;
            m4[e] = p.m;
            l4[e] = p.l;
        }
        f[0] = __builtin_bit_cast(b8v_t, h4);
        f[1] = __builtin_bit_cast(b8v_t, m4);
        f[2] = __builtin_bit_cast(b8v_t, l4);
    }
};

// Four neighbouring sums (times 2^-scale) through the epilogue; cols of them are there.
__device__ __forceinline__ void epilogue4(const LinearEpi &e, size_t at, const f4v_t &v, int scale, const float (&bias)[4],
                                          const float (&extra)[4], int cols, float (&o)[4]) {
    float slope[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        o[n] = scale ? __builtin_ldexpf(v[n], -scale) : v[n];
        if (e.bias) o[n] += bias[n];
    }
    if (e.go) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            activate<true>(o[n], e.act, slope[n]);
            o[n] = through_slope(extra[n], slope[n]);
        }
        return;
    }
    if (e.slope) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            o[n] = activate<true>(o[n], e.act, slope[n]);
            if (n < cols) e.slope[at + n] = slope[n];
        }
    } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) o[n] = activate<false>(o[n], e.act, slope[n]);
    }
    if (e.residual) {
#pragma unroll
        for (int n = 0; n < 4; ++n) o[n] += extra[n];
    }
}

// SA, SB: the operands' kinds.  BM x BN by WM x WN waves; stages of SK k blocks,
// NST of them in LDS.  STREAM: B is floats as they lie (StreamSide), and KG groups
// of waves share a stage's k blocks.
template <Src SA, Src SB, int BM, int BN, int WM, int WN, int SK, int NST, bool STREAM = false, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void linear_planes(PlanesArgs g) {
    using A = PlaneSide<SA, BM, SK, as_codes(SA, SB)>;
    using B = std::conditional_t<STREAM, StreamSide<SB, BN, 2>, PlaneSide<SB, BN, SK, as_codes(SA, SB)>>;
    constexpr int PA = A::P, PB = B::P;
    constexpr int NW = WM * WN * KG, FM = BM / WM / kPlaneRows, FN = BN / WN / kPlaneRows;
    constexpr int NU = A::kUnits + B::kUnits, PER = (NU + NW - 1) / NW;  // a wave's; the last may be moved twice
    constexpr int NSC = A::kScaleUnits + B::kScaleUnits, SPER = (NSC + NW - 1) / NW;
    constexpr int kScalesAt = A::kBytes + B::kBytes, kStage = kScalesAt + 256 * NSC;
    __shared__ __attribute__((aligned(16))) char lds[NST * kStage];

    if constexpr (SA == Src::kFloatR || SA == Src::kCodesR) {
        const int past = static_cast<int>(blockIdx.x) - g.tiles_m * g.tiles_n * g.p.slices;
        if (past >= 0) return part_sums_block(g.sums, past, reinterpret_cast<double *>(lds));  // uniform
    }
    int tm, tn;
    const int slice = static_cast<int>(blockIdx.x) % g.p.slices;
    tile_coords(g.tiles_m, g.tiles_n, static_cast<int>(blockIdx.x) / g.p.slices, tm, tn);
    if (g.p.slices > 1) {  // uniform
        g.p.C = g.p.part + static_cast<size_t>(slice) * g.p.M * g.p.N;
        g.p.epi = LinearEpi{};
    }
    const int first = slice * g.slice_stages, end = min(first + g.slice_stages, g.stages);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN % WM, wn = wave % WN, kg = wave / (WM * WN);
    const int ra = tm * A::kBlocks, rb = tn * B::kBlocks;  // first row blocks

    // this wave's units of a stage: consecutive ones of A's, then of B's
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) char *)lds));
    const char *src[PER];
    unsigned off[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int f = min(wave * PER + i, NU - 1);
        if (f < A::kUnits) {
            src[i] = A::start(g.A, g.p.A, ra, f, g.kb, g.rows_a);
            off[i] = A::offset(g.p.A, ra, f, lane);
        } else if constexpr (STREAM) {
            src[i] = B::start(g.p.B, rb);
            off[i] = B::offset(g.p.B, rb, f - A::kUnits, 32, lane);
        } else {
            src[i] = B::start(g.B, g.p.B, rb, f - A::kUnits, g.kb, g.rows_b);
            off[i] = B::offset(g.p.B, rb, f - A::kUnits, lane);
        }
    }
    auto dma = [&](int stage, int slot) {
        const int at = min(stage, end - 1);  // past the end: the last again
        const unsigned base = lds0 + slot * kStage;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int f = min(wave * PER + i, NU - 1);
            unsigned from = off[i];
            const char *p;
            if constexpr (STREAM) {
                const int left = g.p.K - at * SK * kPlaneK;  // 1 at least
                p = src[i] + at * (f < A::kUnits ? A::kStep : B::step(g.p.B));
                if (left < 32 && f >= A::kUnits) from = B::offset(g.p.B, rb, f - A::kUnits, left, lane);  // uniform
            } else {
                p = src[i] + at * (f < A::kUnits ? A::kStep : B::kStep);
            }
            asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(from), "s"(p), "s"(base + f * kFragBytes)
                         : "memory", "m0");
        }
        if constexpr (NSC > 0) {
            const size_t group = at;
#pragma unroll
            for (int i = 0; i < SPER; ++i) {
                const int f = (wave * SPER + i) % NSC;
                const bool a = f < A::kScaleUnits;
                const Operand &o = a ? g.p.A : g.p.B;
                const int first = (a ? ra : rb) * kPlaneRows, row = first + (a ? f : f - A::kScaleUnits) * 64 + lane;
                const char *p = reinterpret_cast<const char *>(o.scales) + group * o.code_rows * 4;
                const unsigned to = 4u * static_cast<unsigned>(min(row, o.rows - 1));
                asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(to), "s"(p),
                             "s"(base + kScalesAt + f * 256)
                             : "memory", "m0");
            }
        }
#pragma clang diagnostic pop
    };
    auto frag = [&](const char *stage, int n) {
        return *reinterpret_cast<const b8v_t *>(stage + n * kFragBytes + lane * 16);
    };
    // a side's fragment from its codes, four: its row's scales
    auto widened = [&](const u4v_t &c, int half, unsigned four, int byte) {  // a scale byte is fp32's exponent
        return widen(c[2 * half], c[2 * half + 1], __uint_as_float((four >> (8 * byte) & 255u) << 23));
    };

    floatx16 acc[FM][FN];
#pragma unroll
    for (int x = 0; x < FM; ++x)
#pragma unroll
        for (int c = 0; c < FN; ++c) acc[x][c] = floatx16{};

    // a k block's products of a block, added to acc
    auto multiply = [](floatx16 &acc, const b8v_t (&a)[PA], const b8v_t (&b)[PB], float sign) {
        auto mm = [&](floatx16 v, int pa, int pb) {
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[pa], b[pb], v, 0, 0, 0);
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
            for (int r = 0; r < 16; ++r) acc[r] = __builtin_fmaf(v[r], sign, acc[r]);
        } else {
#pragma unroll
            for (int p = PB - 1; p >= 0; --p) acc = mm(acc, 0, p);
        }
    };
    int slot = 0;
    if constexpr (STREAM) {
        // A group's wave has one k block a stage.  B's values of the next are read and
        // split beside the last block's products of this one, whose A is read by then.
        static_assert(SK == KG && FN == 1 && FM > 1, "a k block a wave");
        auto read_a = [&](int slot, int x, b8v_t (&fa)[PA]) {
#pragma unroll
            for (int p = 0; p < PA; ++p) fa[p] = frag(lds + slot * kStage, ((wm * FM + x) * SK + kg) * PA + p);
        };
        float v[8];
        b8v_t fb[3];
#pragma unroll
        for (int s = 0; s < NST; ++s) dma(first + s, s);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(PER * (NST - 1)) : "memory");
        B::values(lds + A::kBytes, wn, kg, lane, v);
        B::split(v, fb);
        const float sign = kg ? -1.0f : 1.0f;
        for (int s = first; s < end; ++s) {
            b8v_t fa[PA];
#pragma unroll
            for (int x = 0; x + 1 < FM; ++x) {
                read_a(slot, x, fa);
                multiply(acc[x][0], fa, fb, sign);
            }
            read_a(slot, FM - 1, fa);
            // the next stage has landed, and every wave has read this one
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PER * (NST - 2)) : "memory");
            dma(s + NST, slot);
            slot = slot + 1 == NST ? 0 : slot + 1;
            B::values(lds + slot * kStage + A::kBytes, wn, kg, lane, v);  // (past the end: not used)
            multiply(acc[FM - 1][0], fa, fb, sign);
            B::split(v, fb);
        }
    } else {
#pragma unroll
        for (int s = 0; s < NST - 1; ++s) dma(first + s, s);
        for (int s = first; s < end; ++s) {
            // this stage has landed, and every wave is done with the one before
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((PER + SPER) * (NST - 2)) : "memory");
            dma(s + NST - 1, slot == 0 ? NST - 1 : slot - 1);
            const char *at = lds + slot * kStage, *at_b = at + A::kBytes;
            unsigned sa[FM], sb[FN];  // the rows' scales
            auto row_scales = [&](int first, int row) {
                return *reinterpret_cast<const unsigned *>(at + kScalesAt + first * 256 + (row * kPlaneRows + (lane & 31)) * 4);
            };
            if constexpr (A::kCodes) {
#pragma unroll
                for (int x = 0; x < FM; ++x) sa[x] = row_scales(0, wm * FM + x);
            }
            if constexpr (B::kCodes) {
#pragma unroll
                for (int c = 0; c < FN; ++c) sb[c] = row_scales(A::kScaleUnits, wn * FN + c);
            }
            u4v_t ca[FM], cb[FN];  // two k blocks' codes
#pragma unroll
            for (int k = 0; k < SK; ++k) {
                if constexpr (A::kCodes) {
                    if (k % 2 == 0) {
#pragma unroll
                        for (int c = 0; c < FN; ++c) cb[c] = B::codes16(at_b, wn * FN + c, k / 2, lane);
#pragma unroll
                        for (int x = 0; x < FM; ++x) ca[x] = A::codes16(at, wm * FM + x, k / 2, lane);
                    }
                }
                b8v_t fb[FN][PB];
#pragma unroll
                for (int c = 0; c < FN; ++c) {
                    if constexpr (B::kCodes) {
                        fb[c][0] = widened(cb[c], k % 2, sb[c], k / 2);
                    } else {
#pragma unroll
                        for (int p = 0; p < PB; ++p) fb[c][p] = frag(at_b, ((wn * FN + c) * SK + k) * PB + p);
                    }
                }
                const float sign = (s * SK + k) & 1 ? -1.0f : 1.0f;
#pragma unroll
                for (int x = 0; x < FM; ++x) {
                    b8v_t fa[PA];
                    if constexpr (A::kCodes) {
                        fa[0] = widened(ca[x], k % 2, sa[x], k / 2);
                    } else {
#pragma unroll
                        for (int p = 0; p < PA; ++p) fa[p] = frag(at, ((wm * FM + x) * SK + k) * PA + p);
                    }
#pragma unroll
                    for (int c = 0; c < FN; ++c) multiply(acc[x][c], fa, fb[c], sign);
                }
            }
            slot = slot + 1 == NST ? 0 : slot + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outstanding at exit

    if constexpr (KG == 2) {  // the second group's sums onto the first's
        static_assert(NST * kStage >= BM * BN * 4, "room for the second's");
        f4v_t *const second = reinterpret_cast<f4v_t *>(lds) + wave % (WM * WN) * FM * FN * 256 + lane;
        __syncthreads();  // the last fragments
        if (kg == 1) {
#pragma unroll
            for (int n = 0; n < FM * FN * 4; ++n) {
                const floatx16 &v = acc[n / 4 / FN][n / 4 % FN];
                second[n * 64] = f4v_t{v[4 * (n % 4)], v[4 * (n % 4) + 1], v[4 * (n % 4) + 2], v[4 * (n % 4) + 3]};
            }
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int n = 0; n < FM * FN * 4; ++n) {
                const f4v_t v = second[n * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n / 4 / FN][n / 4 % FN][4 * (n % 4) + e] += v[e];
            }
        }
    }
    if constexpr (PB == 3) {  // (codes hold finite values, and their product's own range is fp32's)
        float worst = 0.0f;  // NaN * 0 and inf * 0 stay NaN
#pragma unroll
        for (int x = 0; x < FM; ++x)
#pragma unroll
            for (int c = 0; c < FN; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) worst = __builtin_fmaf(acc[x][c][r], 0.0f, worst);
        if (__syncthreads_or(worst != worst)) {  // uniform
            constexpr int TN = BN / kDirectTile;
            for (int t = wave; t < BM / kDirectTile * TN; t += NW) {
                const int ti = tm * (BM / kDirectTile) + t / TN, tj = tn * TN + t % TN;
                if (ti * kDirectTile < g.p.M && tj < g.p.tiles_n) direct_tile<SA, SB>(g.p, ti * g.p.tiles_n + tj, first * SK, end * SK, lane);
            }
            return;
        }
    }

    // The tile by LDS (lane (i, h), register r of block (x, c): row 8 (r / 4) + 4 h +
    // r % 4, column i, at column ^ 32 h: the halves in different banks), then by
    // rows, four columns a lane, with the epilogue.
    // A turn's go or residual is on its way while the one before is computed.
    static_assert(NST * kStage >= BM * BN * 4 && BN >= 64, "room for the tile");
    constexpr int kScale = (PA == 3 ? 16 : 0) + (PB == 3 ? 16 : 0);
    constexpr int kRowQuads = BN / 4, kStep = 64 * NW / kRowQuads, kRows = BM / kStep < 4 ? BM / kStep : 4, kTurns = BM / kStep / kRows;
    static_assert(kTurns * kStep * kRows == BM, "turns of kRows rows a lane");
    float *const sums = reinterpret_cast<float *>(lds);
    const float *extra = g.p.epi.go ? g.p.epi.go : g.p.epi.residual;
    const int jt = static_cast<int>(threadIdx.x) % kRowQuads * 4, j = tn * BN + jt;  // a lane keeps its columns
    const int cols = min(4, g.p.N - j), row0 = static_cast<int>(threadIdx.x) / kRowQuads, last = g.p.M - 1 - tm * BM;
    const size_t at0 = static_cast<size_t>(tm) * BM * g.p.N + j;
    float ev[kRows][4];
    auto fetch = [&](int turn) {
#pragma unroll
        for (int t = 0; t < kRows; ++t) {  // (rows past the edge: the last one's)
            const float *q = extra + at0 + static_cast<size_t>(min((turn * kRows + t) * kStep + row0, last)) * g.p.N;
            if (cols == 4) {
                *reinterpret_cast<f4v_t *>(ev[t]) = *reinterpret_cast<const f4u_t *>(q);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) ev[t][e] = e < cols ? q[e] : 0.0f;
            }
        }
    };
    float bias[4] = {};
    if (cols > 0) {
        if (extra) fetch(0);
        if (g.p.epi.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[e] = g.p.epi.bias[min(j + e, g.p.N - 1)];
        }
    }
    const int li = lane & 31, lh = lane >> 5;
    __syncthreads();  // the last fragments
    if (kg == 0) {  // uniform
#pragma unroll
        for (int x = 0; x < FM; ++x)
#pragma unroll
            for (int c = 0; c < FN; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = (wm * FM + x) * kPlaneRows + 8 * (r >> 2) + 4 * lh + (r & 3);
                    sums[row * BN + (((wn * FN + c) * kPlaneRows + li) ^ 32 * lh)] = acc[x][c][r];
                }
    }
    __syncthreads();
    if (cols <= 0) return;  // (no barrier follows)
#pragma unroll 1
    for (int turn = 0; turn < kTurns; ++turn) {
        float now[kRows][4];
#pragma unroll
        for (int t = 0; t < kRows; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) now[t][e] = ev[t][e];
        if (extra && turn + 1 < kTurns) fetch(turn + 1);
#pragma unroll
        for (int t = 0; t < kRows; ++t) {
            const int row = (turn * kRows + t) * kStep + row0;
            if (row > last) continue;
            const f4v_t v = *reinterpret_cast<const f4v_t *>(sums + row * BN + (jt ^ 32 * (row >> 2 & 1)));
            const size_t at = at0 + static_cast<size_t>(row) * g.p.N;
            float o[4];
            epilogue4(g.p.epi, at, v, kScale, bias, now[t], cols, o);
            if (cols == 4) {
                *reinterpret_cast<f4u_t *>(g.p.C + at) = f4u_t{o[0], o[1], o[2], o[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < cols) g.p.C[at + e] = o[e];
            }
        }
    }
}

}  // namespace tship
