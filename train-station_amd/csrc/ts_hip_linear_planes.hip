// The passes that write an operand's planes and the launches of the large
// products (the kernel and the layout: ts_hip_linear_planes.h).
#include <algorithm>

#include "ts_hip_linear_planes.h"

namespace tship {

namespace {

typedef unsigned u4p_t __attribute__((ext_vector_type(4)));

// eight values times scale as their three pieces, a lane's 16 bytes of each
__device__ __forceinline__ void store_pieces(char *to, const float (&v)[8], float scale, int lane) {
    u4p_t h, m, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const Pieces p = split2(v[2 * e], v[2 * e + 1], scale);
        h[e] = p.h;
        m[e] = p.m;
        l[e] = p.l;
    }
    u4p_t *q = reinterpret_cast<u4p_t *>(to) + lane;
    q[0] = h;
    q[kFragBytes / 16] = m;
    q[2 * kFragBytes / 16] = l;
}

// One operand's part of a pass: its waves' jobs, in `blocks` workgroups.
struct PlaneJob {
    Operand o;
    Src src;
    int negate;           // odd k blocks (A beside pieces)
    int K, kb;            // the product's k, in k blocks
    char *out;
    int chunks;           // floats along k: jobs of a row block
    int run, row_blocks;  // along the rows: k blocks of a job
    unsigned blocks;
    uint8_t *codes, *scales;  // floats along k: the values in 8 bits too
    float *sum_parts;         // floats along the rows: their sums, [chunk][rows]
};

// ---- floats along k ----------------------------------------------------------------
// A wave takes a row block and four k blocks (256 bytes of each row).  The values
// in 8 bits: a block of 32 k is two k blocks of the lane and its partner in the
// other half.
constexpr int kAlongBlocks = 4;

__device__ __forceinline__ void planes_along(const PlaneJob &j, size_t job) {
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5, rows = j.o.rows, K = j.K, kb = j.kb;
    const int rb = static_cast<int>(job / j.chunks), b0 = static_cast<int>(job % j.chunks) * kAlongBlocks;
    if (rb * kPlaneRows >= rows) return;
    const int row = rb * kPlaneRows + i;
    const bool live = row < rows;
    const size_t at = static_cast<size_t>(live ? row : 0) * j.o.ld;
    const float *p = j.o.p + at, *tp = j.o.times ? j.o.times + at : nullptr;
    float v[kAlongBlocks][8];
#pragma unroll
    for (int b = 0; b < kAlongBlocks; ++b)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int k = (b0 + b) * kPlaneK + 8 * h + 4 * q;
            float w[4] = {};
            if (live && k + 4 <= K) {
                const pk4u_t t = *reinterpret_cast<const pk4u_t *>(p + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = t[e];
                if (tp) {  // uniform
                    const pk4u_t s = *reinterpret_cast<const pk4u_t *>(tp + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = through_slope(t[e], s[e]);
                }
            } else if (live) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = k + e < K ? (tp ? through_slope(p[k + e], tp[k + e]) : p[k + e]) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[b][4 * q + e] = w[e];
        }
#pragma unroll
    for (int b = 0; b < kAlongBlocks; ++b) {
        if (b0 + b >= kb) break;  // uniform
        store_pieces(j.out + (static_cast<size_t>(rb) * kb + b0 + b) * 3 * kFragBytes, v[b],
                     j.negate && (b & 1) ? -kSplitScale : kSplitScale, lane);
    }
    if (j.codes) {  // uniform
        const size_t pitch = packed_pitch(K);
#pragma unroll
        for (int b = 0; b < kAlongBlocks; b += 2) {
            const size_t c = static_cast<size_t>(b0 + b) * kPlaneK;
            if (c >= pitch) break;  // uniform
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaxf(fabsf(v[b][e]), fabsf(v[b + 1][e])));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (!live) continue;
            const int k = pack_exponent(m);
            const float inv = pow2f(-k);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float lo[4], hi[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo[e] = v[b + t][e];
                    hi[e] = v[b + t][4 + e];
                }
                *reinterpret_cast<u2v_t *>(j.codes + row * pitch + c + t * kPlaneK + 8 * h) = u2v_t{pack4(lo, inv), pack4(hi, inv)};
            }
            if (h == 0)
                j.scales[(c / kPackGroup * rows + row) * 4 + c / kPackBlock % 4] = static_cast<uint8_t>(k + kPackBias);
        }
    }
}

// ---- floats along the rows -----------------------------------------------------------
// element (row, k) at p[k * ld + row].  A wave takes a row block and `run` k blocks;
// with sum_parts the rows' sums over them (f64) too.
__device__ __forceinline__ void planes_across(const PlaneJob &j, size_t job) {
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5, ld = j.o.ld, rows = j.o.rows, K = j.K, kb = j.kb;
    const int rb = static_cast<int>(job % j.row_blocks), chunk = static_cast<int>(job / j.row_blocks);
    const int from = chunk * j.run, to = min(from + j.run, kb);
    if (from >= kb) return;
    const int row = rb * kPlaneRows + i;
    const bool live = row < rows;
    const float *p = j.o.p + (live ? row : 0), *tp = j.o.times ? j.o.times + (live ? row : 0) : nullptr;
    double sum = 0.0;
#pragma unroll 2
    for (int b = from; b < to; ++b) {
        const int k = b * kPlaneK + 8 * h;
        float v[8];
        if ((b + 1) * kPlaneK <= K) {  // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[static_cast<size_t>(k + e) * ld];
            if (tp) {  // uniform
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = through_slope(v[e], tp[static_cast<size_t>(k + e) * ld]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const size_t at = static_cast<size_t>(k + e) * ld;
                v[e] = k + e < K ? (tp ? through_slope(p[at], tp[at]) : p[at]) : 0.0f;
            }
        }
        if (!live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
        if (j.sum_parts) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += v[e];
        }
        store_pieces(j.out + (static_cast<size_t>(rb) * kb + b) * 3 * kFragBytes, v, j.negate && (b & 1) ? -kSplitScale : kSplitScale,
                     lane);
    }
    if (j.sum_parts) {
        sum += __shfl_xor(sum, 32, 64);
        if (h == 0 && live) j.sum_parts[static_cast<size_t>(chunk) * rows + row] = static_cast<float>(sum);
    }
}

// ---- codes -----------------------------------------------------------------------------

// Codes along k.  A wave takes a row block and a group of 128 k, the lane's scales in one word.
__device__ __forceinline__ void planes_codes_along(const PlaneJob &j, size_t job) {
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5, rows = j.o.rows, kb = j.kb;
    const size_t pitch = j.o.pitch;
    const int groups = static_cast<int>(pitch / kPackGroup);
    const int rb = static_cast<int>(job / groups), g = static_cast<int>(job % groups);
    if (rb * kPlaneRows >= rows) return;
    const int row = rb * kPlaneRows + i;
    const bool live = row < rows;
    const size_t r = live ? row : 0;
    const unsigned four = reinterpret_cast<const unsigned *>(j.o.scales)[static_cast<size_t>(g) * rows + r];
    u2v_t c[8];
#pragma unroll
    for (int b = 0; b < 8; ++b)
        c[b] = *reinterpret_cast<const u2v_t *>(j.o.codes + r * pitch + static_cast<size_t>(g) * kPackGroup + b * kPlaneK + 8 * h);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        if (g * 8 + b >= kb) break;  // uniform
        bf8_t w = widen(c[b][0], c[b][1], pow2f(static_cast<int>(four >> (8 * (b / 2)) & 255u) - kPackBias));
        if (!live) w = bf8_t{};
        *(reinterpret_cast<bf8_t *>(j.out + (static_cast<size_t>(rb) * kb + g * 8 + b) * kFragBytes) + lane) = w;
    }
}

// Codes along the rows: k is the code row, the product's rows its columns.  A wave
// takes 32 columns (a row block, and a scale's block) of 64 code rows; a lane four
// columns of eight.
__device__ __forceinline__ void planes_codes_across(const PlaneJob &j, size_t job) {
    const int lane = threadIdx.x & 63, i = lane & 7, o = lane >> 3, kb = j.kb, code_rows = static_cast<int>(j.o.code_rows);
    const uint8_t *codes = j.o.codes, *scales = j.o.scales;
    const size_t pitch = j.o.pitch;
    const int rb = static_cast<int>(job % j.row_blocks), b0 = static_cast<int>(job / j.row_blocks) * 4;
    if (b0 >= kb) return;
    const int k0 = b0 * kPlaneK + 8 * o;
    const size_t col = static_cast<size_t>(rb) * kPlaneRows;
    const uint8_t *sp = scales + (col / kPackGroup * code_rows) * 4 + col / kPackBlock % 4;
    unsigned c[8];
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // rows past the end: the last one's scale, codes of zero
        const size_t k = min(k0 + e, code_rows - 1);
        c[e] = *reinterpret_cast<const unsigned *>(codes + k * pitch + col + 4 * i);
        if (k0 + e >= code_rows) c[e] = 0;
        s[e] = pow2f(static_cast<int>(sp[4 * k]) - kPackBias);
    }
    const int b = b0 + (o >> 1), h = o & 1;
    if (b >= kb) return;
    bf2_t lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo[e] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[e], s[e], false);
        hi[e] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[e], s[e], true);
    }
    bf8_t *to = reinterpret_cast<bf8_t *>(j.out + (static_cast<size_t>(rb) * kb + b) * kFragBytes) + 32 * h + 4 * i;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        bf8_t w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = n < 2 ? lo[e][n & 1] : hi[e][n & 1];
        to[n] = w;
    }
}

// Several operands' planes by one launch.
struct PlaneJobs {
    PlaneJob job[kMaxPlaneTasks];
    int count;
};

__global__ __launch_bounds__(kBlock) void write_planes(PlaneJobs jobs) {
    unsigned block = blockIdx.x;
#pragma unroll
    for (int n = 0; n < kMaxPlaneTasks; ++n) {
        const PlaneJob &j = jobs.job[n];
        if (n >= jobs.count) return;  // (uniform, as the rest)
        if (block >= j.blocks) {
            block -= j.blocks;
            continue;
        }
        const size_t job = static_cast<size_t>(block) * (kBlock / 64) + (threadIdx.x >> 6);
        if (j.src == Src::kFloatK) planes_along(j, job);
        else if (j.src == Src::kFloatR) planes_across(j, job);
        else if (j.src == Src::kCodesK) planes_codes_along(j, job);
        else planes_codes_across(j, job);
        return;
    }
}

// ---- launches ----------------------------------------------------------------------------

int row_blocks(size_t rows) { return static_cast<int>((rows + kPlaneRows - 1) / kPlaneRows); }
int k_blocks(size_t K) { return static_cast<int>((K + 2 * kPlaneK - 1) / (2 * kPlaneK)) * 2; }
size_t plane_bytes(size_t rows, size_t K, Src s) {
    return static_cast<size_t>(row_blocks(rows)) * k_blocks(K) * (pieces_of(s)) * kFragBytes;
}

unsigned wave_grid(size_t jobs) { return static_cast<unsigned>((jobs + kBlock / 64 - 1) / (kBlock / 64)); }

// k blocks a wave of planes_across takes: as many as leave eight waves a SIMD
int across_run(size_t rows, size_t K) {
    const size_t waves = static_cast<size_t>(device_cu_count()) * 32, all = static_cast<size_t>(row_blocks(rows)) * k_blocks(K);
    const size_t run = all / waves;
    return static_cast<int>(run < 2 ? 2 : run > 16 ? 16 : run);
}
int across_chunks(size_t rows, size_t K) {
    const int run = across_run(rows, K);
    return (k_blocks(K) + run - 1) / run;
}

PlaneJob plane_job(const PlaneTask &t) {
    const LinearProduct &p = *t.p;
    const Operand &o = t.b ? p.B : p.A;
    const Src src = t.b ? p.b : p.a;
    PlaneJob j = {o, src, !t.b, p.K, k_blocks(p.K), t.out, 0, 0, row_blocks(o.rows), 0, t.codes, t.scales, t.sum_parts};
    const size_t rb = j.row_blocks;
    if (src == Src::kFloatK) {
        const size_t blocks = t.codes ? packed_pitch(p.K) / kPlaneK : j.kb;
        j.chunks = static_cast<int>((blocks + kAlongBlocks - 1) / kAlongBlocks);
        j.blocks = wave_grid(rb * j.chunks);
    } else if (src == Src::kFloatR) {
        j.run = across_run(o.rows, p.K);
        j.blocks = wave_grid(rb * across_chunks(o.rows, p.K));
    } else {
        j.blocks = wave_grid(rb * (src == Src::kCodesK ? o.pitch / kPackGroup : (j.kb + 3) / 4));
    }
    return j;
}

template <Src SA, Src SB, int BM, int BN, int WM, int WN, int SK, int NST, bool STREAM = false, int KG = 1>
void launch_planes(PlanesArgs g, hipStream_t s) {
    g.tiles_m = (g.p.M + BM - 1) / BM;
    g.tiles_n = (g.p.N + BN - 1) / BN;
    g.stages = as_codes(SA, SB) ? static_cast<int>(g.p.A.pitch / kPackGroup) : g.kb / SK;
    g.slice_stages = (g.stages + g.p.slices - 1) / g.p.slices;
    launch((linear_planes<SA, SB, BM, BN, WM, WN, SK, NST, STREAM, KG>),
           dim3(g.tiles_m * g.tiles_n * g.p.slices + g.sums.blocks), dim3(64 * WM * WN * KG), 0, s, g);
}

// The tile, and the slices of K, that cost least: rounds over the chip x a tile's
// share of K x its area, the smaller tiles 1.03 and 1.1 times as dear, and a larger
// one 1.15 or 1.3 times where a CU has but one workgroup to fill its waits; slices
// cost a launch and their sums' way to memory and back.  us in 128 x 128, 128 x 64,
// 64 x 64, pieces on both sides: 8192 x 4096 x 4096 1242, 1295, 1419; 2048 x 4096 x
// 1024 89.6, 95, 98; 1024 x 4096 x 2048 98, 88, 106; 2048 x 1024 x 4096 163, -, 95;
// 1024 x 1024 x 1024 45, -, 23.  One side's: 604, 631, 764; 48.5, 53, 59; 51, 50, 59;
// 1003 x 2050 x 3000 66, 58, 53.  Codes: 253, 268, 298; 28, 28, 29; 29, 26, 26;
// 2048 x 1024 x 4096 40, 29, 27; 1999 x 777 x 1531 22, 16, 14.  (128 x 256 and
// 256 x 256 by eight waves: no faster at the largest, and slower below.)
struct PlanesPlan {
    int bm, bn, slices;
};
PlanesPlan choose_plan(size_t M, size_t N, size_t K, Src a, Src b) {
    const size_t cus = device_cu_count();
    const double each = as_codes(a, b) ? 0.8e-6 : of_codes(a) ? 1.4e-6 : 2.6e-6;  // us per k of a column of a tile, one a CU
    PlanesPlan best = {128, 128, 1};
    double least = 1e30;
    auto take = [&](size_t bm, size_t bn, double dear, double alone) {
        const size_t tiles = (M + bm - 1) / bm * ((N + bn - 1) / bn);
        for (size_t n = 1; n <= 8 && (n == 1 || (K >= n * 512 && tiles * n <= 4 * cus)); n *= 2) {
            const size_t rounds = (tiles * n + cus - 1) / cus;
            double us = rounds * bm * bn * (rounds == 1 ? alone : dear) * each * K / n;
            if (n > 1) us += 6 + 2e-6 * M * N * n;
            if (us < least) {
                least = us;
                best = {static_cast<int>(bm), static_cast<int>(bn), static_cast<int>(n)};
            }
        }
    };
    take(128, 128, 1.0, 1.15);
    take(128, 64, 1.03, 1.3);
    take(64, 64, 1.1, 1.1);
    return best;
}

// Tiles of a product whose B streams: 128 columns, all rows up to 128 (half the
// rows everywhere, and four stages: 128 x 4096 x 4096 133 us, 138 here; 256 x 4096 x
// 4096 216, 208; 300 x 8000 x 1000 155, 145), and the slices of K that fill the chip
// (doublings: 300 x 8000 x 1000 162, 155), of 128 k at least.
PlanesPlan stream_plan(size_t M, size_t N, size_t K) {
    PlanesPlan p = {M <= 64 ? 64 : 128, 128, 1};
    const size_t tiles = (M + p.bm - 1) / p.bm * ((N + 127) / 128), cus = device_cu_count();
    const size_t n = std::min(cus / tiles, K / 128);
    if (n > 1) p.slices = static_cast<int>(n);
    return p;
}

size_t round_256(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

// Large by its operations (forward and backward, us, by planes and directly: 8192 x 300 x
// 200 (0.98e9) 82, 115; 4118 x 448 x 225 (0.83e9) 68, 87; 750 x 600 x 700 (0.63e9) 67, 64;
// 1024 x 512 x 512 (0.54e9) 65, 50; codes, 2048 x 512 x 512 (1.07e9) 8.6, 9.6, 1024 x 512 x
// 512 8.2, 7.5), or a large C of few k, whose stores bound it: 1 x 4096 x 4096 74, 87; 32 x
// 4096 x 4096 89, 108; 32 x 2048 x 2048 (4e6) 68, 63; 1 x 1024 x 8192 (8e6) 57, 47.
bool planes_take(size_t M, size_t N, size_t K) {
    const double c = 1.0 * M * N;
    return M >= 128 && N >= 128 && K > 0 && (2 * c * K >= 0.8e9 || c >= (K < 16 ? 12e6 : 6e6));
}

// Few rows beside a large weight: its planes would be written for a few readings.
// Forward and backward, us, streamed, from planes, directly: 512 x 4096 x 4096 346,
// 405; 256 x 2500 x 2500 125, 158; 128 x 4096 x 4096 138, 257; 64 x 4096 x 4096 93, -,
// 145; 60 x 3000 x 3000 81, -, 113; 8 x 8192 x 8192 233, -, 310.  And where it is not
// taken: 700 x 3000 x 3000 383, 349; 512 x 1024 x 1024 98, -, 80; 64 x 2048 x 2048 with
// an 8-bit checkpoint 87, -, 82; 1 x 1024 x 8192 57, -, 47.
bool streams_take(size_t M, size_t N, size_t K, size_t ld) {
    const double weight = 1.0 * N * K;
    return M > 0 && M <= 512 && N >= 128 && K >= 64 && (2 * M * weight >= 1.5e9 || weight >= (M < 32 ? 12e6 : 6e6)) && ld % 4 == 0 &&
           ld <= size_t(1) << 20;  // (a tile's offsets in 32 bits)
}

size_t streams_workspace_floats(size_t M, size_t N, size_t K, Src a) {
    const PlanesPlan plan = stream_plan(M, N, K);
    return (round_256(plane_bytes(M, K, a)) + (plan.slices > 1 ? round_256(plan.slices * M * N * sizeof(float)) : 0)) / sizeof(float);
}

size_t planes_workspace_floats(size_t M, size_t N, size_t K, Src a, Src b) {
    const PlanesPlan plan = choose_plan(M, N, K, a, b);
    const size_t planes = as_codes(a, b) ? 0 : (round_256(plane_bytes(M, K, a)) + round_256(plane_bytes(N, K, b))) / sizeof(float);
    return planes + (plan.slices > 1 ? round_256(plan.slices * M * N * sizeof(float)) / sizeof(float) : 0);
}

size_t planes_sum_floats(size_t N, size_t K) { return static_cast<size_t>(across_chunks(N, K)) * N; }

char *planes_of_a(const LinearProduct &, float *workspace) { return reinterpret_cast<char *>(workspace); }
char *planes_of_b(const LinearProduct &p, float *workspace) {
    return reinterpret_cast<char *>(workspace) + round_256(plane_bytes(p.M, p.K, p.a));
}

void planes_write(const PlaneTask *tasks, int count, hipStream_t s) {
    PlaneJobs jobs = {};
    jobs.count = count;
    unsigned blocks = 0;
    for (int n = 0; n < count; ++n) {
        jobs.job[n] = plane_job(tasks[n]);
        blocks += jobs.job[n].blocks;
    }
    if (blocks) launch(write_planes, dim3(blocks), dim3(kBlock), 0, s, jobs);
}

void planes_multiply(const LinearProduct &p, float *workspace, const float *sum_parts, float *sums, hipStream_t s) {
    char *pa = planes_of_a(p, workspace), *pb = planes_of_b(p, workspace);
    const PlanesPlan plan = p.streams ? stream_plan(p.M, p.N, p.K) : choose_plan(p.M, p.N, p.K, p.a, p.b);
    PlanesArgs g = {pa, pb, direct_product(p), k_blocks(p.K), row_blocks(p.M), row_blocks(p.N), 0, 0, 0, 0, {}};
    g.p.slices = plan.slices;
    if (sums) g.sums = part_sums(sum_parts, across_chunks(p.N, p.K), p.N, sums);
    if (p.streams && plan.slices > 1) g.p.part = reinterpret_cast<float *>(pb);
    else if (plan.slices > 1)
        g.p.part = as_codes(p.a, p.b) ? workspace : reinterpret_cast<float *>(pb + round_256(plane_bytes(p.N, p.K, p.b)));
    with_sources(p.a, p.b, [&](auto a, auto b) {
        constexpr Src A = a.value, B = b.value;
        if constexpr (A != Src::kFloatR && A != Src::kCodesR && !as_codes(A, B)) {
            if (p.streams) {
                if (plan.bm == 64) launch_planes<A, B, 64, 128, 1, 4, 2, 3, true, 2>(g, s);
                else launch_planes<A, B, 128, 128, 1, 4, 2, 3, true, 2>(g, s);
                return;
            }
        }
        // waves and stages: 128 codes a stage; else 32 k, two stages, but 16 k and three where
        // 128 x 128 has three pieces on both sides (8192 x 4096 x 4096 1242 us by eight waves,
        // 1302 by four), and four where the smallest tile has them on one (1024 x 4096 x 2048
        // 59 us, 61 in three of 32)
        if constexpr (as_codes(A, B)) {
            if (plan.bm == 64) launch_planes<A, B, 64, 64, 2, 2, 8, 2>(g, s);
            else if (plan.bn == 64) launch_planes<A, B, 128, 64, 2, 2, 8, 2>(g, s);
            else launch_planes<A, B, 128, 128, 2, 2, 8, 2>(g, s);
        } else if constexpr (pieces_of(A) == 3) {
            if (plan.bm == 64) launch_planes<A, B, 64, 64, 2, 2, 2, 2>(g, s);
            else if (plan.bn == 64) launch_planes<A, B, 128, 64, 2, 2, 2, 2>(g, s);
            else launch_planes<A, B, 128, 128, 4, 2, 1, 3>(g, s);
        } else {
            if (plan.bm == 64) launch_planes<A, B, 64, 64, 2, 2, 1, 4>(g, s);
            else if (plan.bn == 64) launch_planes<A, B, 128, 64, 2, 2, 2, 2>(g, s);
            else launch_planes<A, B, 128, 128, 2, 4, 2, 2>(g, s);
        }
    });
    join_slices(g.p, s);
}

}  // namespace tship
