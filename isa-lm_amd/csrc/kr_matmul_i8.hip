// Products of 8-bit integers with a scale a token and a scale an output
// (krh_matmul_i8, krh_matmul_i8_swiglu): Y[t][r] = (sum_k W[r][k] x[t][k]) xd[t] wd[r].
//
// The sums are exact in 32 bits whatever their order, so the reduction is split
// and its parts are joined freely, and every form gives the same bits: one
// float conversion and two products an output.
#include <cfloat>
#include <cmath>
#include <type_traits>
#include "kr_internal.h"
#include "kr_numerics.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int I8_COLS = (1 << 17) - 1;   // 2^14 * cols < 2^31
constexpr size_t I8_LD = 1 << 23;        // a tile's rows within 32-bit offsets

struct I8Args {
    float *y;
    size_t ldy;
    const int8_t *w[2];   // the second with GLU
    const float *wd[2];
    size_t ldw[2];
    const int8_t *x;
    size_t ldx;
    const float *xd, *bias;
    int rows, cols, ntok, add;
};

// the first n of 16 bytes, then zeros
__device__ __forceinline__ v4i i8_cut(v4i v, int n) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = n - 4 * i;
        if (left < 4) v[i] = left <= 0 ? 0 : v[i] & (int)((1u << 8 * left) - 1);
    }
    return v;
}
__device__ __forceinline__ float i8_scaled(int sum, float xd, float wd) { return kr_fmul(kr_fmul((float)sum, xd), wd); }
// silu(g) u = g / (1 + e^-g) u within 8 half steps. The power of two takes the product g log2 e in two parts;
// below -88, where e^-g leaves the floats, silu is 0 (to 6e-37). (The C library's
// expf and the division, which krh_silu_mul takes, are 90 instructions an output and
// would be a third of a prompt's time.)
__device__ __forceinline__ float i8_silu_mul(float g, float u) {
    const float x = fminf(fmaxf(g, -88.0f), 88.0f);
    const float t = x * -1.44269502f;
    const float lo = __builtin_fmaf(x, -1.92596299e-8f, __builtin_fmaf(x, -1.44269502f, -t));
    float e = __builtin_amdgcn_exp2f(t);
    e = __builtin_fmaf(e, lo * 0.693147182f, e);
    const float s = g < -88.0f ? 0.0f : __builtin_amdgcn_rcpf(1.0f + e);
    return kr_fmul(kr_fmul(g, s), u);
}

// Tiles of BT tokens and BR rows (GLU: MB rows of each matrix in turn), WT x WR
// waves with an even part each, or WK times as many, each with a part of the
// reduction. That goes in stages of BK values, which pass from memory to LDS
// without registers, NB stages in a ring: one barrier a stage, and a stage's loads
// are under way while the NB - 1 before it are worked on. A row's 16-byte chunks lie
// in LDS in an order of the row's own, so that the rows that a wave reads one chunk
// of are in different banks; the order is taken from the source's side, as the
// loads fill LDS in lane order.
//
// What bounds them. The largest tile (256 x 256, waves of 128 x 64): the matrix cores are
// busy 53% of the cycles, at 1.9 GHz of 2.4, and the waves wait 39% of theirs, 3% for LDS
// to take a read: a stage's 192 KB of reads and 64 KB of loads are as much as LDS
// passes in the 2048 clocks of its products, and a barrier ends it; 2047
// tokens of the 8B shape's w1 and w3 take 252 us (1.9 POP/s; 267 with waves of 128 x 128,
// one a SIMD; 333 in tiles of 128 x 128). Tiles of 128 x 128 run at 1.2 to 1.5 GHz (2047 tokens, 4096
// rows of 4096, matrix cores busy 58%). 64 to 512 tokens, and pairs of 100: what every workgroup stages
// of tokens and rows, which passes from the L2s at 10 to 14 TB/s (256 tokens, 4096 rows of 4096: 155 MB
// in 12.0 us). Small tiles: the way of a stage's operands from
// LDS, with a wave a SIMD 0.4 us a stage, which the split of the reduction over 8 waves
// shares out: 64 tokens, 4096 rows of 4096, 7.3 us (18.4 in tiles of 64 x 64 without it,
// 12.5 with operands from memory). Few tokens: HBM, where all compute units have a
// tile, for which tiles have 16 rows: one token, 4096 rows of 14,336 12.1 us (4.9 TB/s), 16
// 13.5 (19.8 in tiles of 32 rows, on half of the units; 20.9 with operands from memory,
// of which a unit reads about 16 bytes a clock); of a pair of 14,336 rows of 4096 25.7 and 26.4 (28.4 in
// tiles of 32 rows of each).
typedef int v16i __attribute__((ext_vector_type(16)));

// 16 bytes a lane from base + off to LDS at `to` (one address a wave) + 16 lane.
// No register waits for it: a wait on the vector memory counter ends it. (The
// compiler does not see into it, so it holds the 5 clocks that a load waits for an
// address register which a vector instruction has written. m0 is
// reserved, which a clobber would not change, and no other instruction here takes it.)
__device__ __forceinline__ void i8_to_lds(unsigned to, const int8_t *base, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}
// all but the last N of this wave's loads have ended, and all waves are here
template <int N> __device__ __forceinline__ void i8_stage_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
template <int KC> __device__ __forceinline__ int i8_chunk(int row, int c) { return c ^ (KC == 8 ? (row >> 1) & 7 : row & 15); }

template <int BT_, int BR_, int WT_, int WR_, int BK_, int NB_, int WK_ = 1, int MB_ = 32> struct I8Tile {
    static constexpr int BT = BT_, BR = BR_, WT = WT_, WR = WR_, BK = BK_, NB = NB_, WK = WK_;
    static constexpr int MB = MB_;                                 // tokens and rows of a product, of G 16-byte chunks each
    static constexpr int G = 64 / MB, Q = MB * MB / 256;           // a product's values of a lane: Q times four
    static constexpr int WAVES = WT * WR * WK, T = 64 * WAVES, KC = BK / 16, MT = BT / WT / MB, NT = BR / WR / MB;
    static constexpr int PER = 64 / KC;                            // rows a wave's load covers
    static constexpr int LX = BT / PER / WAVES, LW = BR / PER / WAVES;   // loads a wave and stage
    static_assert(LX * PER * WAVES == BT && LW * PER * WAVES == BR && MB % PER == 0 && BK % (16 * G * WK) == 0, "whole loads");
};

// the schedule of P products with R reads spread evenly behind them
template <int P, int R, int I = 0> __device__ __forceinline__ void i8_schedule() {
    if constexpr (I < P) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr ((I + 1) * R / P > I * R / P) __builtin_amdgcn_sched_group_barrier(0x100, (I + 1) * R / P - I * R / P, 0);
        i8_schedule<P, R, I + 1>();
    }
}

template <class S, bool GLU> __global__ void __launch_bounds__(S::T) k_i8_tile(const I8Args a, int nt, int nr) {
    constexpr int KC = S::KC, BK = S::BK, NB = S::NB;
    constexpr int XB = S::BT * BK, WB = S::BR * BK;
    __shared__ alignas(16) int8_t s_ring[NB * (XB + WB)];
    int8_t *const s_x = s_ring, *const s_w = s_ring + NB * XB;
    constexpr int MB = S::MB;
    const int lane = threadIdx.x & 63, h = lane / MB, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // Consecutive workgroups go to the dies in turn: each die has consecutive tiles,
    // 8 token tiles of a row tile after one another, which share what its L2 holds
    const int all = nt * nr, q = all / 8, rem = all % 8, die = blockIdx.x % 8;
    const int l = die * q + min(die, rem) + (int)blockIdx.x / 8;
    const int band = l / (8 * nr) * 8, wide = min(8, nt - band), in = l - band * nr;
    const int t0 = (band + in % wide) * S::BT, r0 = in / wide * (GLU ? S::BR / 2 : S::BR);
    // where this lane's chunks of a stage are: byte offsets from the tile's first row
    const int8_t *xb = a.x + (size_t)t0 * a.ldx;
    const int8_t *w0 = a.w[0] + (size_t)r0 * a.ldw[0], *w1 = GLU ? a.w[1] + (size_t)r0 * a.ldw[1] : nullptr;
    unsigned xo[S::LX], wo[S::LW];
    const int sub = lane / KC, slot = lane % KC;
#pragma unroll
    for (int j = 0; j < S::LX; j++) {
        const int row = (j * S::WAVES + wave) * S::PER + sub;
        xo[j] = (unsigned)min(row, a.ntok - 1 - t0) * (unsigned)a.ldx + i8_chunk<KC>(row, slot) * 16;
    }
    auto second = [&](int j) { return GLU && ((j * S::WAVES + wave) * S::PER / MB & 1); };
    auto ldw = [&](int j) { return (unsigned)(second(j) ? a.ldw[1] : a.ldw[0]); };
    auto mrow = [&](int row) { return min(GLU ? row / (2 * MB) * MB + row % MB : row, a.rows - 1 - r0); };
#pragma unroll
    for (int j = 0; j < S::LW; j++) {
        const int row = (j * S::WAVES + wave) * S::PER + sub;
        wo[j] = (unsigned)mrow(row) * ldw(j) + i8_chunk<KC>(row, slot) * 16;
    }
    const unsigned lx = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t *)s_x;
    const unsigned lw = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t *)s_w;
    const int stages = (a.cols + BK - 1) / BK;
    auto load = [&](int st) {
        const int k = st * BK, buf = st % NB;
        const bool whole = k + BK <= a.cols;
#pragma unroll
        for (int j = 0; j < S::LX; j++) {
            const int g = j * S::WAVES + wave;
            unsigned off = xo[j];
            if (!whole) {   // past the row's stride: any of its values, which meet zeros
                const int c = i8_chunk<KC>(g * S::PER + sub, slot) * 16;
                if (k + c >= (int)a.ldx) off -= c;
            }
            i8_to_lds(lx + buf * XB + g * 1024, xb + k, off);
        }
#pragma unroll
        for (int j = 0; j < S::LW; j++) {
            const int g = j * S::WAVES + wave;
            unsigned off = wo[j];
            if (!whole) {
                const int c = i8_chunk<KC>(g * S::PER + sub, slot) * 16;
                if (k + c >= (int)ldw(j)) off -= c;
            }
            i8_to_lds(lw + buf * WB + g * 1024, (second(j) ? w1 : w0) + k, off);
        }
    };
    // zeros for what the last stage's rows of W have past their end, so that nothing there counts
    auto clear = [&](int st) {
        const int left = a.cols - st * BK;
        for (int i = threadIdx.x; i < S::BR * KC; i += S::T) {
            const int c = i8_chunk<KC>(i / KC, i % KC) * 16;
            v4i *p = (v4i *)(s_w + st % NB * WB + i * 16);
            if (c >= left) {
                *p = v4i{};
            } else if (c + 16 > left) {
                *p = i8_cut(*p, left - c);
            }
        }
        __syncthreads();
    };
    typedef std::conditional_t<MB == 32, v16i, v4i> Sum;
    Sum acc[S::MT][S::NT] = {};
    const int wk = wave / (S::WT * S::WR), wg = wave % (S::WT * S::WR), wt = wg / S::WR, wr = wg % S::WR, n = lane % MB;
    constexpr int KS = BK / (16 * S::G) / S::WK;   // steps of a stage, of which the wave's are wk * KS ..
    // Small tiles ask for a stage's operands at once, whose way from LDS would else
    // be most of a step; larger ones for the next step's among a step's products
    constexpr bool ALL = S::MT * S::NT <= 2 || S::WK > 1;
    constexpr int D = ALL ? KS : 2;
    v4i xv[D][S::MT], wv[D][S::NT];
    // a product's operands, step k of a stage
    auto read = [&](int st, int k, v4i (&x)[S::MT], v4i (&w)[S::NT]) {
        const int c = i8_chunk<KC>(n, S::G * (wk * KS + k) + h) * 16;
        const int8_t *sx = s_x + st % NB * XB + (wt * S::MT * MB + n) * BK + c;
        const int8_t *sw = s_w + st % NB * WB + (wr * S::NT * MB + n) * BK + c;
#pragma unroll
        for (int m = 0; m < S::MT; m++) x[m] = *(const v4i *)(sx + m * MB * BK);
#pragma unroll
        for (int m = 0; m < S::NT; m++) w[m] = *(const v4i *)(sw + m * MB * BK);
    };
    auto products = [&](const v4i (&x)[S::MT], const v4i (&w)[S::NT]) {
#pragma unroll
        for (int m = 0; m < S::MT; m++)
#pragma unroll
            for (int c = 0; c < S::NT; c++) {
                if constexpr (MB == 32) acc[m][c] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[m], w[c], acc[m][c], 0, 0, 0);
                else acc[m][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[m], w[c], acc[m][c], 0, 0, 0);
            }
    };
#pragma unroll
    for (int st = 0; st < NB - 1; st++)
        if (st < stages) load(st);
    const int cut = a.cols % BK ? stages - 1 : -1;
    for (int st = 0; st < stages; st++) {
        if (NB > 2 && st + NB - 2 < stages - 1) {
            i8_stage_wait<(NB - 2) * (S::LX + S::LW)>();
        } else {
            i8_stage_wait<0>();
        }
        if (st == cut) clear(cut);
        if (st + NB - 1 < stages) load(st + NB - 1);
        if constexpr (ALL) {
#pragma unroll
            for (int k = 0; k < KS; k++) read(st, k, xv[k], wv[k]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < KS; k++) products(xv[k], wv[k]);
        } else {
            read(st, 0, xv[0], wv[0]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if (k + 1 < KS) read(st, k + 1, xv[(k + 1) & 1], wv[(k + 1) & 1]);
                products(xv[k & 1], wv[k & 1]);
                i8_schedule<S::MT * S::NT, S::MT + S::NT>();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // value i of a tile is token (i & 3) + 8 (i >> 2) + 4 h, and row n
    constexpr int M = GLU ? 2 : 1;
    const bool whole = t0 + S::BT <= a.ntok && r0 + S::BR / M <= a.rows;
    // values i0 .. i0 + 3 of the token tile at tm, rows r + n
    auto quad = [&](int tm, int r, const float (&xd)[4], const v4i &s0, const v4i &s1, const float *wd, float bias) {
        float *y = a.y + (size_t)tm * a.ldy + r;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = i8_scaled(s0[i], xd[i], wd[0]);
            if constexpr (GLU) v[i] = i8_silu_mul(v[i], i8_scaled(s1[i], xd[i], wd[1]));
        }
        if (!GLU && a.bias) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = kr_fadd(v[i], bias);
        }
        auto live = [&](int i) { return whole || (r < a.rows && tm + i < a.ntok); };
        if (!GLU && a.add) {
            float old[4];
#pragma unroll
            for (int i = 0; i < 4; i++) old[i] = live(i) ? y[i * a.ldy] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = kr_fadd(old[i], v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (live(i)) y[i * a.ldy] = v[i];
    };
    int r[S::NT / M];
    float wd[S::NT / M][M], bias[S::NT / M];
#pragma unroll
    for (int c = 0; c < S::NT / M; c++) {
        r[c] = r0 + (wr * S::NT / M + c) * MB + n;
        const int at = min(r[c], a.rows - 1);
        wd[c][0] = a.wd[0][at];
        if constexpr (GLU) wd[c][1] = a.wd[1][at];
        bias[c] = !GLU && a.bias ? a.bias[at] : 0.0f;
    }
    auto part = [](const Sum &v, int q) { return v4i{ v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3] }; };
    auto tokens = [&](int m, int q) { return t0 + (wt * S::MT + m) * MB + 8 * q + 4 * h; };
    auto scales = [&](int tm, float (&xd)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) xd[i] = a.xd[min(tm + i, a.ntok - 1)];
    };
    if constexpr (S::WK == 1) {
#pragma unroll
        for (int m = 0; m < S::MT; m++) {
            float xd[S::Q][4];
#pragma unroll
            for (int q = 0; q < S::Q; q++) scales(tokens(m, q), xd[q]);
#pragma unroll
            for (int c = 0; c < S::NT / M; c++)
#pragma unroll
                for (int q = 0; q < S::Q; q++)
                    quad(tokens(m, q), r[c], xd[q], part(acc[m][c * M], q), part(acc[m][c * M + M - 1], q), wd[c], bias[c]);
        }
    } else {
        // the parts' sums meet in the ring, RM tiles at a time, and each wave has its share of the values
        constexpr int NC = S::NT / M, P = S::MT * NC, ROOM = NB * (XB + WB) / (S::WAVES * M * MB * MB * 4), RM = ROOM >= P ? P : ROOM >= 4 ? 4 : ROOM >= 2 ? 2 : 1;
        static_assert(ROOM > 0 && P % RM == 0, "the parts fit");
        v4i *const s_part = (v4i *)s_ring;
#pragma unroll
        for (int p0 = 0; p0 < P; p0 += RM) {
            __syncthreads();
#pragma unroll
            for (int p = 0; p < RM; p++)
#pragma unroll
                for (int q = 0; q < S::Q; q++)
#pragma unroll
                    for (int c = 0; c < M; c++)
                        s_part[(((wave * RM + p) * S::Q + q) * M + c) * 64 + lane] = part(acc[(p0 + p) / NC][(p0 + p) % NC * M + c], q);
            __syncthreads();
#pragma unroll
            for (int p = 0; p < RM; p++) {
                // quads of the tile in turn over the parts' waves
                for (int q = (wk - p * S::Q % S::WK + S::WK) % S::WK; q < S::Q; q += S::WK) {
                    float xd[4];
                    const int tm = tokens((p0 + p) / NC, q), cc = (p0 + p) % NC;
                    scales(tm, xd);
                    v4i sum[M] = {};
#pragma unroll
                    for (int k = 0; k < S::WK; k++)
#pragma unroll
                        for (int c = 0; c < M; c++)
                            sum[c] += s_part[(((k * S::WT * S::WR + wg) * RM + p) * S::Q + q) * M * 64 + c * 64 + lane];
                    quad(tm, r[cc], xd, sum[0], sum[M - 1], wd[cc], bias[cc]);
                }
            }
        }
    }
}

// The forms, and what they take: with n tiles a CU, base + n out + (n == 1 ? one : n many) cols / 4096
// us, as measured (288 to 16,384 rows of 288 to 16,384, 1 to 2047 tokens, and pairs of 300 to 20,000 rows of 300 to
// 8192: but for 2 of 160 sizes and 4 of 135 the form of the least estimate is within 7% of the fastest).
// At 4096 rows of 4096 in us, 16 x 16 / 32 x 16 / 32 x 32 / 64 x 32 / 64 x 64 / 128 x 64 / 128 x 128 split /
// whole / 256 x 256: 16 tokens 5.5 / 5.6 / 6.8 / 7.9 / 10.2 / -, 32 6.2 / 5.9 / 6.9 / 7.9 / 10.3 / 14.0 / 22.6 / 23.1 / -,
// 64 10.5 / 9.8 / 7.3 / 8.2 / 10.6 / 14.2 / 23.0 / 23.3 / 49.5, 256 - / 33.4 / 17.2 / 15.8 / 12.0 / 15.5 / 23.5 / 24.0 / 51,
// 512 - / - / 31.1 / 28.9 / 21.2 / 16.9 / 24.3 / 24.5 / 51, 2047 - / - / 112 / 103 / 70 / 57 / 49 / 39 / 56.
enum { I8_16x16, I8_32x32, I8_64x32, I8_64x64, I8_128x64, I8_128x128_SPLIT, I8_128x128, I8_256x256, I8_32x16, I8_FORMS };
struct I8Cost {
    int bt, br;
    float base, out, one, many;
};
constexpr I8Cost I8_COST[2][I8_FORMS] = {
    { { 16, 16, 1.9f, 0.6f, 2.2f, 1.9f }, { 32, 32, 2.3f, 1.0f, 4.2f, 3.0f }, { 64, 32, 2.8f, 1.2f, 5.0f, 5.0f },
      { 64, 64, 2.0f, 3.2f, 6.2f, 6.2f }, { 128, 64, 4.8f, 1.6f, 11, 11 }, { 128, 128, 7.0f, 1.2f, 19, 19 },
      { 128, 128, 4.0f, 0.2f, 23, 19.5f }, { 256, 256, 4.5f, 6.0f, 58, 58 }, { 32, 16, 1.7f, 1.4f, 2.4f, 2.9f } },
    // a pair: br rows of each matrix; no 64 x 64 but 64 x 32, and no 32 x 16
    { { 16, 16, 3.0f, 0.8f, 2.1f, 2.5f }, { 32, 32, 3.1f, 1.5f, 5.0f, 7.8f }, { 64, 32, 2.4f, 3.1f, 6.4f, 9.6f }, {},
      { 128, 32, 2.0f, 3.7f, 10.4f, 12.8f }, { 128, 64, 0.6f, 5.4f, 21.1f, 21.1f }, { 128, 64, 3.5f, 0.5f, 25.5f, 23.9f },
      { 256, 128, 5.0f, 5.6f, 47.9f, 64.5f }, {} }
};
int i8_form(int rows, int cols, int ntok, bool glu) {
    int best = I8_32x32;
    float least = FLT_MAX;
    for (int f = 0; f < I8_FORMS; f++) {
        const I8Cost &c = I8_COST[glu][f];
        if (c.bt == 0) continue;
        const double tiles = (double)((ntok + c.bt - 1) / c.bt) * ((rows + (long long)c.br - 1) / c.br);
        const float n = (float)ceil(tiles / 256), us = c.base + n * c.out + (n == 1 ? c.one : n * c.many) * (cols / 4096.0f);
        if (us < least) least = us, best = f;
    }
    return best;
}

// a launch holds 2^32 - 1 threads
template <class F, class... A> void i8_start(F f, const char *what, long long blocks, int threads, const A &...args) {
    if (blocks > UINT32_MAX / threads) {
        kr_fail(ML_E_SHAPE, what, hipSuccess);
        return;
    }
    hipLaunchKernelGGL(f, dim3((unsigned)blocks), dim3(threads), 0, kr_stream(), args...);
    kr_check_launch(what);
}
template <class S, bool GLU> void i8_tiles(const I8Args &a, const char *what) {
    const int nt = (a.ntok + S::BT - 1) / S::BT, nr = (a.rows + (GLU ? S::BR / 2 : S::BR) - 1) / (GLU ? S::BR / 2 : S::BR);
    i8_start(k_i8_tile<S, GLU>, what, (long long)nt * nr, S::T, a, nt, nr);
}

template <bool GLU> void i8_launch(const I8Args &a, const char *what) {
    constexpr int R = GLU ? 64 : 32;   // 32 rows of a matrix
    const int form = i8_form(a.rows, a.cols, a.ntok, GLU);
    switch (form) {
    // a pair's ring of three has two workgroups a CU: 8 tokens of 14,336 rows of 4096 25.7 us, of four 30.4
    case I8_16x16: return i8_tiles<I8Tile<16, GLU ? 32 : 16, 1, 1, 512, GLU ? 3 : 4, 8, 16>, GLU>(a, what);
    case I8_32x32: return i8_tiles<I8Tile<32, R, 1, 1, 256, 4, 8>, GLU>(a, what);
    case I8_64x32: return i8_tiles<I8Tile<64, R, 1, 1, 256, GLU ? 3 : 4, 8>, GLU>(a, what);
    case I8_128x64: return i8_tiles<I8Tile<128, 64, 2, 1, 256, 3, 4>, GLU>(a, what);
    case I8_128x128_SPLIT: return i8_tiles<I8Tile<128, 128, 2, 2, 128, 4, 2>, GLU>(a, what);
    case I8_128x128: return i8_tiles<I8Tile<128, 128, 4, 2, 128, 2>, GLU>(a, what);
    case I8_256x256: return i8_tiles<I8Tile<256, 256, 2, 4, 128, 2>, GLU>(a, what);
    default:
        if constexpr (!GLU) {
            if (form == I8_32x16) return i8_tiles<I8Tile<32, 16, 1, 1, 512, 4, 8, 16>, GLU>(a, what);
            return i8_tiles<I8Tile<64, 64, 1, 1, 256, 4, 8>, GLU>(a, what);
        }
    }
}

bool i8_refuse(bool ok, const char *what) {
    if (!ok) kr_fail(ML_E_SHAPE, what, hipSuccess);
    return !ok;
}
bool i8_not_ready(const char *what) {
    if (!kr_stream()) kr_fail(ML_E_ISA, what, hipSuccess);
    return !kr_stream();
}
bool i8_size_ok(int rows, int cols) { return rows > 0 && rows <= INT32_MAX - 1024 && cols > 0 && cols <= I8_COLS; }
bool i8_aligned(const void *p) { return !((uintptr_t)p & 15); }
bool i8_mat_ok(const krh_mat8 *w) {
    return w && w->q && w->d && i8_aligned(w->q) && i8_size_ok(w->rows, w->cols) && w->ld % 16 == 0 &&
           w->ld >= (size_t)w->cols && w->ld <= I8_LD;
}
bool i8_args_ok(const krh_mat8 *w, const float *y, size_t ldy, const int8_t *xq, size_t ldx, const float *xd) {
    return y && xq && xd && i8_aligned(xq) && ldy >= (size_t)w->rows && ldx % 16 == 0 && ldx >= (size_t)w->cols && ldx <= I8_LD;
}

}  // namespace

extern "C" int krh_matmul_i8_form(int rows, int cols, int ntok, int swiglu) {
    return i8_size_ok(rows, cols) && ntok > 0 && ntok <= KRH_ROWS_MAX ? i8_form(rows, cols, ntok, swiglu != 0) : -1;
}

extern "C" void krh_matmul_i8(float *Y, size_t ldy, const krh_mat8 *W, const int8_t *xq, size_t ldx, const float *xd,
                              const float *bias, int T, int accumulate) {
    if (i8_refuse(i8_mat_ok(W), "matmul_i8: the matrix") ||
        i8_refuse(T >= 0 && T <= KRH_ROWS_MAX, "matmul_i8 tokens"))
        return;
    if (T == 0) return;
    if (i8_refuse(i8_args_ok(W, Y, ldy, xq, ldx, xd), "matmul_i8: a missing or unaligned array, or row strides") ||
        i8_not_ready("matmul_i8 before krh_init"))
        return;
    const I8Args a = { Y, ldy, { W->q, nullptr }, { W->d, nullptr }, { W->ld, 0 }, xq, ldx, xd, bias, W->rows, W->cols, T,
                       accumulate != 0 };
    i8_launch<false>(a, "matmul_i8");
}

extern "C" void krh_matmul_i8_swiglu(float *H, size_t ldh, const krh_mat8 *w1, const krh_mat8 *w3, const int8_t *xq,
                                     size_t ldx, const float *xd, int T) {
    if (i8_refuse(i8_mat_ok(w1) && i8_mat_ok(w3) && w1->rows == w3->rows && w1->cols == w3->cols,
                  "matmul_i8_swiglu: the matrices") ||
        i8_refuse(T >= 0 && T <= KRH_ROWS_MAX, "matmul_i8_swiglu tokens"))
        return;
    if (T == 0) return;
    if (i8_refuse(i8_args_ok(w1, H, ldh, xq, ldx, xd), "matmul_i8_swiglu: a missing or unaligned array, or row strides") ||
        i8_not_ready("matmul_i8_swiglu before krh_init"))
        return;
    const I8Args a = { H, ldh, { w1->q, w3->q }, { w1->d, w3->d }, { w1->ld, w3->ld }, xq, ldx, xd, nullptr, w1->rows,
                       w1->cols, T, 0 };
    i8_launch<true>(a, "matmul_i8_swiglu");
}
