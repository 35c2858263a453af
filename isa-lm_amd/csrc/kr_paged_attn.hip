// Attention of one token of each sequence over a paged cache
// (krh_paged_attention).
//
// The rows of all sequences, in tiles of 32 (16), are cut into equal shares, one
// a wave and KV head (pa_bound): the lengths decide on the device, so a batch of
// all lengths loads the chip as one long sequence does. A wave passes over each
// sequence's part of its share once, with the running maximum and sum of the
// softmax. A sequence within one share is then done; the others' parts are
// joined by a second launch (k_paged_join), which finds them by the same
// arithmetic. Where all are short each is a share, and there is no second launch.
// (Joined by the last share to end instead, whose parts pass between the dies'
// caches: 20 to 40 us more with atomics that pass those caches, 60 to 90 with
// fences.)
//
// Both products run on the matrix cores, transposed so that nothing passes
// through LDS: S^T = K Q^T has the tile's rows as rows and query heads as
// columns, and the lane that holds a head's scores of 8 (4) consecutive rows
// holds them as the operand P^T of O^T = V^T P^T. K's rows are read straight into
// operand registers (the order of the contraction is free, so a lane reads 8
// dims at a time); V's are transposed 2 by 2 in registers by byte permutes (F32:
// none, a float is an operand by itself).
//
// The halves' products are exact in 32 bits, so a float operand is split in two
// halves, x = hi + lo with |x - hi - lo| <= 2^-22 |x|: the queries (scaled by a
// power of two a head) and the weights (times 2^15 after the power, which is exact:
// lo is a whole half down to 2^-17 of the largest weight, and below that weights
// err by up to 2^-40 of it). The products of both are in the same sums
// (hi and lo as columns of one product, for up to 8 query heads a KV head, took
// 1 to 4% more, for their exchange). int8 rows become halves exactly; their scale
// multiplies the score, or the weight. F32 caches take the 32-bit product, whose
// rate still passes what HBM delivers.
//
// Bound by HBM where the rows are many: 8B shape, F16, 64 sequences of up to 6144
// rows 123 us (5.5 TB/s; plain reads of 4 GB reach 5.3 to 6.5 by their grid), one of
// 120,001 rows 91 (5.4), 16 of up to 4001 24 (5.0). 8-bit rows by a tile's latency
// and instructions: 24 sequences of 64 dims 23 us (4.0).
#include <cfloat>
#include <type_traits>
#include "kr_paged_dev.h"

namespace {

// Rows of a tile: 32, and 16 for heads past 128 dims, whose rows fill the registers
constexpr int pa_tile(int hd) { return hd > 128 ? 16 : 32; }
constexpr int PA_UP = 15;   // the weights' scale (log2; halves end at 2^16)
// the least power of two that 8-bit rows' weights are over: the scale 0 of rows of
// zeros has one with it
constexpr int PA_EV = -80;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef unsigned uint2v __attribute__((ext_vector_type(2)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

struct PaArgs {
    float *o;
    const float *q;
    const int *len;
    float *mass;
    size_t mass_ld;
    float *part;    // [n_kv][n_seq + shares][group][hd]: a share's sums of a sequence, at their numbers' sum
    float *pml;     // [n_kv][n_seq + shares][group][2]: their maximum (log2) and weight
    float *z;       // [n_seq][nh][z_ld]: the scores (log2), for the mass
    size_t z_ld;
    int nh, max_len, window, shares;
    int whole, tl, least;     // whole: a share a sequence; tl: log2 of a tile's rows; least: tiles a share is worth
    float scale, cap;
};

// rows [first, len) of a sequence, in tiles from the one that holds `first`; a
// sequence of no rows has one tile, whose output is zeros
struct PaSpan {
    int len, first, begin, tiles;
};
__device__ __forceinline__ PaSpan pa_span(const PaArgs &a, int len) {   // len within [0, max_len]
    PaSpan r;
    r.len = len;
    r.first = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
    r.begin = r.first & -(1 << a.tl);
    r.tiles = max(1, (r.len - r.begin + (1 << a.tl) - 1) >> a.tl);
    return r;
}

// All sequences' tiles, and how many shares they make: share u has tiles
// [u T / n, (u + 1) T / n). With it the spans of 64 sequences, one a lane.
struct PaAll {
    int tiles, shares;
    int base, len, sum;   // the lanes' sequences from `base` on: lengths, inclusive sums of tiles
    int before;           // tiles of the sequences before `base`
};
__device__ __forceinline__ void pa_fetch(const PgView &p, const PaArgs &a, PaAll &r, int base, int &bad) {
    const int i = base + (int)(threadIdx.x & 63);
    r.base = base;
    r.len = i < p.n_seq ? kr_page_len(a.len[i], a.max_len, bad) : 0;
    r.sum = pg_scan(i < p.n_seq ? pa_span(a, r.len).tiles : 0);
}
__device__ __forceinline__ PaAll pa_all(const PgView &p, const PaArgs &a, int &bad) {
    PaAll r;
    int t = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += 64) {
        r.before = t;
        pa_fetch(p, a, r, i0, bad);
        t += __builtin_amdgcn_readlane(r.sum, 63);
    }
    r.tiles = t;
    r.shares = max(1, min(a.shares, (t + a.least - 1) / a.least));
    return r;
}
__device__ __forceinline__ int pa_len(const PgView &p, const PaArgs &a, PaAll &r, int s, int &bad) {
    if (s - r.base >= 64 || s < r.base) pa_fetch(p, a, r, s & ~63, bad);
    return __builtin_amdgcn_readlane(r.len, s - r.base);
}
// the sequence that holds tile t of all; t becomes the tile's number in it
__device__ __forceinline__ int pa_find(const PgView &p, const PaArgs &a, PaAll &r, int &t, int &bad) {
    if (t >= r.before) {
        t -= r.before;
    } else {
        pa_fetch(p, a, r, 0, bad);
    }
    for (;;) {
        const int all = __builtin_amdgcn_readlane(r.sum, 63);
        if (t < all) break;
        t -= all;
        pa_fetch(p, a, r, r.base + 64, bad);
    }
    const int n = __popcll(__ballot(r.sum <= t));
    if (n) t -= __builtin_amdgcn_readlane(r.sum, n - 1);
    return r.base + n;
}
__device__ __forceinline__ int pa_bound(const PaAll &all, int u) { return (int)((long long)all.tiles * u / all.shares); }
// the share that holds tile t
__device__ __forceinline__ int pa_share(const PaAll &all, int t) {
    return (int)((((long long)t + 1) * all.shares - 1) / all.tiles);
}

// tanh within 4 half steps of a float: below 0.6 x + x t P(t), t = x^2, P fitted to
// (tanh(x) / x - 1) / t for the least of the largest t |error|, 0.1 half steps; from
// there 1 - 2 / (e^2x + 1). (The C library's tanhf, which the token loop's
// soft-caps call, is three quotients: a float cache's 10,000 rows 168 us.)
__device__ __forceinline__ float pa_tanh(float x) {
    const float t = x * x, y = fabsf(x);
    float p = __builtin_fmaf(-0x1.830bfap-8f, t, 0x1.54e018p-6f);
    p = __builtin_fmaf(p, t, -0x1.b89edap-5f);
    p = __builtin_fmaf(p, t, 0x1.1109dcp-3f);
    p = __builtin_fmaf(p, t, -0x1.55553ep-2f);
    const float e = __builtin_amdgcn_exp2f(y * 2.8853900817779268f);
    const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return y < 0.6f ? __builtin_fmaf(x * t, p, x) : copysignf(far, x);
}
// over the 4 lanes of a column: both halves, then both rows of each, swapped in registers
__device__ __forceinline__ float pa_max_g(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pa_sum_g(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float4v pa_weigh(half8 v, half8 p, float4v o) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o, 0, 0, 0);
}
__device__ __forceinline__ float4v pa_weigh(half4 v, half4 p, float4v o) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(v, p, o, 0, 0, 0);
}

// halves of 4 int8 (xor 0x80: 0..255) as 1024 + u - 1152, exact
__device__ __forceinline__ unsigned pa_h2(unsigned u, unsigned sel) {
    const half2v h = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, sel));
    return __builtin_bit_cast(unsigned, h - half2v{ (_Float16)1152.0f, (_Float16)1152.0f });
}

// what a lane holds of a tile, as it lies in memory. K: per product step its
// NT rows 4 apart; V: W dims of each of its 4 NT rows.
template <int KT, int CL> struct PaRaw {
    static constexpr int W = CL / 16;                                  // dims a lane has of a V row
    static constexpr int KS = KT == PG_F32 ? CL / 16 : CL / 32;        // loads a K row
    static constexpr int KB = KT == PG_F32 ? 4 : KT == PG_F16 ? 4 : 2; // words a load
    static constexpr int VB = KT == PG_F32 ? W : KT == PG_F16 ? W / 2 : W / 4;
    static constexpr int NT = pa_tile(CL) / 16, R = 4 * NT;            // products a tile, V rows a lane
    unsigned k[NT][KS][KB], v[R][VB];
    float kd[KT == PG_Q8 ? R : 1], vd[KT == PG_Q8 ? R : 1];
};

template <int N> __device__ __forceinline__ void pa_load(unsigned (&x)[N], const void *p) {
    static_assert(N == 1 || N == 2 || N % 4 == 0, "whole loads");
    if constexpr (N == 1) {
        x[0] = *(const unsigned *)p;
    } else if constexpr (N == 2) {
        const uint2v t = *(const uint2v *)p;
        x[0] = t.x;
        x[1] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4v t = ((const uint4v *)p)[i / 4];
            x[i] = t.x;
            x[i + 1] = t.y;
            x[i + 2] = t.z;
            x[i + 3] = t.w;
        }
    }
}

// Whether two tiles' rows fit in registers: the next tile's are read while one
// is worked on; where they do not, its K rows are, once this tile's are used.
constexpr bool pa_two(int kt, int cl) { return cl <= (kt == PG_F32 ? 64 : 128) || kt == PG_Q8; }
constexpr int pa_waves(int kt, int cl) { return cl > (kt == PG_Q8 ? 128 : 64) ? 1 : 2; }   // a SIMD

template <int KT, int CL, bool FULL> struct PaWave {
    using Raw = PaRaw<KT, CL>;
    static constexpr int W = Raw::W, KS = Raw::KS, NT = Raw::NT, R = Raw::R, TILE = 16 * NT;
    static constexpr int EB = KT == PG_F32 ? 4 : KT == PG_F16 ? 2 : 1;
    static constexpr int KD = KT == PG_F32 ? 4 : 8;   // dims a K load
    static constexpr bool HALF = KT != PG_F32;

    const PgView &p;
    const PaArgs &a;
    static constexpr int NB = HALF ? 2 : 1;           // operands of the queries: hi and lo
    const int lane, n, g, kvh, hd, group;
    const bool live;   // whether this lane's column is a query head
    int seq, t_ids, bad;
    PaSpan sp;
    int ids;   // the pages of 64 half tiles from t_ids on, one a lane
    std::conditional_t<HALF, half8, float4v> qf[KS][NB];   // the queries as operands
    float cs, m_run, l_run;
    // Q8: the largest weight times V scale so far (of the maximum now); with o's
    // sums they are over 2^ev = v_end, which it is below
    float v_run, v_end;
    int ev;
    float4v o[W];

    __device__ __forceinline__ PaWave(const PgView &p_, const PaArgs &a_, int kvh_)
        : p(p_), a(a_), lane(threadIdx.x & 63), n(lane & 15), g(lane >> 4), kvh(kvh_), hd(FULL ? CL : p_.hd),
          group(a_.nh / p_.n_kv), live(n < group), bad(0) {}

    __device__ __forceinline__ size_t head() const { return (size_t)seq * a.nh + kvh * group + (live ? n : 0); }

    // the pages of the half tiles from row t0 on that have rows attended; -1 elsewhere
    __device__ __forceinline__ void find(int t0) {
        t_ids = t0;
        const int r = t0 + 16 * lane;
        ids = r + 16 > sp.first && r < sp.len ? pg_page(p, seq, r, bad) : -1;
    }
    // pool rows of the halves of the tile at t0; a half without rows attended takes the other's
    __device__ __forceinline__ void rows_of(int t0, size_t &lo, size_t &hi) {
        const int i = (t0 - t_ids) >> 4, pl = __builtin_amdgcn_readlane(ids, i);
        if constexpr (NT == 1) {
            lo = hi = kr_page_row(pl, p.n_kv, kvh, p.shift, t0);
        } else {
            const int ph = __builtin_amdgcn_readlane(ids, i + 1);
            lo = kr_page_row(pl >= 0 ? pl : ph, p.n_kv, kvh, p.shift, t0);
            hi = kr_page_row(ph >= 0 ? ph : pl, p.n_kv, kvh, p.shift, t0 + 16);
        }
    }

    // the queries as operands
    __device__ __forceinline__ void queries() {
        const float *q = a.q + head() * hd;
        int e = 0;
        if constexpr (HALF) {
            float x[KS][8], m = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = j * 32 + g * 8;
                const bool in = live && (FULL || d < hd);
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4v t = in ? *(const float4v *)(q + d + i) : float4v{ 0, 0, 0, 0 };
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        x[j][i + c] = t[c];
                        m = fmaxf(m, fabsf(t[c]));
                    }
                }
            }
            m = pa_max_g(m);
            if (m > 0.0f && m < INFINITY) e = 13 - ilogbf(m);
#pragma unroll
            for (int j = 0; j < KS; j++) {
                half8 h, l;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = ldexpf(x[j][i], e);
                    h[i] = (_Float16)y;
                    l[i] = (_Float16)(y - (float)h[i]);
                }
                qf[j][0] = h;
                qf[j][1] = l;
            }
        } else {
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = j * 16 + g * 4;
                const float4v t = live && (FULL || d < hd) ? *(const float4v *)(q + d) : float4v{ 0, 0, 0, 0 };
                qf[j][0] = t;
            }
        }
        // a product's factor: the scale, in log2 unless the cap comes first
        cs = ldexpf(a.cap > 0.0f ? a.scale : a.scale * 1.4426950408889634f, -e);
    }

    // this lane's K rows of a tile are R (n / 4) + n % 4 and 4 after it
    __device__ __forceinline__ void load_k(Raw &raw, size_t lo, size_t hi) const {
        const int r0 = R * (n >> 2) + (n & 3);
        const size_t r = NT == 1 || r0 < 16 ? lo + r0 : hi + (r0 - 16);
#pragma unroll
        for (int b = 0; b < NT; b++) {
            const char *at = (const char *)p.k + (r + 4 * b) * hd * EB;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                // past the head's dims the queries are zero: its first dims again
                const int d = (j * 4 + g) * KD;
                pa_load(raw.k[b][j], at + (FULL || d < hd ? d : 0) * EB);
            }
        }
    }
    // its V rows R g .. R g + R - 1, dims n W ..
    __device__ __forceinline__ void load_v(Raw &raw, size_t lo, size_t hi) const {
        const int r0 = R * g;
        const size_t r = NT == 1 || r0 < 16 ? lo + r0 : hi + (r0 - 16);
        if constexpr (KT == PG_Q8) {
#pragma unroll
            for (int i = 0; i < R; i += 4) {
                const float4v x = *(const float4v *)(p.kd + r + i), y = *(const float4v *)(p.vd + r + i);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    raw.kd[i + c] = x[c];
                    raw.vd[i + c] = y[c];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const char *at = (const char *)p.v + (r + i) * hd * EB;
            if constexpr (FULL) {
                pa_load(raw.v[i], at + n * W * EB);
            } else {
                // 4 dims at a time where a lane has them, else 8 (head_dim is a
                // multiple of 8); past the head's dims any, of outputs that are not stored
                constexpr int P = W < 8 ? W : 8, PW = P * EB / 4;
#pragma unroll
                for (int d = 0; d < W; d += P) {
                    unsigned x[PW];
                    pa_load(x, at + (n * W + d < hd ? n * W + d : 0) * EB);
#pragma unroll
                    for (int w = 0; w < PW; w++) raw.v[i][d * EB / 4 + w] = x[w];
                }
            }
        }
    }

    // products of the tile's rows R g + i with query head n
    __device__ __forceinline__ void scores(const Raw &raw, float (&sc)[R]) const {
#pragma unroll
        for (int b = 0; b < NT; b++) {
            float4v acc = { 0, 0, 0, 0 };
#pragma unroll
            for (int j = 0; j < KS; j++) {
                if constexpr (HALF) {
                    uint4v w;
                    if constexpr (KT == PG_F16) {
                        w = uint4v{ raw.k[b][j][0], raw.k[b][j][1], raw.k[b][j][2], raw.k[b][j][3] };
                    } else {
                        const unsigned x = raw.k[b][j][0] ^ 0x80808080u, y = raw.k[b][j][1] ^ 0x80808080u;
                        w = uint4v{ pa_h2(x, 0x04010400), pa_h2(x, 0x04030402), pa_h2(y, 0x04010400), pa_h2(y, 0x04030402) };
                    }
#pragma unroll
                    for (int x = 0; x < NB; x++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w), qf[j][x], acc, 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.k[b][j][c]), qf[j][0][c], acc, 0,
                                                                   0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) sc[4 * b + i] = acc[i];
        }
    }

    // the softmax's step over the tile at t0, then its V rows by their weights
    __device__ __forceinline__ void rest(Raw &raw, float (&sc)[R], int t0) {
        const bool whole = t0 >= sp.first && t0 + TILE <= sp.len;
        const int r0 = t0 + R * g;
        float m_tile = -INFINITY;
#pragma unroll
        for (int i = 0; i < R; i++) sc[i] *= KT == PG_Q8 ? cs * raw.kd[i] : cs;
        if (a.cap > 0.0f) {
            const float inv_cap = 1.0f / a.cap;
#pragma unroll
            for (int i = 0; i < R; i++) sc[i] = pa_tanh(sc[i] * inv_cap) * (a.cap * 1.4426950408889634f);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < R; i++) {
                const bool in = r0 + i >= sp.first && r0 + i < sp.len;
                sc[i] = in ? sc[i] : -INFINITY;
                // rows that are not attended may hold anything
                if constexpr (KT == PG_Q8) {
                    raw.vd[i] = in ? raw.vd[i] : 0.0f;
                } else {
#pragma unroll
                    for (int w = 0; w < Raw::VB; w++) raw.v[i][w] = in ? raw.v[i][w] : 0u;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) m_tile = fmaxf(m_tile, sc[i]);
        if (a.z && live) {
            float *z = a.z + head() * a.z_ld + r0;
#pragma unroll
            for (int i = 0; i < R; i += 4) *(float4v *)(z + i) = float4v{ sc[i], sc[i + 1], sc[i + 2], sc[i + 3] };
        }
        // the maximum, one for a column's four lanes, moves where a lane has a larger score
        const bool moved = __any(m_tile > m_run);
        float f = 1.0f;
        if (moved) {
            const float m_new = fmaxf(m_run, pa_max_g(m_tile));
            f = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= f;
        }
        // weights of no finite maximum: 0 for -inf, NaN for NaN
        const float base = m_run == -INFINITY ? 0.0f : m_run;
        float v_tile = 0.0f;
#pragma unroll
        for (int i = 0; i < R; i++) {
            sc[i] = __builtin_amdgcn_exp2f(sc[i] - base);
            l_run += sc[i];
            if constexpr (KT == PG_Q8) {
                // a rounded product: left to itself the compiler rounds it to a
                // half twice, once from the exact product, and at a tie the hi
                // that is multiplied is not the one taken off for lo
                sc[i] *= raw.vd[i];
                asm("" : "+v"(sc[i]));
                v_tile = fmaxf(v_tile, fabsf(sc[i]));
            }
        }
        // 8-bit rows' weights carry their V scales, and what both are over to end in
        // halves goes by their product: a large scale without weight moves nothing,
        // and it comes down again with the weights of an earlier maximum
        if constexpr (KT == PG_Q8) {
            if (moved || __any(v_tile >= v_end)) {
                v_run = fmaxf(v_run * f, pa_max_g(v_tile));
                const int e = max(PA_EV, (int)(__float_as_uint(v_run) >> 23) - 126);   // v_run < 2^e
                f = ldexpf(f, ev - e);
                ev = e;
                v_end = ldexpf(1.0f, e);
#pragma unroll
                for (int c = 0; c < W; c++) o[c] *= f;
            }
        } else if (moved) {
#pragma unroll
            for (int c = 0; c < W; c++) o[c] *= f;
        }
        const float up = KT == PG_Q8 ? ldexpf(1.0f, PA_UP - ev) : (float)(1 << PA_UP);
        // the weights as operands: R halves, or floats
        typedef _Float16 halfr __attribute__((ext_vector_type(R)));
        typedef unsigned uintr __attribute__((ext_vector_type(R / 2)));
        halfr ph[2];
        float pf[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            float x = sc[i];
            if constexpr (HALF) {
                x *= up;
                const _Float16 hi = (_Float16)x;
                ph[0][i] = hi;
                ph[1][i] = (_Float16)(x - (float)hi);
            } else {
                pf[i] = x;
            }
        }
        if constexpr (KT == PG_F32) {
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int c = 0; c < W; c++)
                    o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.v[i][c]), pf[i], o[c], 0, 0, 0);
        } else if constexpr (KT == PG_F16) {
#pragma unroll
            for (int c = 0; c < W; c++) {
                uintr w;
#pragma unroll
                for (int i = 0; i < R / 2; i++)
                    w[i] = __builtin_amdgcn_perm(raw.v[2 * i + 1][c / 2], raw.v[2 * i][c / 2],
                                                 c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int x = 0; x < 2; x++) o[c] = pa_weigh(__builtin_bit_cast(halfr, w), ph[x], o[c]);
            }
        } else {
#pragma unroll
            for (int c4 = 0; c4 < W; c4 += 4) {
                uintr w[4];
#pragma unroll
                for (int i = 0; i < R / 2; i++) {
                    const unsigned x = raw.v[2 * i][c4 / 4] ^ 0x80808080u, y = raw.v[2 * i + 1][c4 / 4] ^ 0x80808080u;
                    const unsigned u = __builtin_amdgcn_perm(y, x, 0x05010400u);
                    const unsigned v = __builtin_amdgcn_perm(y, x, 0x07030602u);
                    w[0][i] = pa_h2(u, 0x04010400);
                    w[1][i] = pa_h2(u, 0x04030402);
                    w[2][i] = pa_h2(v, 0x04010400);
                    w[3][i] = pa_h2(v, 0x04030402);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
#pragma unroll
                    for (int x = 0; x < 2; x++) o[c4 + c] = pa_weigh(__builtin_bit_cast(halfr, w[c]), ph[x], o[c4 + c]);
                }
            }
        }
    }

    __device__ __forceinline__ void load(Raw &raw, int t0) {
        size_t lo, hi;
        rows_of(t0, lo, hi);
        load_k(raw, lo, hi);
        load_v(raw, lo, hi);
    }

    // rows [t0, t1) of the sequence, whole tiles but at its end: at most 64 half
    // tiles, whose pages are in ids. The first rows are asked for before the queries
    // are. The rows ahead are asked for without a condition, the last tile's once
    // more at the end: behind a branch the compiler could not tell them from this
    // tile's loads in its waits.
    __device__ __forceinline__ void pass(int t0, int t1, bool begin) {
        float sc[R];
        const int last = t0 + (t1 - t0 - 1) / TILE * TILE;
        if constexpr (pa_two(KT, CL)) {
            Raw x, y;
            load(x, t0);
            if (begin) queries();
            for (;;) {
                load(y, min(t0 + TILE, last));
                scores(x, sc);
                rest(x, sc, t0);
                t0 += TILE;
                if (t0 > last) break;
                load(x, min(t0 + TILE, last));
                scores(y, sc);
                rest(y, sc, t0);
                t0 += TILE;
                if (t0 > last) break;
            }
        } else {
            Raw x;
            size_t lo, hi;
            rows_of(t0, lo, hi);
            load_k(x, lo, hi);
            if (begin) queries();
            for (;;) {
                load_v(x, lo, hi);
                scores(x, sc);
                rows_of(min(t0 + TILE, last), lo, hi);
                load_k(x, lo, hi);
                rest(x, sc, t0);
                t0 += TILE;
                if (t0 > last) break;
            }
        }
    }

    // tiles [t, end) of sequence `seq`, then its output or this share's part of it
    __device__ __forceinline__ void part(int t, int end, size_t slot) {
        m_run = -INFINITY;
        l_run = 0.0f;
        ev = PA_EV;
        v_run = v_end = 0.0f;
#pragma unroll
        for (int c = 0; c < W; c++) o[c] = float4v{ 0, 0, 0, 0 };
        const bool alone = t == 0 && end == sp.tiles;
        if (sp.len > 0) {
            const int r1 = min(sp.len, sp.begin + end * TILE);
            const int r0 = sp.begin + t * TILE;
            for (int r = r0; r < r1; r += (64 / NT) * TILE) {
                find(r);
                pass(r, min(r1, r + (64 / NT) * TILE), r == r0);
            }
        }
        const float l = pa_sum_g(l_run);
        float f = alone ? 1.0f / l : 1.0f;
        if constexpr (HALF) f = ldexpf(f, KT == PG_Q8 ? ev - PA_UP : -PA_UP);
        if (sp.len == 0) f = 0.0f;
        if (g == 0 && live && (!alone || a.z)) {
            *(float2v *)(a.pml + (slot * group + n) * 2) = float2v{ m_run, l };
        }
        float *out = alone ? a.o + head() * hd : a.part + (slot * group + n) * hd;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d0 = (4 * g + i) * W;
#pragma unroll
            for (int c = 0; c < W; c += 4)
                if (live && (FULL || d0 + c < hd))
                    *(float4v *)(out + d0 + c) = float4v{ o[c][i] * f, o[c + 1][i] * f, o[c + 2][i] * f, o[c + 3][i] * f };
        }
    }
};

template <int KT, int CL, bool FULL>
__global__ void __launch_bounds__(64, pa_waves(KT, CL)) k_paged_shares(const PgView p, const PaArgs a, int *fault) {
    const int u = blockIdx.x, kvh = blockIdx.y;
    PaWave<KT, CL, FULL> w(p, a, kvh);
    if (a.whole) {
        w.seq = u;
        w.sp = pa_span(a, kr_page_len(a.len[u], a.max_len, w.bad));
        w.part(0, w.sp.tiles, 0);
        kr_report(fault, w.bad);
        return;
    }
    PaAll all = pa_all(p, a, w.bad);
    if (u < all.shares) {
        int left = pa_bound(all, u + 1) - pa_bound(all, u), t = pa_bound(all, u);
        for (w.seq = pa_find(p, a, all, t, w.bad); left > 0; w.seq++, t = 0) {
            w.sp = pa_span(a, pa_len(p, a, all, w.seq, w.bad));
            const int end = min(w.sp.tiles, t + left);
            w.part(t, end, (size_t)kvh * (p.n_seq + a.shares) + w.seq + u);
            left -= end - t;
        }
    }
    kr_report(fault, w.bad);
}

// The shares of a sequence: their first slot and number, by the arithmetic that made them.
struct PaParts {
    size_t slot;
    int n;
};
__device__ __forceinline__ PaParts pa_parts(const PgView &p, const PaArgs &a, int s, int kvh, PaSpan &sp) {
    int bad = 0;   // reported by the shares
    PaAll all = pa_all(p, a, bad);
    int before = 0;
    for (int i = threadIdx.x & 63; i < (s & ~63); i += 64) before += pa_span(a, kr_page_len(a.len[i], a.max_len, bad)).tiles;
    for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o);
    sp = pa_span(a, pa_len(p, a, all, s, bad));
    const int end = __builtin_amdgcn_readfirstlane(before) + __builtin_amdgcn_readlane(all.sum, s - all.base);
    const int u0 = pa_share(all, end - sp.tiles), u1 = pa_share(all, end - 1);
    return { (size_t)kvh * (p.n_seq + a.shares) + s + u0, u1 - u0 + 1 };
}

// A head's maximum and 1 / its sum, by one wave
__device__ __forceinline__ void pa_stats(const float *ml, int group, int n, float &m, float &inv) {
    const int lane = threadIdx.x & 63;
    auto get = [&](int i) { return i < n ? *(const float2v *)(ml + (size_t)i * group * 2) : float2v{ -INFINITY, 0.0f }; };
    const float2v own = get(lane);   // up to 64 parts are read once
    m = own.x;
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, get(i).x);
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    float l = lane < n ? own.y * __builtin_amdgcn_exp2f(own.x - m) : 0.0f;
    for (int i = lane + 64; i < n; i += 64) {
        const float2v x = get(i);
        l += x.y * __builtin_amdgcn_exp2f(x.x - m);
    }
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
    inv = 1.0f / l;
}

// Workgroups x < nh: head x's parts (2^dl lanes hold its dims four at a time, the
// workgroup's other factor the parts side by side). The others, with a mass:
// PJ_ROWS rows of one KV head each, mass[r] += its weights over the query heads.
constexpr int PJ_T = 256, PJ_ROWS = 1024, PJ_U = 4;
__global__ void __launch_bounds__(PJ_T) k_paged_join(const PgView p, const PaArgs a, int dl, int blocks) {
    __shared__ float4v s_o[PJ_T];
    __shared__ float s_m[KR_PAGE_GROUP_MAX], s_i[KR_PAGE_GROUP_MAX];
    const int s = blockIdx.y, x = blockIdx.x, tid = threadIdx.x, group = a.nh / p.n_kv;
    PaSpan sp;
    if (x < a.nh) {
        const int kvh = x / group, col = x % group;
        const PaParts r = pa_parts(p, a, s, kvh, sp);
        if (r.n <= 1) return;
        const float *ml = a.pml + (r.slot * group + col) * 2, *part = a.part + (r.slot * group + col) * p.hd;
        const int l = tid & ((1 << dl) - 1), lanes = PJ_T >> dl, d = 4 * l < p.hd ? 4 * l : 0, i0 = tid >> dl;
        // the first parts are under way while their weights are found
        float4v v[PJ_U];
        float w[PJ_U];
#pragma unroll
        for (int k = 0; k < PJ_U; k++) {
            const int i = min(i0 + k * lanes, r.n - 1);
            v[k] = *(const float4v *)(part + (size_t)i * group * p.hd + d);
            w[k] = ml[(size_t)i * group * 2];
        }
        float m, inv;
        pa_stats(ml, group, r.n, m, inv);
        float4v acc = { 0, 0, 0, 0 };
        for (int k0 = 0;;) {
#pragma unroll
            for (int k = 0; k < PJ_U; k++)
                if (i0 + (k0 + k) * lanes < r.n) acc += v[k] * __builtin_amdgcn_exp2f(w[k] - m);
            k0 += PJ_U;
            if (i0 + k0 * lanes >= r.n) break;
#pragma unroll
            for (int k = 0; k < PJ_U; k++) {
                const int i = min(i0 + (k0 + k) * lanes, r.n - 1);
                v[k] = *(const float4v *)(part + (size_t)i * group * p.hd + d);
                w[k] = ml[(size_t)i * group * 2];
            }
        }
        s_o[tid] = acc;
        for (int h = lanes >> 1; h >= 1; h >>= 1) {
            __syncthreads();
            if ((tid >> dl) < h) s_o[tid] = acc = acc + s_o[tid + (h << dl)];
        }
        if (tid >> dl == 0 && 4 * l < p.hd) *(float4v *)(a.o + ((size_t)s * a.nh + x) * p.hd + d) = acc * inv;
        return;
    }
    const int kvh = (x - a.nh) / blocks, block = (x - a.nh) % blocks;
    const PaParts r = pa_parts(p, a, s, kvh, sp);
    const int r0 = sp.first + block * PJ_ROWS;
    if (r0 >= sp.len) return;
    const float *z = a.z + ((size_t)s * a.nh + kvh * group) * a.z_ld;
    float *mass = a.mass + ((size_t)s * p.n_kv + kvh) * a.mass_ld;
    // the first heads' scores are under way while the maxima are found
    constexpr int K = PJ_ROWS / PJ_T;
    float sum[K], old[K], zs[PJ_U][K];
    int at[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        at[k] = min(r0 + k * PJ_T + tid, sp.len - 1);
        sum[k] = 0.0f;
        old[k] = mass[at[k]];
#pragma unroll
        for (int h = 0; h < PJ_U; h++) zs[h][k] = h < group ? z[h * a.z_ld + at[k]] : 0.0f;
    }
    for (int h = tid >> 6; h < group; h += PJ_T / 64) {
        float m, inv;
        pa_stats(a.pml + (r.slot * group + h) * 2, group, r.n, m, inv);
        if ((tid & 63) == 0) {
            s_m[h] = m;
            s_i[h] = inv;
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < PJ_U; h++)
        if (h < group) {
            const float m = s_m[h], inv = s_i[h];
#pragma unroll
            for (int k = 0; k < K; k++) sum[k] += __builtin_amdgcn_exp2f(zs[h][k] - m) * inv;
        }
    for (int h = PJ_U; h < group; h++) {
        const float m = s_m[h], inv = s_i[h];
#pragma unroll
        for (int k = 0; k < K; k++) sum[k] += __builtin_amdgcn_exp2f(z[h * a.z_ld + at[k]] - m) * inv;
    }
#pragma unroll
    for (int k = 0; k < K; k++)
        if (r0 + k * PJ_T + tid < sp.len) mass[at[k]] = old[k] + sum[k];
}

// Shares in all, of every KV head: three waves a CU, which have the next tile's
// rows under way, keep HBM busy. 8-bit rows, which take a tile's work to read half
// as much, have four, and twelve up to 64 dims (measured at 64; the kernel of narrower
// heads has eight resident). Fewer where the rows are few: a
// share is worth PA_BYTES of K and V at least (halves: twice that). The lengths
// are the device's, so this is what they may be at most.
// Measured from HBM (us, 2 / 3 / 4 / 8 / 12 waves a CU): 8B shape, halves, 16
// sequences 32.8 / 32.8 / 33.0 / 37.6 / 40.5, 64 129.6 / 129.5 / 132.8 / 136.0 / 140.5,
// one of 120,001 rows 91.7 / 92.0 / 94.8 / 101.6 / 108.3; 8 bits, 24 sequences of 64 dims
// 46.0 / 36.9 / 32.0 / 30.4 / 30.6 and with the mass 57.6 / 47.2 / 49.3 / 46.2 / 42.9,
// 16 of 128 dims 34.0 / 29.7 / 29.2 / 33.2 / 36.7.
// 16 / 32 KB: halves, one sequence of 4000 rows 14.6 / 12.4; floats of 48 dims, 8
// of up to 250 9.8 / 11.6; 8 bits of 48 dims, 16 of up to 8000 17.4 / 19.8.
// PA_CUS is a constant so that a workspace has one size before and after krh_init.
constexpr int PA_CUS = 256, PA_BYTES = 16 * 1024;
int pa_least(const krh_pages *kv) {
    const bool f16 = kv->kv_type == ML_F16;
    const int tile = 2 * pa_tile(kv->head_dim) * kv->head_dim * (f16 ? 2 : kv->kv_type == ML_F32 ? 4 : 1);
    const int bytes = f16 ? 2 * PA_BYTES : PA_BYTES;
    return tile < bytes ? bytes / tile : 1;
}
int pa_shares(const krh_pages *kv, int n_seq, int rows) {
    const long long tile = pa_tile(kv->head_dim), tiles = n_seq * ((rows + tile - 1) / tile), least = pa_least(kv);
    const int waves = PA_CUS * (kv->kv_type != ML_Q8_0 ? 3 : kv->head_dim > 64 ? 4 : 12);
    const long long most = (tiles + least - 1) / least, want = waves / kv->n_kv_heads;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

// Rows up to which a sequence is one wave's, a KV head, and there is no second
// launch (it is not known how many of them are used, and the mass takes the launch
// anyway). About 0.7 us a tile of halves or 8 bits of 128 dims, twice that for
// floats of 64, against the join's 4 to 10 us, the more the more sequences. Measured
// (us, shares / whole): 8B shape, halves, one sequence of 256 rows 10.2 / 9.9, of 384
// 10.2 / 12.9, 64 of up to 512 25.8 / 18.7; 8 bits of 64 dims, 256 rows 11.3 / 9.3,
// 384 11.3 / 12.3; floats of 48 dims, 128 rows 9.5 / 8.5, 192 9.4 / 11.0; halves of
// 256 dims, 128 rows, 1 and 8 sequences 10.6 / 11.3 and 13.0 / 11.1.
constexpr int PA_WHOLE = 256, PA_WHOLE_MANY = 128;
int pa_whole(const krh_pages *kv, int n_seq) {
    const int rows =
        PA_WHOLE * 128 / ((kv->head_dim <= 128 ? 128 : 256) * (kv->kv_type != ML_F32 ? 1 : kv->head_dim <= 64 ? 2 : 4));
    return (long long)n_seq * kv->n_kv_heads >= PA_WHOLE_MANY ? 2 * rows : rows;
}

// the workspace's pieces, in floats
struct PaSizes {
    size_t part, pml, z_ld, z;
};
PaSizes pa_sizes(const krh_pages *kv, int n_seq, int nh, int max_len, int shares, bool mass) {
    PaSizes r;
    const size_t slots = (size_t)kv->n_kv_heads * (n_seq + shares) * (nh / kv->n_kv_heads);
    r.part = shares > 1 ? slots * kv->head_dim : 0;
    r.pml = shares > 1 || mass ? (slots * 2 + 3) & ~(size_t)3 : 0;
    r.z_ld = mass ? ((size_t)max_len + 31) / 32 * 32 : 0;
    r.z = (size_t)n_seq * nh * r.z_ld;
    return r;
}

bool pa_args_ok(const krh_pages *kv, int n_seq, int n_heads, int max_len) {
    return pg_pages_ok(kv) && n_seq > 0 && n_seq <= KRH_ROWS_MAX && max_len > 0 && max_len <= KR_PAGE_LEN_MAX &&
           (long long)n_seq * (max_len / 16 + 1) <= INT32_MAX / 2 && n_heads > 0 &&
           n_heads % kv->n_kv_heads == 0 && n_heads / kv->n_kv_heads <= KR_PAGE_GROUP_MAX;
}

using PaKernel = void (*)(const PgView, const PaArgs, int *);

// Heads take the next width of 64, 128 and 256 dims; a kernel of its own has them
// where they fill it (without, halves take 0 to 2% more, 8 bits 0 to 6, floats 1 and of
// 256 dims 7).
template <int KT, int CL> PaKernel pa_kernel(int hd) {
    return hd == CL ? k_paged_shares<KT, CL, true> : k_paged_shares<KT, CL, false>;
}
template <int KT> PaKernel pa_kernel(int hd) {
    return hd <= 64 ? pa_kernel<KT, 64>(hd) : hd <= 128 ? pa_kernel<KT, 128>(hd) : pa_kernel<KT, 256>(hd);
}

}  // namespace

extern "C" size_t krh_paged_attention_ws(const krh_pages *kv, int n_seq, int n_heads, int max_len, int mass) {
    if (!pa_args_ok(kv, n_seq, n_heads, max_len)) return 0;
    const PaSizes r = pa_sizes(kv, n_seq, n_heads, max_len, pa_shares(kv, n_seq, max_len), mass != 0);
    return sizeof(float) * (r.part + r.pml + r.z + 4);
}

extern "C" void krh_paged_attention(float *o, const krh_pages *kv, const int *table, int table_ld, const int *len,
                                    int n_seq, const float *q, int n_heads, int max_len, int window, float scale,
                                    float softcap, float *mass, size_t mass_ld, void *ws) {
    if (n_seq == 0) return;
    if (pg_refuse(pa_args_ok(kv, n_seq, n_heads, max_len), "paged_attention sizes") ||
        pg_refuse(o && table && table_ld > 0 && len && q && ws && pg_aligned(o) && pg_aligned(q) && pg_aligned(ws),
                  "paged_attention: a missing or unaligned array") ||
        // a soft-cap that is a normal float with its reciprocal and its log2 e times
        pg_refuse(window >= 0 && (softcap == 0.0f || (softcap >= FLT_MIN && softcap <= 0x1p126f)) &&
                      (!mass || mass_ld >= (size_t)max_len),
                  "paged_attention: window, soft-cap or mass rows"))
        return;
    if (pg_not_ready("paged_attention before krh_init")) return;
    // a window's rows, and those before them in its first tile
    const int rows = window > 0 && window < max_len - 32 ? window + 31 : max_len;
    const bool whole = !mass && rows <= pa_whole(kv, n_seq);
    const int shares = whole ? n_seq : pa_shares(kv, n_seq, rows);
    const PaSizes r = pa_sizes(kv, n_seq, n_heads, max_len, whole ? 1 : shares, mass != nullptr);
    const int blocks = mass ? (rows + PJ_ROWS - 1) / PJ_ROWS : 0;
    if (pg_refuse(n_heads + (long long)kv->n_kv_heads * blocks <= INT32_MAX / PJ_T,
                  "paged_attention: too many rows for a mass"))
        return;
    float *w = (float *)ws;
    PaArgs a = {};
    a.o = o, a.q = q, a.len = len, a.mass = mass, a.mass_ld = mass_ld;
    a.part = w, a.pml = w + r.part, a.z = mass ? w + r.part + r.pml : nullptr, a.z_ld = r.z_ld;
    a.nh = n_heads, a.max_len = max_len, a.window = window, a.shares = shares, a.least = pa_least(kv);
    a.tl = pg_log2(pa_tile(kv->head_dim));
    a.whole = whole;
    a.scale = scale, a.cap = softcap;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const int hd = kv->head_dim;
    const PaKernel f = kv->kv_type == ML_F32 ? pa_kernel<PG_F32>(hd) : kv->kv_type == ML_F16 ? pa_kernel<PG_F16>(hd)
                                                                                                    : pa_kernel<PG_Q8>(hd);
    hipLaunchKernelGGL(f, dim3(shares, kv->n_kv_heads), dim3(64), 0, kr_stream(), p, a, kr_fault_word());
    kr_check_launch("paged_attention");
    if ((shares > 1 && !whole) || mass) {
        hipLaunchKernelGGL(k_paged_join, dim3(n_heads + kv->n_kv_heads * blocks, n_seq), dim3(PJ_T), 0, kr_stream(), p, a,
                           pg_log2(hd / 4), blocks);
        kr_check_launch("paged_attention");
    }
}
