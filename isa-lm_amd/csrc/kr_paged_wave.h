// One wave's pass over a share of several sequences' paged rows, and the shares'
// arithmetic: what the attention of one token of each sequence consists of
// (kr_paged_attn.hip says how its products run). The attention over shared rows
// passes over the rows that are a sequence's own with it.
#pragma once
#include <type_traits>
#include "kr_paged_dev.h"

// krh_paged_attention; fine: an F32 cache's products of a row in several sums (PaWave)
void kr_paged_attention(bool fine, float *o, const krh_pages *kv, const int *table, int table_ld, const int *len, int n_seq,
                        const float *q, int n_heads, int max_len, int window, float scale, float softcap, float *mass,
                        size_t mass_ld, void *ws);

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

// A group's first rows are passed over for all of its sequences at once, and the
// waves have the rows behind them: group[g] .. group[g + 1] are its sequences,
// shared[g] its rows.
constexpr int PA_GROUPS = 64;   // one a lane
struct PaShared : PaArgs {
    const int *group, *shared;
    int n_groups, max_shared;
};
// How many rows of sequence i, this lane's, go before: every lane of the wave calls it
__device__ __forceinline__ int pa_skip(const PgView &, const PaArgs &, int, int &) { return 0; }
__device__ __forceinline__ int pa_skip(const PgView &p, const PaShared &a, int i, int &bad);

// rows [first, len) of a sequence, in tiles from the one that holds `first`; a
// sequence of no rows has one tile, whose output is zeros. `skip` rows go before.
struct PaSpan {
    int len, first, begin, tiles;
};
__device__ __forceinline__ PaSpan pa_span(const PaArgs &a, int len, int skip) {   // len within [0, max_len]
    PaSpan r;
    r.len = len;
    r.first = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
    if (skip > 0) r.first = max(r.first, min(skip, len));
    r.begin = r.first & -(1 << a.tl);
    r.tiles = max(1, (r.len - r.begin + (1 << a.tl) - 1) >> a.tl);
    return r;
}

// All sequences' tiles, and how many shares they make: share u has tiles
// [u T / n, (u + 1) T / n). With it the spans of 64 sequences, one a lane.
struct PaAll {
    int tiles, shares;
    int base, len, skip, sum;   // the lanes' sequences from `base` on: lengths, rows before, inclusive sums of tiles
    int before;           // tiles of the sequences before `base`
};
template <class A> __device__ __forceinline__ void pa_fetch(const PgView &p, const A &a, PaAll &r, int base, int &bad) {
    const int i = base + (int)(threadIdx.x & 63);
    r.base = base;
    r.len = i < p.n_seq ? kr_page_len(a.len[i], a.max_len, bad) : 0;
    r.skip = pa_skip(p, a, i, bad);
    r.sum = pg_scan(i < p.n_seq ? pa_span(a, r.len, r.skip).tiles : 0);
}
// most: the shares that there are at most
template <class A> __device__ __forceinline__ PaAll pa_all(const PgView &p, const A &a, int &bad, int most) {
    PaAll r;
    int t = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += 64) {
        r.before = t;
        pa_fetch(p, a, r, i0, bad);
        t += __builtin_amdgcn_readlane(r.sum, 63);
    }
    r.tiles = t;
    r.shares = max(1, min(most, (t + a.least - 1) / a.least));
    return r;
}
template <class A> __device__ __forceinline__ PaSpan pa_of(const PgView &p, const A &a, PaAll &r, int s, int &bad) {
    if (s - r.base >= 64 || s < r.base) pa_fetch(p, a, r, s & ~63, bad);
    const int skip = std::is_same_v<A, PaArgs> ? 0 : __builtin_amdgcn_readlane(r.skip, s - r.base);
    return pa_span(a, __builtin_amdgcn_readlane(r.len, s - r.base), skip);
}
// the sequence that holds tile t of all; t becomes the tile's number in it
template <class A> __device__ __forceinline__ int pa_find(const PgView &p, const A &a, PaAll &r, int &t, int &bad) {
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

// The power of two by which a head's queries are scaled to become halves, the largest of them m: to 2^13 or more, but that
// the scores' factor, scale times the other power, stays a normal float
__device__ __forceinline__ int pa_power(float m, float scale) {
    if (!(m > 0.0f && m < INFINITY)) return 0;
    // |scale| 2^-e >= 2^(s - 127) 2^-e
    const int s = (int)(__float_as_uint(scale) >> 23 & 255);
    return min(13 - ilogbf(m), s - 1);
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

// FINE: an F32 cache's products as four sums, added at the end. Of the output's error
// against 64 bits one sum of 256 floats is most: 8 sequences of 1024 rows of 256 dims
// 1.1e-6, with four sums 4.0e-7, in 20.1 us instead of 19.8.
template <int KT, int CL, bool FULL, class A = PaArgs, bool FINE = false> struct PaWave {
    using Raw = PaRaw<KT, CL>;
    static constexpr int W = Raw::W, KS = Raw::KS, NT = Raw::NT, R = Raw::R, TILE = 16 * NT;
    static constexpr int EB = KT == PG_F32 ? 4 : KT == PG_F16 ? 2 : 1;
    static constexpr int KD = KT == PG_F32 ? 4 : 8;   // dims a K load
    static constexpr bool HALF = KT != PG_F32;

    const PgView &p;
    const A &a;
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

    __device__ __forceinline__ PaWave(const PgView &p_, const A &a_, int kvh_)
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
            e = pa_power(m, a.scale);
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
            [[maybe_unused]] float4v more[3] = {};
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
                } else if constexpr (FINE) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float4v &sum = c == 0 ? acc : more[c - 1];
                        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.k[b][j][c]), qf[j][0][c], sum, 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.k[b][j][c]), qf[j][0][c], acc, 0,
                                                                   0, 0);
                }
            }
            if constexpr (FINE && !HALF) acc = (acc + more[0]) + (more[1] + more[2]);
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
        constexpr bool own = std::is_same_v<A, PaArgs>;   // no rows go before
        const bool alone = own && t == 0 && end == sp.tiles;
        if (own ? sp.len > 0 : sp.first < sp.len) {
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

// The shares of a sequence: their first slot and number, by the arithmetic that made them.
struct PaParts {
    size_t slot;
    int n;
};
template <class A>
__device__ __forceinline__ PaParts pa_parts(const PgView &p, const A &a, int s, int kvh, PaSpan &sp, int most) {
    int bad = 0;   // reported by the shares
    PaAll all = pa_all(p, a, bad, most);
    int before = 0;
    for (int i = threadIdx.x & 63; i < (s & ~63); i += 64)
        before += pa_span(a, kr_page_len(a.len[i], a.max_len, bad), pa_skip(p, a, i, bad)).tiles;
    for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o);
    sp = pa_of(p, a, all, s, bad);
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

}  // namespace
