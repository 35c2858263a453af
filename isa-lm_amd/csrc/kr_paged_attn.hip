// Attention of one token of each sequence over a paged cache (krh_paged_attention).
//
// A workgroup takes a chunk of one sequence's rows for one KV head, its four waves
// every fourth tile of 32 rows; each wave passes over its rows once with the running
// maximum and sum of the softmax. The waves' parts are joined in LDS, a
// sequence's chunks by a second launch.
//
// Both products run on the matrix cores, transposed so that nothing passes
// through LDS: S^T = K Q^T has rows as the tile's rows and query heads as its
// columns, and the lane that holds a head's scores of 8 consecutive rows holds
// them as the operand P^T of O^T = V^T P^T. K's rows are read straight into
// operand registers (the order of the contraction is free, so a lane reads 8
// dims at a time); V's are transposed 2 by 2 in registers by byte permutes
// (F32: none, a float is an operand by itself).
//
// The halves' products are exact in 32 bits, so a float operand is split in
// two halves, x = hi + lo with |x - hi - lo| <= 2^-22 |x|: the queries (scaled by a
// power of two a head) and the weights (scaled by 2^14, so that weights 2^-28
// of the largest keep hi and lo whole). A KV head of up to 8 query heads has the
// hi parts in columns 0-7 and the lo parts in 8-15 of one product. int8 rows become halves
// exactly (their scale multiplies the score, or the weight); F32 caches take
// the 32-bit product, whose rate still passes what HBM delivers.
#include <type_traits>
#include "kr_paged_dev.h"

namespace {

constexpr int PA_T = 256, PA_W = PA_T / 64, PA_TILE = 32, PA_STEP = PA_W * PA_TILE;
constexpr float PA_UP = 0x1p14f;   // the weights' scale (halves end at 2^16)

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
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
    float *part;    // [n_seq][nh][n_split][hd]: a chunk's sums
    float *pml;     // [n_seq][nh][n_split][2]: their maximum (log2) and weight
    float *fin;     // [n_seq][nh][2]: the whole row's, for the mass
    float *z;       // [n_seq][nh][z_ld]: the scores (log2), for the mass
    size_t z_ld;
    int nh, max_len, window, chunk, n_split;
    float scale, cap;
};

// rows [first, len) of a sequence in chunks from the tile that holds `first`
struct PaSpan {
    int len, first, begin, parts;
};
__device__ __forceinline__ PaSpan pa_span(const PaArgs &a, int s, int &bad) {
    PaSpan r;
    r.len = kr_page_len(a.len[s], a.max_len, bad);
    r.first = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
    r.begin = r.first & ~(PA_TILE - 1);
    r.parts = (r.len - r.begin + a.chunk - 1) / a.chunk;
    return r;
}

__device__ __forceinline__ float pa_swap8(float x) {   // the lane 8 away in its row of 16
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
}
__device__ __forceinline__ float pa_max_g(float v) {   // over the 4 lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// halves of 4 int8 (xor 0x80: 0..255) as 1024 + u - 1152, exact
__device__ __forceinline__ unsigned pa_h2(unsigned u, unsigned sel) {
    const half2v h = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, sel));
    return __builtin_bit_cast(unsigned, h - half2v{ (_Float16)1152.0f, (_Float16)1152.0f });
}

// what a lane holds of a tile, as it lies in memory. K: per product step its
// rows r and r + 4; V: W dims of each of its 8 rows.
template <int KT, int CL> struct PaRaw {
    static constexpr int W = CL / 16;                                  // dims a lane has of a V row
    static constexpr int KS = KT == PG_F32 ? CL / 16 : CL / 32;        // loads a K row
    static constexpr int KB = KT == PG_F32 ? 4 : KT == PG_F16 ? 4 : 2; // words a load
    static constexpr int VB = KT == PG_F32 ? W : KT == PG_F16 ? W / 2 : W / 4;
    unsigned k[2][KS][KB], v[8][VB];
};

template <int N> __device__ __forceinline__ void pa_load(unsigned (&x)[N], const void *p) {
    static_assert(N == 1 || N == 2 || N % 4 == 0, "whole loads");
    if (N == 1) {
        x[0] = *(const unsigned *)p;
    } else if (N == 2) {
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

template <int KT, int CL, int NB, bool FULL>
__global__ void __launch_bounds__(PA_T, KT == PG_F32 ? 1 : 2) k_paged_split(const PgView p, const PaArgs a, int *fault) {
    using Raw = PaRaw<KT, CL>;
    constexpr int W = Raw::W, KS = Raw::KS, EB = KT == PG_F32 ? 4 : KT == PG_F16 ? 2 : 1;
    constexpr int KD = KT == PG_F32 ? 4 : 8;   // dims a K load
    constexpr bool HALF = KT != PG_F32;
    __shared__ float s_o[PA_W - 1][W * 4][64];
    __shared__ float s_m[PA_W][16], s_l[PA_W][16];

    const int s = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4, hd = FULL ? CL : p.hd, group = a.nh / p.n_kv;
    int bad = 0;
    const PaSpan sp = pa_span(a, s, bad);
    if (split >= (sp.parts > 1 ? sp.parts : 1)) return;

    const int col = NB == 1 && HALF ? n & 7 : n;
    const bool live = col < group, is_lo = NB == 1 && HALF && n >= 8;
    const size_t head = (size_t)s * a.nh + kvh * group + (live ? col : 0);

    // the queries as operands
    const float *q = a.q + head * hd;
    float qf[HALF ? 1 : KS][4];
    half8 qh[HALF ? KS : 1][NB];
    int e = 0;
    if (HALF) {
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
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = ldexpf(x[j][i], e);
                const _Float16 hi = (_Float16)y;
                const _Float16 lo = (_Float16)(y - (float)hi);
                if (NB == 1) {
                    qh[j][0][i] = is_lo ? lo : hi;
                } else {
                    qh[j][0][i] = hi;
                    qh[j][NB - 1][i] = lo;
                }
            }
    } else {
#pragma unroll
        for (int j = 0; j < KS; j++) {
            const int d = j * 16 + g * 4;
            const float4v t = live && (FULL || d < hd) ? *(const float4v *)(q + d) : float4v{ 0, 0, 0, 0 };
#pragma unroll
            for (int c = 0; c < 4; c++) qf[j][c] = t[c];
        }
    }

    float m_run = -INFINITY, l_run = 0.0f;
    int ev = -120;   // Q8: the weights carry the V scales over 2^ev
    float4v o[W];
#pragma unroll
    for (int c = 0; c < W; c++) o[c] = float4v{ 0, 0, 0, 0 };

    const int c0 = sp.begin + split * a.chunk, c1 = min(sp.len, c0 + a.chunk);
    Raw raw;
    float kd[8], vd[8];
    size_t row_lo = 0, row_hi = 0;   // pool rows of the tile's two halves
    // a half's page, looked up where the half has rows that are attended
    auto find = [&](int t0) {
        const int pl = t0 + 16 > sp.first ? pg_page(p, s, t0, bad) : -1;
        const int ph = t0 + 16 < sp.len ? pg_page(p, s, t0 + 16, bad) : -1;
        const int lo = __builtin_amdgcn_readfirstlane(pl >= 0 ? pl : ph), hi = __builtin_amdgcn_readfirstlane(ph >= 0 ? ph : pl);
        row_lo = kr_page_row(lo, p.n_kv, kvh, p.shift, t0);
        row_hi = kr_page_row(hi, p.n_kv, kvh, p.shift, t0 + 16);
    };
    const int kr0 = 8 * (n >> 2) + (n & 3);   // this lane's K rows of the tile: kr0, kr0 + 4
    auto load_k = [&]() {
        const size_t r = (kr0 < 16 ? row_lo + kr0 : row_hi + (kr0 - 16));
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const char *at = (const char *)p.k + (r + 4 * b) * hd * EB;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = (j * 4 + g) * KD;
                const bool in = FULL || d < hd;
                pa_load(raw.k[b][j], at + (in ? d : 0) * EB);
                if (!FULL)
#pragma unroll
                    for (int i = 0; i < Raw::KB; i++) raw.k[b][j][i] = in ? raw.k[b][j][i] : 0u;
            }
        }
    };
    const int vr0 = 8 * g;   // its V rows: vr0 .. vr0 + 7
    auto load_v = [&]() {
        const size_t r = vr0 < 16 ? row_lo + vr0 : row_hi + (vr0 - 16);
        if (KT == PG_Q8) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4v x = *(const float4v *)(p.kd + r + i), y = *(const float4v *)(p.vd + r + i);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    kd[i + c] = x[c];
                    vd[i + c] = y[c];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const char *at = (const char *)p.v + (r + i) * hd * EB;
            if (FULL) {
                pa_load(raw.v[i], at + n * W * EB);
            } else {
                // 4 dims at a time where a lane has them, else 8 (head_dim is a multiple of 8)
                constexpr int P = W < 8 ? W : 8, PW = P * EB / 4;
#pragma unroll
                for (int d = 0; d < W; d += P) {
                    const bool in = n * W + d < hd;
                    unsigned x[PW];
                    pa_load(x, at + (in ? n * W + d : 0) * EB);
#pragma unroll
                    for (int w = 0; w < PW; w++) raw.v[i][d * EB / 4 + w] = in ? x[w] : 0u;
                }
            }
        }
    };

    int t0 = c0 + wave * PA_TILE;
    if (t0 < c1) {
        find(t0);
        load_k();
    }
    for (; t0 < c1; t0 += PA_STEP) {
        load_v();
        // scores: rows t0 + 8 g + i of head `col`, i < 8
        float sc[8];
#pragma unroll
        for (int b = 0; b < 2; b++) {
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
                    const half8 kf = __builtin_bit_cast(half8, w);
#pragma unroll
                    for (int x = 0; x < NB; x++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[j][x], acc, 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.k[b][j][c]), qf[j][c], acc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) sc[4 * b + i] = acc[i];
        }
        // the next tile's K while the rest runs
        if (t0 + PA_STEP < c1) {
            find(t0 + PA_STEP);
            load_k();
        }
        const bool whole = t0 >= sp.first && t0 + PA_TILE <= sp.len;
        const int r0 = t0 + 8 * g;
        float m_tile = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float x = sc[i];
            if (HALF) {
                if (NB == 1) x += pa_swap8(x);
                x = ldexpf(x, -e);
            }
            x *= a.scale;
            if (KT == PG_Q8) x *= kd[i];
            sc[i] = x;
        }
        if (a.cap > 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++) sc[i] = a.cap * kr_tanhf(sc[i] / a.cap);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sc[i] *= 1.4426950408889634f;
            if (!whole && (r0 + i < sp.first || r0 + i >= sp.len)) sc[i] = -INFINITY;
            m_tile = fmaxf(m_tile, sc[i]);
        }
        if (a.z && live && !is_lo) {
            float *z = a.z + head * a.z_ld + r0;
            *(float4v *)z = float4v{ sc[0], sc[1], sc[2], sc[3] };
            *(float4v *)(z + 4) = float4v{ sc[4], sc[5], sc[6], sc[7] };
        }
        m_tile = pa_max_g(m_tile);
        int ev_new = ev;
        if (KT == PG_Q8) {
            float vm = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (!whole && (r0 + i < sp.first || r0 + i >= sp.len)) vd[i] = 0.0f;
                vm = fmaxf(vm, fabsf(vd[i]));
            }
            vm = pa_max_g(vm);
            ev_new = max(ev, min((int)(__float_as_uint(vm) >> 23) - 126, 120));
        }
        if (__any(m_tile > m_run || ev_new > ev)) {
            const float m_new = fmaxf(m_run, m_tile);
            const float f = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            const float fo = KT == PG_Q8 ? ldexpf(f, ev - ev_new) : f;
            m_run = m_new;
            ev = ev_new;
            l_run *= f;
#pragma unroll
            for (int c = 0; c < W; c++) o[c] *= fo;
        }
        const float m_use = m_run == -INFINITY ? 0.0f : m_run;
        const float vs = KT == PG_Q8 ? ldexpf(1.0f, -ev) : 1.0f;
        half8 ph[NB];
        float pf[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float x = __builtin_amdgcn_exp2f(sc[i] - m_use);
            if (HALF) x *= PA_UP;
            l_run += x;
            if (KT == PG_Q8) x *= vd[i] * vs;
            if (HALF) {
                const _Float16 hi = (_Float16)x;
                const float rest = x - (float)hi;
                if (NB == 1) {
                    ph[0][i] = is_lo ? (_Float16)rest : hi;
                } else {
                    ph[0][i] = hi;
                    ph[NB - 1][i] = (_Float16)rest;
                }
            } else {
                pf[i] = x;
            }
        }
        // rows that are not attended may hold anything
        if (KT != PG_Q8 && !whole) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = r0 + i >= sp.first && r0 + i < sp.len;
#pragma unroll
                for (int w = 0; w < Raw::VB; w++) raw.v[i][w] = in ? raw.v[i][w] : 0u;
            }
        }
        if constexpr (KT == PG_F32) {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int c = 0; c < W; c++)
                    o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.v[i][c]), pf[i], o[c], 0, 0, 0);
        } else if constexpr (KT == PG_F16) {
#pragma unroll
            for (int c = 0; c < W; c++) {
                uint4v w;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w[i] = __builtin_amdgcn_perm(raw.v[2 * i + 1][c / 2], raw.v[2 * i][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                const half8 vf = __builtin_bit_cast(half8, w);
#pragma unroll
                for (int x = 0; x < NB; x++) o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[x], o[c], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int c4 = 0; c4 < W; c4 += 4) {
                uint4v w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned x = raw.v[2 * i][c4 / 4] ^ 0x80808080u, y = raw.v[2 * i + 1][c4 / 4] ^ 0x80808080u;
                    const unsigned u = __builtin_amdgcn_perm(y, x, 0x05010400u), v = __builtin_amdgcn_perm(y, x, 0x07030602u);
                    w[0][i] = pa_h2(u, 0x04010400);
                    w[1][i] = pa_h2(u, 0x04030402);
                    w[2][i] = pa_h2(v, 0x04010400);
                    w[3][i] = pa_h2(v, 0x04030402);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const half8 vf = __builtin_bit_cast(half8, w[c]);
#pragma unroll
                    for (int x = 0; x < NB; x++)
                        o[c4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[x], o[c4 + c], 0, 0, 0);
                }
            }
        }
    }
    if (lane == 0) kr_report(fault, bad);

    // the waves' parts
    if (NB == 1 && HALF) {
#pragma unroll
        for (int c = 0; c < W; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[c][i] += pa_swap8(o[c][i]);
    }
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    if (g == 0) {
        s_m[wave][n] = m_run;
        s_l[wave][n] = l_run;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < PA_W; w++) m = fmaxf(m, s_m[w][n]);
#pragma unroll
    for (int w = 0; w < PA_W; w++) l += s_m[w][n] == -INFINITY ? s_l[w][n] : s_l[w][n] * __builtin_amdgcn_exp2f(s_m[w][n] - m);
    // a part of no finite score holds nothing, or NaN
    float f = m_run == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m);
    if (KT == PG_Q8) f = ldexpf(f, ev);
#pragma unroll
    for (int c = 0; c < W; c++) o[c] *= f;
    if (wave > 0) {
#pragma unroll
        for (int c = 0; c < W; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) s_o[wave - 1][4 * c + i][lane] = o[c][i];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < PA_W - 1; w++)
#pragma unroll
        for (int c = 0; c < W; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[c][i] += s_o[w][4 * c + i][lane];
    if (!live || is_lo) return;
    const bool alone = sp.parts <= 1;
    float *out;
    if (alone) {
        out = a.o + head * hd;
        const float inv = 1.0f / l;
#pragma unroll
        for (int c = 0; c < W; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[c][i] = sp.len > 0 ? o[c][i] * inv : 0.0f;
    } else {
        out = a.part + (head * a.n_split + split) * hd;
    }
    if (g == 0) {
        if (!alone) {
            a.pml[(head * a.n_split + split) * 2] = m;
            a.pml[(head * a.n_split + split) * 2 + 1] = l;
        } else if (a.fin) {
            a.fin[head * 2] = m;
            a.fin[head * 2 + 1] = l;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d0 = (4 * g + i) * W;
#pragma unroll
        for (int c = 0; c < W; c += 4)
            if (FULL || d0 + c < hd) *(float4v *)(out + d0 + c) = float4v{ o[c][i], o[c + 1][i], o[c + 2][i], o[c + 3][i] };
    }
}

// A head's chunks: 2^dl lanes hold its dims four at a time, the workgroup's other
// factor the chunks side by side.
constexpr int PJ_T = 512;
__global__ void __launch_bounds__(PJ_T) k_paged_join(const PgView p, const PaArgs a, int dl) {
    __shared__ float4v s_o[PJ_T];
    __shared__ float s_l[PJ_T / 64];
    const int s = blockIdx.y, tid = threadIdx.x;
    int bad = 0;   // reported by the chunks
    const PaSpan sp = pa_span(a, s, bad);
    if (sp.parts <= 1) return;
    const size_t head = (size_t)s * a.nh + blockIdx.x;
    const float *ml = a.pml + head * a.n_split * 2, *part = a.part + head * a.n_split * p.hd;
    float m = -INFINITY;
    for (int i = tid & 63; i < sp.parts; i += 64) m = fmaxf(m, ml[2 * i]);
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const int l = tid & ((1 << dl) - 1), lanes = PJ_T >> dl;
    float4v acc = { 0, 0, 0, 0 };
    float sum = 0.0f;
#pragma unroll 8
    for (int i = tid >> dl; i < sp.parts; i += lanes) {
        const float f = __builtin_amdgcn_exp2f(ml[2 * i] - m);
        sum += ml[2 * i + 1] * f;
        if (4 * l < p.hd) acc += *(const float4v *)(part + (size_t)i * p.hd + 4 * l) * f;
    }
    // the lanes of one group have the same sum: one of each counts
    float ls = l == 0 ? sum : 0.0f;
    for (int o = 32; o >= 1; o >>= 1) ls += __shfl_xor(ls, o);
    if ((tid & 63) == 0) s_l[tid >> 6] = ls;
    s_o[tid] = acc;
    __syncthreads();
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < PJ_T / 64; i++) all += s_l[i];
    if (tid >> dl) return;
    for (int i = 1; i < lanes; i++) acc += s_o[(i << dl) + l];
    const float inv = 1.0f / all;
    if (4 * l < p.hd) *(float4v *)(a.o + head * p.hd + 4 * l) = acc * inv;
    if (a.fin && l == 0) {
        a.fin[head * 2] = m;
        a.fin[head * 2 + 1] = all;
    }
}

// mass[r] += the row's weights over the KV head's query heads, in head order
__global__ void __launch_bounds__(PA_T) k_paged_mass(const PgView p, const PaArgs a, float up) {
    const int s = blockIdx.z, kvh = blockIdx.y, group = a.nh / p.n_kv;
    int bad = 0;
    const PaSpan sp = pa_span(a, s, bad);
    const int r = sp.first + (int)(blockIdx.x * PA_T + threadIdx.x);
    if (r >= sp.len) return;
    float sum = 0.0f;
    for (int h = 0; h < group; h++) {
        const size_t head = (size_t)s * a.nh + kvh * group + h;
        sum += __builtin_amdgcn_exp2f(a.z[head * a.z_ld + r] - a.fin[2 * head]) * (up / a.fin[2 * head + 1]);
    }
    a.mass[((size_t)s * p.n_kv + kvh) * a.mass_ld + r] += sum;
}

// Rows a chunk, a multiple of a workgroup's step: about PA_PARTS chunks in all
// within [PA_LEAST, PA_MOST] rows.
constexpr int PA_PARTS = 2048, PA_LEAST = 128, PA_MOST = 512;
int pa_chunk(int n_seq, int n_kv, int rows) {
    const long long c = (long long)n_seq * n_kv * rows / PA_PARTS;
    return (int)((c < PA_LEAST ? PA_LEAST : c > PA_MOST ? PA_MOST : c) + PA_STEP - 1) / PA_STEP * PA_STEP;
}
// the most chunks that any number of rows up to `rows` is cut into: those of the
// largest chunk, or one more than PA_PARTS over the heads
int pa_most_parts(int n_seq, int n_kv, int rows) {
    const long long heads = (long long)n_seq * n_kv, big = (rows + PA_MOST - 1) / PA_MOST, even = PA_PARTS / heads + 1;
    const long long least = (rows + PA_LEAST - 1) / PA_LEAST, n = big > even ? big : even;
    return (int)(n < least ? n : least);
}

// the workspace's pieces, in floats, for n_split chunks
struct PaSizes {
    size_t part, pml, fin, z_ld, z;
};
PaSizes pa_sizes(const krh_pages *kv, int n_seq, int nh, int max_len, int n_split, bool mass) {
    PaSizes r;
    const size_t heads = (size_t)n_seq * nh;
    r.part = n_split > 1 ? heads * n_split * kv->head_dim : 0;
    r.pml = n_split > 1 ? (heads * n_split * 2 + 3) & ~(size_t)3 : 0;
    r.fin = mass ? (heads * 2 + 3) & ~(size_t)3 : 0;
    r.z_ld = mass ? ((size_t)max_len + PA_TILE - 1) / PA_TILE * PA_TILE : 0;
    r.z = heads * r.z_ld;
    return r;
}

bool pa_args_ok(const krh_pages *kv, int n_seq, int n_heads, int max_len) {
    return pg_pages_ok(kv) && n_seq > 0 && n_seq <= KRH_ROWS_MAX && max_len > 0 && max_len <= INT32_MAX / 2 && n_heads > 0 &&
           n_heads % kv->n_kv_heads == 0 && n_heads / kv->n_kv_heads <= KR_PAGE_GROUP_MAX;
}

using PaKernel = void (*)(const PgView, const PaArgs, int *);

template <int KT, int CL> PaKernel pa_kernel(int group, int hd) {
    if constexpr (KT == PG_F32) {
        return hd == CL ? k_paged_split<KT, CL, 1, true> : k_paged_split<KT, CL, 1, false>;
    } else {
        if (hd != CL) return k_paged_split<KT, CL, 2, false>;
        return group <= 8 ? k_paged_split<KT, CL, 1, true> : k_paged_split<KT, CL, 2, true>;
    }
}
template <int KT> PaKernel pa_kernel(int group, int hd) {
    return hd <= 64 ? pa_kernel<KT, 64>(group, hd) : hd <= 128 ? pa_kernel<KT, 128>(group, hd) : pa_kernel<KT, 256>(group, hd);
}

}  // namespace

extern "C" size_t krh_paged_attention_ws(const krh_pages *kv, int n_seq, int n_heads, int max_len, int mass) {
    if (!pa_args_ok(kv, n_seq, n_heads, max_len)) return 0;
    const PaSizes r = pa_sizes(kv, n_seq, n_heads, max_len, pa_most_parts(n_seq, kv->n_kv_heads, max_len), mass != 0);
    return sizeof(float) * (r.part + r.pml + r.fin + r.z + 4);
}

extern "C" void krh_paged_attention(float *o, const krh_pages *kv, const int *table, int table_ld, const int *len,
                                    int n_seq, const float *q, int n_heads, int max_len, int window, float scale,
                                    float softcap, float *mass, size_t mass_ld, void *ws) {
    if (n_seq == 0) return;
    if (pg_refuse(pa_args_ok(kv, n_seq, n_heads, max_len), "paged_attention sizes") ||
        pg_refuse(o && table && table_ld > 0 && len && q && ws && pg_aligned(o) && pg_aligned(q) && pg_aligned(ws),
                  "paged_attention: a missing or unaligned array") ||
        pg_refuse(window >= 0 && softcap >= 0.0f && (!mass || mass_ld >= (size_t)max_len),
                  "paged_attention: window, soft-cap or mass rows"))
        return;
    // a window's rows, and those before them in its first tile
    const int rows = window > 0 && window < max_len - PA_TILE ? window + PA_TILE - 1 : max_len;
    const int chunk = pa_chunk(n_seq, kv->n_kv_heads, rows), n_split = (rows + chunk - 1) / chunk;
    const PaSizes r = pa_sizes(kv, n_seq, n_heads, max_len, n_split, mass != nullptr);
    float *w = (float *)ws;
    PaArgs a = {};
    a.o = o, a.q = q, a.len = len, a.mass = mass, a.mass_ld = mass_ld;
    a.part = w, a.pml = w + r.part, a.fin = mass ? w + r.part + r.pml : nullptr;
    a.z = mass ? w + r.part + r.pml + r.fin : nullptr, a.z_ld = r.z_ld;
    a.nh = n_heads, a.max_len = max_len, a.window = window, a.chunk = chunk, a.n_split = n_split;
    a.scale = scale, a.cap = softcap;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const int group = n_heads / kv->n_kv_heads, hd = kv->head_dim;
    const PaKernel f = kv->kv_type == ML_F32 ? pa_kernel<PG_F32>(group, hd) : kv->kv_type == ML_F16 ? pa_kernel<PG_F16>(group, hd)
                                                                                                    : pa_kernel<PG_Q8>(group, hd);
    hipLaunchKernelGGL(f, dim3(n_split, kv->n_kv_heads, n_seq), dim3(PA_T), 0, kr_stream(), p, a, kr_fault_word());
    kr_check_launch("paged_attention");
    if (n_split > 1) {
        hipLaunchKernelGGL(k_paged_join, dim3(n_heads, n_seq), dim3(PJ_T), 0, kr_stream(), p, a, pg_log2(hd / 4));
        kr_check_launch("paged_attention");
    }
    if (mass) {
        hipLaunchKernelGGL(k_paged_mass, dim3((rows + PA_T - 1) / PA_T, kv->n_kv_heads, n_seq), dim3(PA_T), 0, kr_stream(), p, a,
                           kv->kv_type == ML_F32 ? 1.0f : PA_UP);
        kr_check_launch("paged_attention");
    }
}
