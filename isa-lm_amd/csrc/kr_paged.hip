// Several sequences over one paged cache: the rows of new tokens into their
// pages (per-head norm and rotation on the way), attention of one token of each
// sequence, and eviction by accumulated attention weight.
#include "kr_paged_dev.h"

namespace {

constexpr int PG_T = 256;

// ---- rows into and out of pages ----
// An item is one head's vector of one token; 2^lps >= hd / 8 lanes share it,
// eight values each, so a wave holds two to eight items of the usual heads and
// its accesses are contiguous. Bound by HBM (8 bytes a query value, 4 + the cache's
// width a key or value) without a norm, 8-bit rows and norms by the instructions
// an item takes: with four values a lane 2047 tokens of the 1B shape took 14.7 us
// normalized into 8 bits, 11 into halves as they are.

// Sums and maxima over the n <= 32 lanes of an item (n a power of two), in
// registers: pairs, fours, then the mirrors of 8 and 16 lanes, whose parts agree
// by then, and the two rows of 16 swapped.
template <int CTRL> __device__ __forceinline__ unsigned pg_dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <class T, class F> __device__ __forceinline__ T pg_reduce(T v, int n, F f) {
    constexpr int W = sizeof(T) / 4;
    struct Words { unsigned w[W]; };
    auto other = [&](auto move) {
        Words x = __builtin_bit_cast(Words, v);
#pragma unroll
        for (int i = 0; i < W; i++) x.w[i] = move(x.w[i]);
        return __builtin_bit_cast(T, x);
    };
    if (n > 1) v = f(v, other([](unsigned x) { return pg_dpp<0xb1>(x); }));
    if (n > 2) v = f(v, other([](unsigned x) { return pg_dpp<0x4e>(x); }));
    if (n > 4) v = f(v, other([](unsigned x) { return pg_dpp<0x141>(x); }));
    if (n > 8) v = f(v, other([](unsigned x) { return pg_dpp<0x140>(x); }));
    const bool row = threadIdx.x & 16;
    if (n > 16)
        v = f(v, other([&](unsigned x) {
            const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
            return row ? s[0] : s[1];
        }));
    return v;
}
__device__ __forceinline__ double pg_sum(double v, int n) {
    return pg_reduce(v, n, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ float pg_max(float v, int n) {
    return pg_reduce(v, n, [](float a, float b) { return fmaxf(a, b); });
}

// 1 / sqrt(x) to a last bit or two of 64 by two steps from the instruction's
// estimate (the library's quotient and root took more of the kernel's time than
// its memory)
__device__ __forceinline__ double pg_rsqrt(double x) {
    if (!(x > 0.0 && x < (double)INFINITY)) return 1.0 / sqrt(x);
    double r = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; i++) r = __builtin_fma(r * 0.5, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}

struct QkvArgs {
    float *qo;
    const float *q, *k, *v, *qw, *kw, *cs, *sn;
    const int *seq, *row, *pos;
    size_t ldqo, ldq, ldk, ldv;
    float eps;
    double inv_hd;
    int ntok, nh, n_pos;
};

struct Pg8 {
    float v[8];
};
__device__ __forceinline__ Pg8 pg_get(const float *p) {
    const float4 x = *(const float4 *)p, y = *(const float4 *)(p + 4);
    return { { x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w } };
}
__device__ __forceinline__ void pg_put(float *p, const Pg8 &x) {
    *(float4 *)p = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
    *(float4 *)(p + 4) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
}

// row `at` (in rows of the pool) of K or V from eight values a lane, l < hd / 8;
// the conversions of krh_store_kv, but that an 8-bit row's factor is 127 times
// the rounded reciprocal of its maximum, as tensor libraries form 127 / max (a
// step of the factor at most: an element next to a border may fall on its other side)
template <int KT>
__device__ __forceinline__ void pg_store(void *dst, float *d, size_t at, int hd, const Pg8 &x, int l, bool live, int n) {
    const size_t e = at * hd + 8 * l;
    if constexpr (KT == PG_F32) {
        if (live) pg_put((float *)dst + e, x);
    } else if constexpr (KT == PG_F16) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = (unsigned)kr_f2h(x.v[2 * i]) | (unsigned)kr_f2h(x.v[2 * i + 1]) << 16;
        if (live) *(uint4 *)((uint16_t *)dst + e) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x.v[i]));
        m = pg_max(live ? m : 0.0f, n);
        const bool zero = m < KR_QUANT_TINY;
        const float id = zero ? 0.0f : kr_fmul(127.0f, kr_fdiv(1.0f, m));
        unsigned w[2] = { 0, 0 };
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!zero) w[i / 4] |= ((unsigned)kr_q8_elem(x.v[i], id) & 255u) << (8 * (i % 4));
        if (live) *(uint2 *)((int8_t *)dst + e) = make_uint2(w[0], w[1]);
        if (l == 0) d[at] = zero ? 0.0f : kr_fdiv(m, 127.0f);
    }
}

template <int KT> __global__ void __launch_bounds__(PG_T) k_paged_qkv(const PgView p, const QkvArgs a, int lps, int *fault) {
    const unsigned n = 1u << lps, per = a.nh + 2 * p.n_kv, item = (blockIdx.x * PG_T + threadIdx.x) >> lps;
    if (item >= a.ntok * per) return;   // whole items: the lanes that shuffle leave together
    const int l = (int)(threadIdx.x & (n - 1)), t = (int)(item / per), h = (int)(item % per), hd = p.hd;
    const bool live = 8 * l < hd, isq = h < a.nh, isk = !isq && h < a.nh + p.n_kv;
    const int kvh = h - a.nh - (isk || isq ? 0 : p.n_kv), d = live ? 8 * l : 0;
    const float *src = isq ? a.q + (size_t)t * a.ldq + (size_t)h * hd
                           : (isk ? a.k + (size_t)t * a.ldk : a.v + (size_t)t * a.ldv) + (size_t)kvh * hd;
    Pg8 x = pg_get(src + d);
    int bad = 0, row = 0, page = 0;
    int pos = a.cs ? a.pos[t] : 0;
    if (!isq) {
        const int seq = kr_page_in(a.seq[t], p.n_seq, KR_BAD_SEQ, bad);
        row = kr_page_in(a.row[t], INT_MAX, KR_BAD_PAGE, bad);
        page = pg_page(p, seq, row, bad);
    }
    // the value looks at the position too: of a bad token neither row is stored
    if (a.cs) pos = kr_page_in(pos, a.n_pos, KR_BAD_POS, bad);
    const bool keep = bad == 0;
    if (isq || isk) {
        const float *w = isq ? a.qw : a.kw;
        if (w) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i++) s = __builtin_fma((double)x.v[i], (double)x.v[i], s);
            s = pg_sum(live ? s : 0.0, n);
            const float inv = (float)pg_rsqrt(__builtin_fma(s, a.inv_hd, (double)a.eps));
            const Pg8 g = pg_get(w + d);
#pragma unroll
            for (int i = 0; i < 8; i++) x.v[i] = kr_fmul(kr_fmul(x.v[i], inv), g.v[i]);
        }
        if (a.cs) {
            const size_t at = (size_t)pos * (hd >> 1) + d / 2;
            const float4 c4 = *(const float4 *)(a.cs + at), s4 = *(const float4 *)(a.sn + at);
            const float c[4] = { c4.x, c4.y, c4.z, c4.w }, s[4] = { s4.x, s4.y, s4.z, s4.w };
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float u = x.v[2 * i], v = x.v[2 * i + 1];
                x.v[2 * i] = kr_fsub(kr_fmul(u, c[i]), kr_fmul(v, s[i]));
                x.v[2 * i + 1] = kr_fadd(kr_fmul(u, s[i]), kr_fmul(v, c[i]));
            }
        }
    }
    if (l == 0) kr_report(fault, bad);
    if (isq) {
        if (live) pg_put(a.qo + (size_t)t * a.ldqo + (size_t)h * hd + d, x);
        return;
    }
    if (!keep) return;
    pg_store<KT>(isk ? p.k : p.v, isk ? p.kd : p.vd, kr_page_row(page, p.n_kv, kvh, p.shift, row), hd, x, l, live, n);
}

template <int KT> __device__ __forceinline__ Pg8 pg_load8(const void *src, const float *d, size_t at, int hd, int l) {
    const size_t e = at * hd + 8 * l;
    if constexpr (KT == PG_F32) {
        return pg_get((const float *)src + e);
    } else if constexpr (KT == PG_F16) {
        const uint4 h = *(const uint4 *)((const uint16_t *)src + e);
        const unsigned w[4] = { h.x, h.y, h.z, h.w };
        Pg8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x.v[i] = kr_h2f((uint16_t)(w[i / 2] >> (16 * (i % 2))));
        return x;
    } else {
        const uint2 c = *(const uint2 *)((const int8_t *)src + e);
        const unsigned w[2] = { c.x, c.y };
        const float s = d[at];
        Pg8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x.v[i] = kr_fmul((float)(int8_t)(w[i / 4] >> (8 * (i % 4))), s);
        return x;
    }
}

template <int KT>
__global__ void __launch_bounds__(PG_T) k_paged_load(const PgView p, float *k, size_t ldk, float *v, size_t ldv, int n_rows,
                                                     const int *seqs, const int *rows, int lps, int *fault) {
    const unsigned n = 1u << lps, per = 2 * p.n_kv, item = (blockIdx.x * PG_T + threadIdx.x) >> lps;
    const int l = (int)(threadIdx.x & (n - 1));
    if (item >= n_rows * per || 8 * l >= p.hd) return;
    const int i = (int)(item / per), h = (int)(item % per), kvh = h < p.n_kv ? h : h - p.n_kv;
    int bad = 0;
    const int seq = kr_page_in(seqs[i], p.n_seq, KR_BAD_SEQ, bad), row = kr_page_in(rows[i], INT_MAX, KR_BAD_PAGE, bad);
    const size_t at = kr_page_row(pg_page(p, seq, row, bad), p.n_kv, kvh, p.shift, row);
    const bool isk = h < p.n_kv;
    Pg8 x = {};
    if (!bad) x = pg_load8<KT>(isk ? p.k : p.v, isk ? p.kd : p.vd, at, p.hd, l);
    if (l == 0) kr_report(fault, bad);
    pg_put((isk ? k + (size_t)i * ldk : v + (size_t)i * ldv) + (size_t)kvh * p.hd + 8 * l, x);
}

// ---- eviction ----

// Weights in an order of unsigned integers: larger is heavier, NaN the
// heaviest, -0 as +0
__device__ __forceinline__ unsigned ev_key(float w) {
    const unsigned u = __float_as_uint(w + 0.0f);   // -0 + 0 = +0
    return w != w ? 0xffffffffu : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// and back, where it was no NaN and no -0
__device__ __forceinline__ float ev_weight(unsigned u) {
    return __uint_as_float(u ^ ((unsigned)((int)~u >> 31) | 0x80000000u));
}

constexpr int EV_T = 1024, EV_W = EV_T / 64, EV_D = 11, EV_B = 1 << EV_D;   // radix digits of 11, 11 and 10 bits
constexpr int EV_U = 8;   // rows a lane reads ahead

struct EvArgs {
    const int *len;
    const float *mass;
    size_t mass_ld;
    int max_len, keep, recent;
    const int *out_table;
    int out_ld;
    int *out_len;
    float *out_mass;
    size_t out_mass_ld;
    int *cnt;   // [n_seq]: rows kept
    int *idx;   // [n_seq][n_kv][keep]: which, in order
    float *w;   // [n_seq][n_kv][keep]: their weights
};

// Sums of a count over the waves before this one
__device__ __forceinline__ int ev_before(const int *s, int wave) {
    const int sum = pg_scan(s[threadIdx.x & (EV_W - 1)]);
    return wave ? __builtin_amdgcn_readlane(sum, wave - 1) : 0;
}

// Rows r0 .. r1 - 1, EV_U x 64 at a time, a lane's reads side by side
template <class F> __device__ __forceinline__ void ev_rows(const float *mass, int r0, int r1, F f) {
    const int lane = threadIdx.x & 63;
    int r = r0;
    for (; r + 64 * EV_U <= r1; r += 64 * EV_U) {
        float w[EV_U];
        const float *at = mass + r + lane;
#pragma unroll
        for (int k = 0; k < EV_U; k++) w[k] = at[64 * k];
#pragma unroll
        for (int k = 0; k < EV_U; k++) f(r + lane + 64 * k, true, w[k]);
    }
    if (r >= r1) return;
    float w[EV_U];
#pragma unroll
    for (int k = 0; k < EV_U; k++) w[k] = mass[min(r + lane + 64 * k, r1 - 1)];
#pragma unroll
    for (int k = 0; k < EV_U; k++)
        if (r + 64 * k < r1) f(r + lane + 64 * k, r + lane + 64 * k < r1, w[k]);
}

// How many of the lanes below this one are in `m`
__device__ __forceinline__ int ev_below(unsigned long long m) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0));
}

// From the heaviest digit down: the one where the counts' sum reaches `need`,
// and how many of it are wanted. The whole workgroup; leaves the counts at zero.
__device__ __forceinline__ void ev_digit(int *hist, int *s_sum, int *s_res, int &digit, int &need) {
    const int tid = threadIdx.x, wave = tid >> 6;
    __syncthreads();
    const int hi = EV_B - 1 - 2 * tid, c0 = hist[hi], c1 = hist[hi - 1], sum = pg_scan(c0 + c1);
    if ((tid & 63) == 63) s_sum[wave] = sum;
    __syncthreads();
    const int before = sum - c0 - c1 + ev_before(s_sum, wave);
    if (before < need && before + c0 + c1 >= need) {
        const bool second = before + c0 < need;
        s_res[0] = second ? hi - 1 : hi;
        s_res[1] = need - before - (second ? c0 : 0);
    }
    hist[hi] = hist[hi - 1] = 0;
    __syncthreads();
    digit = s_res[0];
    need = s_res[1];
}

// One workgroup a (sequence, KV head): the weight of the last row kept by a
// radix select, then the kept rows' numbers in order, equal weights from the
// lowest row on. Each wave has an even part of the rows. The rows with the
// first digit's bits go to LDS, where they are few (each wave up to EV_C), and the
// other digits look at those. Bound by the one CU's instructions, three passes over
// the rows: 8 workgroups, 60,000 rows 32 us, 120,000 65; 32,001 rows 23.4, 102 with
// one lane looking through the counts and barriers every 1024 rows, 45 with five
// passes over all rows.
constexpr int EV_C = 512;
__global__ void __launch_bounds__(EV_T) k_evict_select(const EvArgs a, int *fault) {
    __shared__ int hist[EV_B];
    __shared__ unsigned s_key[EV_W][EV_C];
    __shared__ int s_sum[EV_W], s_res[2], s_above[EV_W], s_cand[EV_W], s_take[EV_W], s_tie[EV_W];
    const int kvh = blockIdx.x, s = blockIdx.y, n_kv = gridDim.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bad = 0;
    const int len = kr_page_len(a.len[s], a.max_len, bad);
    if (tid == 0) kr_report(fault, bad);
    const size_t sh = (size_t)s * n_kv + kvh;
    const float *mass = a.mass + sh * a.mass_ld;
    int *idx = a.idx + sh * a.keep;
    float *ow = a.w + sh * a.keep;
    const int kept = min(len, a.keep);
    if (kvh == 0 && tid == 0) a.cnt[s] = kept;
    if (len <= a.keep) {
        for (int r = tid; r < len; r += EV_T) {
            idx[r] = r;
            ow[r] = mass[r];
        }
        return;
    }
    const int old = len - a.recent, want = a.keep - a.recent;   // 0 <= want < old
    for (int r = tid; r < a.recent; r += EV_T) {
        idx[want + r] = old + r;
        ow[want + r] = mass[old + r];
    }
    if (want == 0) return;
    const int part = (old + EV_W - 1) / EV_W, r0 = min(old, wave * part), r1 = min(old, r0 + part);
    const unsigned long long below = ((unsigned long long)1 << lane) - 1;
    int need = want, digit;
    for (int i = tid; i < EV_B; i += EV_T) hist[i] = 0;
    __syncthreads();
    // zeros, which rows that no head looks at all have, count together
    int zeros = 0;
    ev_rows(mass, r0, r1, [&](int, bool in, float w) {
        zeros += __popcll(__ballot(in && w == 0.0f));
        if (in && w != 0.0f) atomicAdd(&hist[ev_key(w) >> (32 - EV_D)], 1);
    });
    if (lane == 0 && zeros) atomicAdd(&hist[0x80000000u >> (32 - EV_D)], zeros);
    ev_digit(hist, s_sum, s_res, digit, need);
    // each wave's rows above that digit, and the keys of those at it
    const unsigned d1 = digit;
    int above = 0, cand = 0;
    ev_rows(mass, r0, r1, [&](int, bool in, float w) {
        const unsigned u = ev_key(w), d = u >> (32 - EV_D);
        above += __popcll(__ballot(in && d > d1));
        const unsigned long long b = __ballot(in && d == d1);
        const int j = cand + __popcll(b & below);
        if (in && d == d1 && j < EV_C) s_key[wave][j] = u;
        cand += __popcll(b);
    });
    if (lane == 0) {
        s_above[wave] = above;
        s_cand[wave] = cand;
    }
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int i = 0; i < EV_W; i++) most = max(most, s_cand[i]);
    const bool few = most <= EV_C;
    // the keys at the first digit, from LDS or from the rows again
    auto keys = [&](auto f) {
        if (few) {
            for (int j = lane; j < cand; j += 64) f(s_key[wave][j]);
        } else {
            ev_rows(mass, r0, r1, [&](int, bool in, float w) {
                const unsigned u = ev_key(w);
                if (in && u >> (32 - EV_D) == d1) f(u);
            });
        }
    };
    unsigned prefix = d1 << (32 - EV_D);
    for (int b = 32 - 2 * EV_D;; b = 0) {   // bits 10 to 20, then 0 to 9
        const int top = b ? 32 - EV_D : 32 - 2 * EV_D;
        keys([&](unsigned u) {
            if (u >> top == prefix >> top) atomicAdd(&hist[u >> b & ((1u << (top - b)) - 1)], 1);
        });
        ev_digit(hist, s_sum, s_res, digit, need);
        prefix |= (unsigned)digit << b;
        if (b == 0) break;
    }
    // rows above `prefix`, and the first `need` of those at it
    int take = 0, ties = 0;
    keys([&](unsigned u) {
        take += u > prefix;
        ties += u == prefix;
    });
    for (int o = 32; o >= 1; o >>= 1) {
        take += __shfl_xor(take, o);
        ties += __shfl_xor(ties, o);
    }
    if (lane == 0) {
        s_take[wave] = above + take;
        s_tie[wave] = ties;
    }
    __syncthreads();
    ties = ev_before(s_tie, wave);
    int at = ev_before(s_take, wave) + min(ties, need);
    ev_rows(mass, r0, r1, [&](int r, bool in, float w) {
        const unsigned u = ev_key(w);
        const unsigned long long bt = __ballot(in && u == prefix);
        const bool got = in && (u > prefix || (u == prefix && ties + __popcll(bt & below) < need));
        const unsigned long long bk = __ballot(got);
        if (got) {
            const int j = at + __popcll(bk & below);
            idx[j] = r;
            ow[j] = w;
        }
        ties += __popcll(bt);
        at += __popcll(bk);
    });
}

__device__ __forceinline__ unsigned ev_load(__amdgpu_buffer_rsrc_t rows, int r, int k) {
    return __builtin_amdgcn_raw_buffer_load_b32(rows, r * 4 + k * 256, 0, 0);
}

// The same where all rows but the recent ones fit LDS, by their keys: one pass
// over the weights, the others over LDS. A launch on few rows is bound by its
// code's way from memory, so there is one copy for all digits and none for
// tails: rows past the last have the key 0, below any weight's. On many it is
// bound by the CU's instructions, 10 or so a row: 32,001 rows, 8 workgroups, 16.5
// us, 17.2 on another card (the select above: 23.4); 16 sequences of up to 4096, 7.5 (10.9).
template <int R> __global__ void __launch_bounds__(EV_T) k_evict_select_lds(const EvArgs a, int *fault) {
    __shared__ int hist[EV_B];
    __shared__ unsigned s_key[R];
    __shared__ int s_sum[EV_W], s_res[2], s_odd[EV_W], s_take[EV_W], s_tie[EV_W];
    const int kvh = blockIdx.x, s = blockIdx.y, n_kv = gridDim.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bad = 0;
    const int len = __builtin_amdgcn_readfirstlane(kr_page_len(a.len[s], a.max_len, bad));
    for (int i = tid; i < EV_B; i += EV_T) hist[i] = 0;
    if (tid == 0) kr_report(fault, bad);
    const size_t sh = (size_t)s * n_kv + kvh;
    const float *mass = a.mass + sh * a.mass_ld;
    int *idx = a.idx + sh * a.keep;
    float *ow = a.w + sh * a.keep;
    const int kept = min(len, a.keep), old = len <= a.keep ? 0 : len - a.recent, want = kept - (len - old);
    if (kvh == 0 && tid == 0) a.cnt[s] = kept;
#pragma unroll 1
    for (int r = tid; r < len - old; r += EV_T) {
        idx[want + r] = old + r;
        ow[want + r] = mass[old + r];
    }
    if (want == 0) return;   // 0 < want < old after this
    constexpr int N = 4, B = 64 * N;   // 256 rows at a time: 512 left waves idle (17.2, 8.3 us)
    const int part = ((old + EV_W - 1) / EV_W + B - 1) / B * B, r0 = wave * part, r1 = min(r0 + part, (old + B - 1) / B * B);
    __syncthreads();
    // zeros, which rows that no head looks at all have, count together
    int zeros = 0, odd = 0;   // odd: weights that their keys do not give back
    const auto rows = __builtin_amdgcn_make_buffer_rsrc((void *)mass, 0, old * 4, 0x00020000);   // 0 past them
    unsigned w[N], next[N];
#pragma unroll
    for (int k = 0; k < N; k++) next[k] = ev_load(rows, r0 + lane, k);
#pragma unroll 1
    for (int r = r0; r < r1; r += B) {
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = next[k];
#pragma unroll
        for (int k = 0; k < N; k++) next[k] = ev_load(rows, r + B + lane, k);
        unsigned long long o = 0;
#pragma unroll
        for (int k = 0; k < N; k++)   // NaN, -0
            o |= __builtin_amdgcn_ballot_w64(__builtin_amdgcn_classf(__uint_as_float(w[k]), 0x23));
        if (__builtin_expect(o != 0, 0)) {
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = w[k] << 1 > 0xff000000u ? 0x7fffffffu : w[k] == 0x80000000u ? 0 : w[k];
            odd = 1;
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const unsigned u = w[k], key = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
            s_key[r + lane + 64 * k] = key;
            zeros += __popcll(__builtin_amdgcn_ballot_w64(u == 0));
            if (u != 0) atomicAdd(&hist[key >> (32 - EV_D)], 1);
        }
    }
    if (r1 > max(r0, old)) {   // rows past the last, read as zeros
        zeros -= r1 - max(r0, old);
        for (int r = max(r0, old) + lane; r < r1; r += 64) s_key[r] = 0;
    }
    if (lane == 0) {
        if (zeros) atomicAdd(&hist[0x80000000u >> (32 - EV_D)], zeros);
        s_odd[wave] = odd;
    }
    int need = want, digit;
    unsigned prefix = 0;
#pragma unroll 1
    for (int b = 32 - EV_D;;) {   // bits 21 to 31, 10 to 20, 0 to 9
        ev_digit(hist, s_sum, s_res, digit, need);
        digit = __builtin_amdgcn_readfirstlane(digit);
        prefix |= (unsigned)digit << b;
        if (b == 0) break;
        const int top = b;
        b = max(0, b - EV_D);
        const unsigned pre = prefix >> top, mask = (1u << (top - b)) - 1;
#pragma unroll 1
        for (int r = r0; r < r1; r += B) {
            unsigned u[N];
#pragma unroll
            for (int k = 0; k < N; k++) u[k] = s_key[r + 64 * k + lane];
#pragma unroll
            for (int k = 0; k < N; k++)
                if (u[k] >> top == pre) atomicAdd(&hist[u[k] >> b & mask], 1);
        }
    }
    // rows above `prefix`, and the first `need` of those at it
    int take = 0, ties = 0;
#pragma unroll 1
    for (int r = r0; r < r1; r += B) {
        unsigned u[N];
#pragma unroll
        for (int k = 0; k < N; k++) u[k] = s_key[r + 64 * k + lane];
#pragma unroll
        for (int k = 0; k < N; k++) {
            take += __popcll(__builtin_amdgcn_ballot_w64(u[k] > prefix));
            ties += __popcll(__builtin_amdgcn_ballot_w64(u[k] == prefix));
        }
    }
    if (lane == 0) {
        s_take[wave] = take;
        s_tie[wave] = ties;
    }
    __syncthreads();
    ties = ev_before(s_tie, wave);
    int at = ev_before(s_take, wave) + min(ties, need);
    const bool give = !__any(s_odd[lane & (EV_W - 1)]);
#pragma unroll 1
    for (int r = r0; r < r1; r += B) {
        unsigned u[N];
#pragma unroll
        for (int k = 0; k < N; k++) u[k] = s_key[r + 64 * k + lane];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const unsigned long long bt = __builtin_amdgcn_ballot_w64(u[k] == prefix);
            bool got = u[k] >= prefix;
            if (bt) {
                if (ties + __popcll(bt) > need) got = got && (u[k] != prefix || ties + ev_below(bt) < need);
                ties += __popcll(bt);
            }
            const unsigned long long bk = __builtin_amdgcn_ballot_w64(got);
            if (got) {
                const unsigned j = 4 * (at + ev_below(bk));
                *(int *)((char *)idx + j) = r + 64 * k + lane;
                *(float *)((char *)ow + j) = ev_weight(u[k]);
            }
            at += __popcll(bk);
        }
    }
    if (give) return;
    __syncthreads();
#pragma unroll 1
    for (int j = tid; j < want; j += EV_T) ow[j] = mass[idx[j]];
}

// Rows into the new pages, in units of U bytes, as many rows a workgroup as its
// threads have units; their weights, and zeros past them. Bound by HBM: each row
// read once and written once (16 sequences of up to 4096 rows, 8B shape, half
// kept: 4.6 TB/s; with four units a thread one after another 4.3, all read before
// the first is written 3.3. Stores past the caches reach 5.0, but the attention
// that reads the new pages next loses as much).
constexpr unsigned EM_BLOCKS = 1 << 12;   // past it a workgroup takes more rows
template <class U> __global__ void __launch_bounds__(PG_T) k_evict_move(const PgView p, const EvArgs a, int rb, int rows,
                                                                        int *fault) {
    const int s = blockIdx.z, kvh = blockIdx.y, per = rb / (int)sizeof(U), kept = a.cnt[s], tid = threadIdx.x;
    const size_t sh = (size_t)s * p.n_kv + kvh;
    const int *idx = a.idx + sh * a.keep, *ot = a.out_table + (size_t)s * a.out_ld;
    if (blockIdx.x == 0 && kvh == 0 && tid == 0) a.out_len[s] = kept;
    int bad = 0;
    for (int j0 = blockIdx.x * rows; j0 < kept; j0 += gridDim.x * rows) {
        const int j = j0 + tid / per, u = tid % per;
        if (tid >= rows * per || j >= kept) continue;
        const int r = idx[j];
        int b = 0;
        const size_t from = kr_page_row(pg_page(p, s, r, b), p.n_kv, kvh, p.shift, r);
        const size_t to = kr_page_row(kr_page_of(ot, a.out_ld, j, p.shift, p.n_pages, b), p.n_kv, kvh, p.shift, j);
        bad |= b;
        if (b) continue;
        ((U *)p.k)[to * per + u] = ((const U *)p.k)[from * per + u];
        ((U *)p.v)[to * per + u] = ((const U *)p.v)[from * per + u];
        if (u == 0 && p.kd) {
            p.kd[to] = p.kd[from];
            p.vd[to] = p.vd[from];
        }
    }
    float *om = a.out_mass + sh * a.out_mass_ld;
    const int end = (int)min(a.out_mass_ld, (size_t)max(a.keep, a.max_len)), blocks = gridDim.x;
    for (int j = blockIdx.x * PG_T + tid; j < end; j += blocks * PG_T) om[j] = j < kept ? a.w[sh * a.keep + j] : 0.0f;
    kr_report(fault, bad);
}

// workgroups for `items` items of 2^lps lanes; 0: more than a launch holds
unsigned item_blocks(size_t items, int lps) {
    const size_t b = ((items << lps) + PG_T - 1) / PG_T;
    return b <= 0x7fffffff / PG_T ? (unsigned)b : 0;   // lanes stay within 31 bits
}

}  // namespace

extern "C" void krh_paged_qkv(float *qo, size_t ldqo, const krh_pages *kv, const int *table, int table_ld, int n_seq,
                              const float *q, size_t ldq, const float *k, size_t ldk, const float *v, size_t ldv,
                              int ntok, int n_heads, const int *seq, const int *row, const int *pos,
                              const float *q_norm, const float *k_norm, float eps, const float *cos_t,
                              const float *sin_t, int n_pos) {
    if (pg_refuse(pg_pages_ok(kv), "paged_qkv: the pages") ||
        pg_refuse(ntok >= 0 && n_heads >= 0 && n_heads <= KRH_ROWS_MAX && n_seq > 0 && table_ld > 0, "paged_qkv sizes"))
        return;
    if (ntok == 0) return;
    const size_t kvd = (size_t)kv->n_kv_heads * kv->head_dim, qd = (size_t)n_heads * kv->head_dim;
    if (pg_refuse(table && k && v && seq && row && (n_heads == 0 || (q && qo)) && (!cos_t) == (!sin_t) &&
                      (!cos_t || (pos && n_pos > 0)) && (n_heads == 0 || (!q_norm) == (!k_norm)),
                  "paged_qkv: a missing array") ||
        pg_refuse(ldk >= kvd && ldv >= kvd && ldk % 4 == 0 && ldv % 4 == 0 && pg_aligned(k) && pg_aligned(v) &&
                      pg_aligned(k_norm) && pg_aligned(cos_t) && pg_aligned(sin_t) &&
                      (n_heads == 0 || (ldq >= qd && ldqo >= qd && ldq % 4 == 0 && ldqo % 4 == 0 && pg_aligned(q) &&
                                        pg_aligned(qo) && pg_aligned(q_norm))),
                  "paged_qkv: row strides or alignment") ||
        // tokens pass in no order: with strides apart one's output would lie on another's query
        pg_refuse(n_heads == 0 || ntok == 1 || qo != q || ldqo == ldq, "paged_qkv: queries in place with another stride"))
        return;
    const int lps = pg_log2(kv->head_dim / 8);
    const unsigned grid = item_blocks((size_t)ntok * (n_heads + 2 * (size_t)kv->n_kv_heads), lps);
    if (pg_refuse(grid > 0, "paged_qkv: too many tokens") || pg_not_ready("paged_qkv before krh_init")) return;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const QkvArgs a = { qo,  q,    k,   v,   q_norm, k_norm, cos_t, sin_t, seq, row,
                        pos, ldqo, ldq, ldk, ldv,    eps,    1.0 / kv->head_dim,
                        ntok, n_heads, n_pos };
    const auto f = kv->kv_type == ML_F32   ? k_paged_qkv<PG_F32>
                   : kv->kv_type == ML_F16 ? k_paged_qkv<PG_F16>
                                           : k_paged_qkv<PG_Q8>;
    hipLaunchKernelGGL(f, dim3(grid), dim3(PG_T), 0, kr_stream(), p, a, lps, kr_fault_word());
    kr_check_launch("paged_qkv");
}

extern "C" void krh_paged_load(float *k, size_t ldk, float *v, size_t ldv, const krh_pages *kv, const int *table,
                               int table_ld, int n_seq, int n, const int *seq, const int *row) {
    if (pg_refuse(pg_pages_ok(kv), "paged_load: the pages") ||
        pg_refuse(n >= 0 && n_seq > 0 && table_ld > 0, "paged_load sizes"))
        return;
    if (n == 0) return;
    const size_t kvd = (size_t)kv->n_kv_heads * kv->head_dim;
    if (pg_refuse(table && k && v && seq && row, "paged_load: a missing array") ||
        pg_refuse(ldk >= kvd && ldv >= kvd && ldk % 4 == 0 && ldv % 4 == 0 && pg_aligned(k) && pg_aligned(v),
               "paged_load: row strides or alignment"))
        return;
    const int lps = pg_log2(kv->head_dim / 8);
    const unsigned grid = item_blocks((size_t)n * 2 * kv->n_kv_heads, lps);
    if (pg_refuse(grid > 0, "paged_load: too many rows") || pg_not_ready("paged_load before krh_init")) return;
    const auto f = kv->kv_type == ML_F32   ? k_paged_load<PG_F32>
                   : kv->kv_type == ML_F16 ? k_paged_load<PG_F16>
                                           : k_paged_load<PG_Q8>;
    hipLaunchKernelGGL(f, dim3(grid), dim3(PG_T), 0, kr_stream(), pg_view(kv, table, table_ld, n_seq), k, ldk, v, ldv,
                       n, seq, row, lps, kr_fault_word());
    kr_check_launch("paged_load");
}

extern "C" size_t krh_paged_evict_ws(int n_seq, int n_kv_heads, int keep) {
    if (n_seq <= 0 || n_kv_heads <= 0 || keep <= 0 || keep > KR_PAGE_LEN_MAX) return 0;
    return sizeof(int) * (2 * (size_t)n_seq * n_kv_heads * keep + n_seq);
}

extern "C" void krh_paged_evict(const krh_pages *kv, const int *table, int table_ld, const int *len, const float *mass,
                                size_t mass_ld, int n_seq, int max_len, int keep, int recent, const int *out_table,
                                int out_table_ld, int *out_len, float *out_mass, size_t out_ld, void *ws) {
    if (n_seq == 0) return;
    if (pg_refuse(pg_pages_ok(kv), "paged_evict: the pages") ||
        pg_refuse(n_seq > 0 && n_seq <= KRH_ROWS_MAX && max_len > 0 && max_len <= KR_PAGE_LEN_MAX && keep > 0 &&
                   keep <= KR_PAGE_LEN_MAX &&   // the copy's steps past the last mass stay within an int
                   recent >= 0 && recent <= keep && table_ld > 0 &&
                   out_table_ld > 0, "paged_evict sizes") ||
        pg_refuse(table && len && mass && out_table && out_len && out_mass && ws && !((uintptr_t)ws & 3) &&
                   out_table != table,
               "paged_evict: a missing array, or the pages onto themselves") ||
        pg_refuse(mass_ld >= (size_t)max_len && out_ld >= (size_t)keep && (out_mass != mass || out_ld == mass_ld),
               "paged_evict: mass rows") ||
        pg_refuse((size_t)out_table_ld * kv->page_size >= (size_t)(keep < max_len ? keep : max_len),
                   "paged_evict: out_table's pages"))
        return;
    if (pg_not_ready("paged_evict before krh_init")) return;
    int *w = (int *)ws;
    const size_t rows = (size_t)n_seq * kv->n_kv_heads * keep;
    const EvArgs a = { len, mass, mass_ld, max_len, keep, recent, out_table, out_table_ld, out_len, out_mass, out_ld,
                       w + 2 * rows, w, (float *)(w + rows) };
    // 40 KB of LDS leave room for a second workgroup on the CU: 64 sequences of up to 4000 rows, 9.4 us (136 KB: 12.7);
    // past 32768 rows the weights are read three times: 60,000, 32 us
    const int most_old = max_len - recent;
    const auto select = most_old <= 8192    ? k_evict_select_lds<8192>
                        : most_old <= 32768 ? k_evict_select_lds<32768>
                                            : k_evict_select;
    hipLaunchKernelGGL(select, dim3(kv->n_kv_heads, n_seq), dim3(EV_T), 0, kr_stream(), a, kr_fault_word());
    kr_check_launch("paged_evict");
    const int rb = kv->head_dim * (kv->kv_type == ML_F32 ? 4 : kv->kv_type == ML_F16 ? 2 : 1);
    const int most = keep < max_len ? keep : max_len;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const int units = rb / (rb % 16 ? 8 : 16), each = PG_T / units;   // rows a workgroup
    static_assert(PG_T >= KR_PAGE_HD_MAX * 4 / 8, "a row's units");
    const unsigned blocks = ((unsigned)most + each - 1) / each;
    hipLaunchKernelGGL(rb % 16 ? k_evict_move<uint2> : k_evict_move<uint4>,
                       dim3(blocks < EM_BLOCKS ? blocks : EM_BLOCKS, kv->n_kv_heads, n_seq), dim3(PG_T), 0, kr_stream(), p,
                       a, rb, each, kr_fault_word());
    kr_check_launch("paged_evict");
}
