// Several sequences over one paged cache: the rows of new tokens into their
// pages (per-head norm and rotation on the way), attention of one token of each
// sequence, and eviction by accumulated attention weight.
#include "kr_internal.h"
#include "kr_numerics.h"
#include "kr_paged.h"
#include "kr_paged_dev.h"

namespace {

constexpr int PG_T = 256;

// ---- rows into and out of pages ----
// An item is one head's vector of one token; 2^LPS >= hd / 4 lanes share it,
// four values each (whole 16-byte accesses), so a wave holds one to eight
// items and its loads are contiguous. Bound by HBM: 8 bytes a query value, 4 +
// the cache's width a key or value.

// over the 2^lps lanes of an item
__device__ __forceinline__ double pg_sum(double v, int n) {
    for (int o = n >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float pg_max(float v, int n) {
    for (int o = n >> 1; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

struct QkvArgs {
    float *qo;
    const float *q, *k, *v, *qw, *kw, *cs, *sn;
    const int *seq, *row, *pos;
    size_t ldqo, ldq, ldk, ldv;
    float eps;
    int ntok, nh, n_pos;
};

// row `at` (in rows of the pool) of K or V from four values a lane, l < hd / 4;
// the conversions of krh_store_kv, but that an 8-bit row's factor is 127 times
// the rounded reciprocal of its maximum, as tensor libraries form 127 / max (a
// step of the factor at most: an element next to a border may fall on its other side)
template <int KT> __device__ __forceinline__ void pg_store(void *dst, float *d, size_t at, int hd, float4 x, int l, bool live, int n) {
    const size_t e = at * hd + 4 * l;
    if (KT == PG_F32) {
        if (live) *(float4 *)((float *)dst + e) = x;
    } else if (KT == PG_F16) {
        const ushort4 h = make_ushort4(kr_f2h(x.x), kr_f2h(x.y), kr_f2h(x.z), kr_f2h(x.w));
        if (live) *(ushort4 *)((uint16_t *)dst + e) = h;
    } else {
        float m = live ? fmaxf(fmaxf(fmaxf(fmaxf(0.0f, fabsf(x.x)), fabsf(x.y)), fabsf(x.z)), fabsf(x.w)) : 0.0f;
        m = pg_max(m, n);
        const bool zero = m < KR_QUANT_TINY;
        const float id = zero ? 0.0f : kr_fmul(127.0f, kr_fdiv(1.0f, m));
        char4 c = make_char4(0, 0, 0, 0);
        if (!zero)
            c = make_char4((signed char)kr_q8_elem(x.x, id), (signed char)kr_q8_elem(x.y, id),
                           (signed char)kr_q8_elem(x.z, id), (signed char)kr_q8_elem(x.w, id));
        if (live) *(char4 *)((int8_t *)dst + e) = c;
        if (l == 0) d[at] = zero ? 0.0f : kr_fdiv(m, 127.0f);
    }
}

template <int KT> __global__ void __launch_bounds__(PG_T) k_paged_qkv(const PgView p, const QkvArgs a, int lps, int *fault) {
    const unsigned n = 1u << lps, per = a.nh + 2 * p.n_kv, item = (blockIdx.x * PG_T + threadIdx.x) >> lps;
    if (item >= a.ntok * per) return;   // whole items: the lanes that shuffle leave together
    const int l = (int)(threadIdx.x & (n - 1)), t = (int)(item / per), h = (int)(item % per), hd = p.hd;
    const bool live = 4 * l < hd, isq = h < a.nh, isk = !isq && h < a.nh + p.n_kv;
    const int kvh = h - a.nh - (isk || isq ? 0 : p.n_kv);
    const float *src = isq ? a.q + (size_t)t * a.ldq + (size_t)h * hd
                           : (isk ? a.k + (size_t)t * a.ldk : a.v + (size_t)t * a.ldv) + (size_t)kvh * hd;
    float4 x = live ? *(const float4 *)(src + 4 * l) : make_float4(0, 0, 0, 0);
    int bad = 0, seq = 0, row = 0, page = 0;
    if (!isq) {
        seq = kr_page_in(a.seq[t], p.n_seq, KR_BAD_SEQ, bad);
        row = kr_page_in(a.row[t], INT_MAX, KR_BAD_PAGE, bad);
        page = pg_page(p, seq, row, bad);
    }
    const bool keep = bad == 0;
    if (isq || isk) {
        const float *w = isq ? a.qw : a.kw;
        if (w) {
            const double s = pg_sum((double)x.x * x.x + (double)x.y * x.y + ((double)x.z * x.z + (double)x.w * x.w), n);
            const float inv = (float)(1.0 / sqrt(s / hd + (double)a.eps));
            if (live) {
                const float4 g = *(const float4 *)(w + 4 * l);
                x = make_float4(kr_fmul(kr_fmul(x.x, inv), g.x), kr_fmul(kr_fmul(x.y, inv), g.y),
                                kr_fmul(kr_fmul(x.z, inv), g.z), kr_fmul(kr_fmul(x.w, inv), g.w));
            }
        }
        if (a.cs) {
            const int pos = kr_page_in(a.pos[t], a.n_pos, KR_BAD_POS, bad);
            if (live) {
                const float2 c = *(const float2 *)(a.cs + (size_t)pos * (hd >> 1) + 2 * l);
                const float2 s = *(const float2 *)(a.sn + (size_t)pos * (hd >> 1) + 2 * l);
                x = make_float4(kr_fsub(kr_fmul(x.x, c.x), kr_fmul(x.y, s.x)), kr_fadd(kr_fmul(x.x, s.x), kr_fmul(x.y, c.x)),
                                kr_fsub(kr_fmul(x.z, c.y), kr_fmul(x.w, s.y)), kr_fadd(kr_fmul(x.z, s.y), kr_fmul(x.w, c.y)));
            }
        }
    }
    if (l == 0) kr_report(fault, bad);
    if (isq) {
        if (live) *(float4 *)(a.qo + (size_t)t * a.ldqo + (size_t)h * hd + 4 * l) = x;
        return;
    }
    if (!keep) return;
    pg_store<KT>(isk ? p.k : p.v, isk ? p.kd : p.vd, kr_page_row(page, p.n_kv, kvh, p.shift, row), hd, x, l, live, n);
}

template <int KT> __device__ __forceinline__ float4 pg_load4(const void *src, const float *d, size_t at, int hd, int l) {
    const size_t e = at * hd + 4 * l;
    if (KT == PG_F32) return *(const float4 *)((const float *)src + e);
    if (KT == PG_F16) {
        const ushort4 h = *(const ushort4 *)((const uint16_t *)src + e);
        return make_float4(kr_h2f(h.x), kr_h2f(h.y), kr_h2f(h.z), kr_h2f(h.w));
    }
    const char4 c = *(const char4 *)((const int8_t *)src + e);
    const float s = d[at];
    return make_float4(kr_fmul((float)c.x, s), kr_fmul((float)c.y, s), kr_fmul((float)c.z, s), kr_fmul((float)c.w, s));
}

template <int KT> __global__ void __launch_bounds__(PG_T) k_paged_load(const PgView p, float *k, size_t ldk, float *v, size_t ldv,
                                                                       int n_rows, const int *seqs, const int *rows, int lps, int *fault) {
    const unsigned n = 1u << lps, per = 2 * p.n_kv, item = (blockIdx.x * PG_T + threadIdx.x) >> lps;
    const int l = (int)(threadIdx.x & (n - 1));
    if (item >= n_rows * per || 4 * l >= p.hd) return;
    const int i = (int)(item / per), h = (int)(item % per), kvh = h < p.n_kv ? h : h - p.n_kv;
    int bad = 0;
    const int seq = kr_page_in(seqs[i], p.n_seq, KR_BAD_SEQ, bad), row = kr_page_in(rows[i], INT_MAX, KR_BAD_PAGE, bad);
    const size_t at = kr_page_row(pg_page(p, seq, row, bad), p.n_kv, kvh, p.shift, row);
    const bool isk = h < p.n_kv;
    float4 x = make_float4(0, 0, 0, 0);
    if (!bad) x = pg_load4<KT>(isk ? p.k : p.v, isk ? p.kd : p.vd, at, p.hd, l);
    if (l == 0) kr_report(fault, bad);
    *(float4 *)((isk ? k + (size_t)i * ldk : v + (size_t)i * ldv) + (size_t)kvh * p.hd + 4 * l) = x;
}

// ---- eviction ----

// Weights in an order of unsigned integers: larger is heavier, NaN the
// heaviest, -0 as +0
__device__ __forceinline__ unsigned ev_key(float w) {
    const unsigned u = __float_as_uint(w == 0.0f ? 0.0f : w);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (u >> 31) ? ~u : u | 0x80000000u;
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

// Inclusive sums over the wave's lanes
__device__ __forceinline__ int ev_scan(int v) {
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(v, o);
        if ((int)(threadIdx.x & 63) >= o) v += t;
    }
    return v;
}

// EV_U rows of 64 from r0 on for each lane, none past r1
template <class F> __device__ __forceinline__ void ev_rows(const float *mass, int r0, int r1, F f) {
    const int lane = threadIdx.x & 63;
    for (int r = r0 + lane; r - lane < r1; r += 64 * EV_U) {
        float w[EV_U];
#pragma unroll
        for (int k = 0; k < EV_U; k++) w[k] = mass[min(r + 64 * k, r1 - 1)];
#pragma unroll
        for (int k = 0; k < EV_U; k++)
            if (r - lane + 64 * k < r1) f(r + 64 * k, r + 64 * k < r1, w[k]);
    }
}

// One workgroup a (sequence, KV head): the weight of the last row kept by a
// radix select, then the kept rows' numbers in order, equal weights from the
// lowest row on. Each wave has an even part of the rows. Bound by the passes'
// latencies: the rows come from L2 after the first (32,001 rows, 8 workgroups:
// 102 us with one lane looking through the digits' counts and barriers every 1024 rows).
__global__ void __launch_bounds__(EV_T) k_evict_select(const EvArgs a, int *fault) {
    __shared__ int hist[EV_B];
    __shared__ int s_sum[EV_W], s_tie[EV_W], s_take[EV_W];
    __shared__ unsigned s_prefix;
    __shared__ int s_need;
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
    const int part = (old + EV_W - 1) / EV_W, r0 = min(old, wave * part), r1 = min(old, r0 + part);
    unsigned prefix = 0;
    int need = want;
    if (want > 0)
        for (int b = 32 - EV_D; ; b = max(0, b - EV_D)) {
            const int top = b == 32 - EV_D ? 32 : b ? 32 - EV_D : 32 - 2 * EV_D;   // bits from here up are known
            for (int i = tid; i < EV_B; i += EV_T) hist[i] = 0;
            __syncthreads();
            ev_rows(mass, r0, r1, [&](int, bool in, float w) {
                const unsigned u = ev_key(w), d = (u >> b) & ((1u << (top - b)) - 1);
                in = in && (top == 32 || (u >> top) == (prefix >> top));
                // the digit of the first lane, often that of many (zeros), counts once
                const unsigned long long any = __ballot(in);
                if (!any) return;
                const unsigned d0 = (unsigned)__builtin_amdgcn_readlane((int)d, __builtin_ctzll(any));
                const unsigned long long same = __ballot(in && d == d0);
                if (lane == __builtin_ctzll(any)) atomicAdd(&hist[d0], (int)__popcll(same));
                else if (in && d != d0) atomicAdd(&hist[d], 1);
            });
            __syncthreads();
            // from the heaviest digit down: where the counts' sum reaches `need`
            const int hi = EV_B - 1 - 2 * tid, c0 = hist[hi], c1 = hist[hi - 1], sum = ev_scan(c0 + c1);
            if (lane == 63) s_sum[wave] = sum;
            __syncthreads();
            int before = sum - c0 - c1;
            for (int i = 0; i < wave; i++) before += s_sum[i];
            if (before < need && before + c0 + c1 >= need) {
                const bool second = before + c0 < need;
                s_prefix = prefix | (unsigned)(second ? hi - 1 : hi) << b;
                s_need = need - before - (second ? c0 : 0);
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
            __syncthreads();
            if (b == 0) break;
        }
    // rows above `prefix`, and the first `need` of those at it
    int ties = 0, take = 0;
    if (want > 0)
        ev_rows(mass, r0, r1, [&](int, bool in, float w) {
            const unsigned u = ev_key(w);
            ties += __popcll(__ballot(in && u == prefix));
            take += __popcll(__ballot(in && u > prefix));
        });
    if (lane == 0) {
        s_tie[wave] = ties;
        s_take[wave] = take;
    }
    __syncthreads();
    int at = 0;
    ties = 0;
    for (int i = 0; i < wave; i++) {
        ties += s_tie[i];
        at += s_take[i];
    }
    at += min(ties, need);
    if (want > 0)
        ev_rows(mass, r0, r1, [&](int r, bool in, float w) {
            const unsigned u = ev_key(w);
            const unsigned long long bt = __ballot(in && u == prefix), below = ((unsigned long long)1 << lane) - 1;
            const bool take = in && (u > prefix || (u == prefix && ties + __popcll(bt & below) < need));
            const unsigned long long bk = __ballot(take);
            if (take) {
                const int j = at + __popcll(bk & below);
                idx[j] = r;
                ow[j] = w;
            }
            ties += __popcll(bt);
            at += __popcll(bk);
        });
    for (int r = tid; r < a.recent; r += EV_T) {
        idx[want + r] = old + r;
        ow[want + r] = mass[old + r];
    }
}

// Rows into the new pages, in units of U bytes, EM_ROWS a workgroup and KV
// head; their weights, and zeros past them. Bound by HBM: each row read once
// and written once (16 sequences of up to 4096 rows, 8B shape, half kept: 4.7
// TB/s).
constexpr int EM_ROWS = 64;
template <class U> __global__ void __launch_bounds__(PG_T) k_evict_move(const PgView p, const EvArgs a, int rb, int *fault) {
    const int s = blockIdx.z, kvh = blockIdx.y, per = rb / (int)sizeof(U), kept = a.cnt[s], tid = threadIdx.x;
    const size_t sh = (size_t)s * p.n_kv + kvh;
    const int *idx = a.idx + sh * a.keep, *ot = a.out_table + (size_t)s * a.out_ld;
    if (blockIdx.x == 0 && kvh == 0 && tid == 0) a.out_len[s] = kept;
    int bad = 0;
    const int j0 = blockIdx.x * EM_ROWS, n = min(kept - j0, EM_ROWS) * per;
    for (int e = tid; e < n; e += PG_T) {
        const int j = j0 + e / per, u = e % per, r = idx[j];
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
                   (!cos_t || (pos && n_pos > 0)) && (n_heads == 0 || (!q_norm) == (!k_norm)), "paged_qkv: a missing array") ||
        pg_refuse(ldk >= kvd && ldv >= kvd && ldk % 4 == 0 && ldv % 4 == 0 && pg_aligned(k) && pg_aligned(v) && pg_aligned(k_norm) &&
                   pg_aligned(cos_t) && pg_aligned(sin_t) &&
                   (n_heads == 0 || (ldq >= qd && ldqo >= qd && ldq % 4 == 0 && ldqo % 4 == 0 && pg_aligned(q) &&
                                     pg_aligned(qo) && pg_aligned(q_norm))), "paged_qkv: row strides or alignment"))
        return;
    const int lps = pg_log2(kv->head_dim / 4);
    const unsigned grid = item_blocks((size_t)ntok * (n_heads + 2 * (size_t)kv->n_kv_heads), lps);
    if (pg_refuse(grid > 0, "paged_qkv: too many tokens")) return;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const QkvArgs a = { qo, q, k, v, q_norm, k_norm, cos_t, sin_t, seq, row, pos, ldqo, ldq, ldk, ldv, eps, ntok, n_heads, n_pos };
    const auto f = kv->kv_type == ML_F32 ? k_paged_qkv<PG_F32> : kv->kv_type == ML_F16 ? k_paged_qkv<PG_F16> : k_paged_qkv<PG_Q8>;
    hipLaunchKernelGGL(f, dim3(grid), dim3(PG_T), 0, kr_stream(), p, a, lps, kr_fault_word());
    kr_check_launch("paged_qkv");
}

extern "C" void krh_paged_load(float *k, size_t ldk, float *v, size_t ldv, const krh_pages *kv, const int *table,
                               int table_ld, int n_seq, int n, const int *seq, const int *row) {
    if (pg_refuse(pg_pages_ok(kv), "paged_load: the pages") || pg_refuse(n >= 0 && n_seq > 0 && table_ld > 0, "paged_load sizes")) return;
    if (n == 0) return;
    const size_t kvd = (size_t)kv->n_kv_heads * kv->head_dim;
    if (pg_refuse(table && k && v && seq && row, "paged_load: a missing array") ||
        pg_refuse(ldk >= kvd && ldv >= kvd && ldk % 4 == 0 && ldv % 4 == 0 && pg_aligned(k) && pg_aligned(v),
               "paged_load: row strides or alignment"))
        return;
    const int lps = pg_log2(kv->head_dim / 4);
    const unsigned grid = item_blocks((size_t)n * 2 * kv->n_kv_heads, lps);
    if (pg_refuse(grid > 0, "paged_load: too many rows")) return;
    const auto f = kv->kv_type == ML_F32 ? k_paged_load<PG_F32> : kv->kv_type == ML_F16 ? k_paged_load<PG_F16> : k_paged_load<PG_Q8>;
    hipLaunchKernelGGL(f, dim3(grid), dim3(PG_T), 0, kr_stream(), pg_view(kv, table, table_ld, n_seq), k, ldk, v, ldv, n, seq, row,
                       lps, kr_fault_word());
    kr_check_launch("paged_load");
}

extern "C" size_t krh_paged_evict_ws(int n_seq, int n_kv_heads, int keep) {
    if (n_seq <= 0 || n_kv_heads <= 0 || keep <= 0) return 0;
    return sizeof(int) * (2 * (size_t)n_seq * n_kv_heads * keep + n_seq);
}

extern "C" void krh_paged_evict(const krh_pages *kv, const int *table, int table_ld, const int *len, const float *mass,
                                size_t mass_ld, int n_seq, int max_len, int keep, int recent, const int *out_table,
                                int out_table_ld, int *out_len, float *out_mass, size_t out_ld, void *ws) {
    if (n_seq == 0) return;
    if (pg_refuse(pg_pages_ok(kv), "paged_evict: the pages") ||
        pg_refuse(n_seq > 0 && n_seq <= KRH_ROWS_MAX && max_len > 0 && keep > 0 && recent >= 0 && recent <= keep && table_ld > 0 &&
                   out_table_ld > 0, "paged_evict sizes") ||
        pg_refuse(table && len && mass && out_table && out_len && out_mass && ws && !((uintptr_t)ws & 3) && out_table != table,
               "paged_evict: a missing array, or the pages onto themselves") ||
        pg_refuse(mass_ld >= (size_t)max_len && out_ld >= (size_t)keep && (out_mass != mass || out_ld == mass_ld),
               "paged_evict: mass rows") ||
        pg_refuse((size_t)out_table_ld * kv->page_size >= (size_t)(keep < max_len ? keep : max_len), "paged_evict: out_table's pages"))
        return;
    int *w = (int *)ws;
    const size_t rows = (size_t)n_seq * kv->n_kv_heads * keep;
    const EvArgs a = { len, mass, mass_ld, max_len, keep, recent, out_table, out_table_ld, out_len, out_mass, out_ld,
                       w + 2 * rows, w, (float *)(w + rows) };
    hipLaunchKernelGGL(k_evict_select, dim3(kv->n_kv_heads, n_seq), dim3(EV_T), 0, kr_stream(), a, kr_fault_word());
    kr_check_launch("paged_evict");
    const int rb = kv->head_dim * (kv->kv_type == ML_F32 ? 4 : kv->kv_type == ML_F16 ? 2 : 1), most = keep < max_len ? keep : max_len;
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    hipLaunchKernelGGL(rb % 16 ? k_evict_move<uint2> : k_evict_move<uint4>,
                       dim3((most + EM_ROWS - 1) / EM_ROWS, kv->n_kv_heads, n_seq), dim3(PG_T), 0, kr_stream(), p, a, rb,
                       kr_fault_word());
    kr_check_launch("paged_evict");
}
