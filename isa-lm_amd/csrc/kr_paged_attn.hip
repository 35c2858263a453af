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
#include "kr_paged_wave.h"

namespace {

template <int KT, int CL, bool FULL, bool FINE>
__global__ void __launch_bounds__(64, pa_waves(KT, CL)) k_paged_shares(const PgView p, const PaArgs a, int *fault) {
    const int u = blockIdx.x, kvh = blockIdx.y;
    PaWave<KT, CL, FULL, PaArgs, FINE> w(p, a, kvh);
    if (a.whole) {
        w.seq = u;
        w.sp = pa_span(a, kr_page_len(a.len[u], a.max_len, w.bad), 0);
        w.part(0, w.sp.tiles, 0);
        kr_report(fault, w.bad);
        return;
    }
    PaAll all = pa_all(p, a, w.bad, a.shares);
    if (u < all.shares) {
        int left = pa_bound(all, u + 1) - pa_bound(all, u), t = pa_bound(all, u);
        for (w.seq = pa_find(p, a, all, t, w.bad); left > 0; w.seq++, t = 0) {
            w.sp = pa_of(p, a, all, w.seq, w.bad);
            const int end = min(w.sp.tiles, t + left);
            w.part(t, end, (size_t)kvh * (p.n_seq + a.shares) + w.seq + u);
            left -= end - t;
        }
    }
    kr_report(fault, w.bad);
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
        const PaParts r = pa_parts(p, a, s, kvh, sp, a.shares);
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
    const PaParts r = pa_parts(p, a, s, kvh, sp, a.shares);
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
template <int KT, int CL, bool FINE> PaKernel pa_kernel(int hd) {
    return hd == CL ? k_paged_shares<KT, CL, true, FINE> : k_paged_shares<KT, CL, false, FINE>;
}
template <int KT, bool FINE = false> PaKernel pa_kernel(int hd) {
    return hd <= 64 ? pa_kernel<KT, 64, FINE>(hd) : hd <= 128 ? pa_kernel<KT, 128, FINE>(hd) : pa_kernel<KT, 256, FINE>(hd);
}

}  // namespace

extern "C" size_t krh_paged_attention_ws(const krh_pages *kv, int n_seq, int n_heads, int max_len, int mass) {
    if (!pa_args_ok(kv, n_seq, n_heads, max_len)) return 0;
    const PaSizes r = pa_sizes(kv, n_seq, n_heads, max_len, pa_shares(kv, n_seq, max_len), mass != 0);
    return sizeof(float) * (r.part + r.pml + r.z + 4);
}

void kr_paged_attention(bool fine, float *o, const krh_pages *kv, const int *table, int table_ld, const int *len, int n_seq,
                        const float *q, int n_heads, int max_len, int window, float scale, float softcap, float *mass,
                        size_t mass_ld, void *ws) {
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
    const PaKernel f = kv->kv_type == ML_F16   ? pa_kernel<PG_F16>(hd)
                       : kv->kv_type == ML_Q8_0 ? pa_kernel<PG_Q8>(hd)
                       : fine                   ? pa_kernel<PG_F32, true>(hd)
                                                : pa_kernel<PG_F32>(hd);
    hipLaunchKernelGGL(f, dim3(shares, kv->n_kv_heads), dim3(64), 0, kr_stream(), p, a, kr_fault_word());
    kr_check_launch("paged_attention");
    if ((shares > 1 && !whole) || mass) {
        hipLaunchKernelGGL(k_paged_join, dim3(n_heads + kv->n_kv_heads * blocks, n_seq), dim3(PJ_T), 0, kr_stream(), p, a,
                           pg_log2(hd / 4), blocks);
        kr_check_launch("paged_attention");
    }
}

extern "C" void krh_paged_attention(float *o, const krh_pages *kv, const int *table, int table_ld, const int *len,
                                    int n_seq, const float *q, int n_heads, int max_len, int window, float scale,
                                    float softcap, float *mass, size_t mass_ld, void *ws) {
    kr_paged_attention(false, o, kv, table, table_ld, len, n_seq, q, n_heads, max_len, window, scale, softcap, mass, mass_ld, ws);
}
