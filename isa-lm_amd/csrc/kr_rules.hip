// Rules on a batch of logit rows before the draw: penalties for the ids a
// sequence has seen, per-id biases and token masks, in one pass.
//
// A workgroup takes RL_N ids of one row: their logits are under way while it
// counts the row's seen ids that fall among them in LDS (integer atomics: the order
// does not matter) and finds the last bias pair of each (a maximum of pair
// numbers). Bound by HBM, 8 bytes a logit, when the seen ids are few: 64 rows of
// 151,936 with 2000 seen 17.0 us, 4.6 TB/s (33 with the ids read after the
// logits, one logit a lane). 512 threads on 4096 ids fill a CU with waves; 256 threads
// 21.6 us, 1024 19.6, 512 on 8192 ids 22.7; 256 on 2048 as fast, at twice the reads of
// the seen ids.
#include "kr_internal.h"
#include "kr_numerics.h"
#include "kr_paged.h"

namespace {

constexpr int RL_T = 512, RL_N = 4096;
constexpr int RL_SEEN = 4, RL_BIAS = 2;   // ids a thread reads with the logits

struct RlArgs {
    float *out;
    const float *logits;
    size_t ldo, ld;
    const krh_logit_rule *rule;
    const int *seen, *n_seen, *bias_id, *n_bias;
    const float *bias;
    size_t seen_ld, bias_ld;
    const unsigned *masks;
    int n, n_masks;
};

struct RlRow {
    krh_logit_rule p;
    const float *bias;
};

// one logit after its penalties, bias and mask bit
__device__ __forceinline__ float rl_apply(const RlRow &r, float x, int c, int b, bool allowed) {
    if (c > 0) {
        x = x > 0.0f ? kr_fdiv(x, r.p.repeat) : kr_fmul(x, r.p.repeat);
        x = kr_fsub(kr_fsub(x, kr_fmul(r.p.frequency, (float)c)), r.p.presence);
    }
    if (b >= 0) x = kr_fadd(x, r.bias[b]);
    return allowed ? x : -INFINITY;
}

// VEC: rows of the logits and the output 16-byte aligned, four ids a lane and
// step (64 rows of 151,936 ids 17.0 us; one at a time 19.5)
template <bool VEC> __global__ void __launch_bounds__(RL_T) k_logit_rules(const RlArgs a, int *fault) {
    constexpr int V = VEC ? 4 : 1, STEPS = RL_N / (RL_T * V);
    __shared__ __align__(16) int cnt[RL_N];
    __shared__ __align__(16) int last[RL_N];
    const int tid = threadIdx.x, i0 = blockIdx.x * RL_N, n = min(RL_N, a.n - i0);
    const size_t r = blockIdx.y;
    const float *in = a.logits + r * a.ld + i0;
    float *out = a.out + r * a.ldo + i0;
    float x[STEPS][V];
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int i = (k * RL_T + tid) * V;
        if constexpr (VEC) {
            if (i + 4 <= n) {
                const float4 t = *(const float4 *)(in + i);
                x[k][0] = t.x, x[k][1] = t.y, x[k][2] = t.z, x[k][3] = t.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++) x[k][c] = i + c < n ? in[i + c] : 0.0f;
            }
        } else {
            x[k][0] = i < n ? in[i] : 0.0f;
        }
    }
    // the row's first ids, as many as count
    const RlRow row = { a.rule[r], a.bias + r * a.bias_ld };
    int n_seen = a.n_seen[r], n_bias = a.n_bias[r];
    asm("" : "+s"(n_seen), "+s"(n_bias));   // waited for together
    int bad = 0;
    const int ns = kr_page_len(a.seen ? n_seen : 0, (int)a.seen_ld, bad);
    const int nb = kr_page_len(a.bias_id ? n_bias : 0, (int)a.bias_ld, bad);
    const int *seen = a.seen + r * a.seen_ld, *ids = a.bias_id + r * a.bias_ld;
    int sj[RL_SEEN], bj[RL_BIAS];
#pragma unroll
    for (int k = 0; k < RL_SEEN; k++) sj[k] = kr_id_at(seen, k * RL_T + tid, ns);
#pragma unroll
    for (int k = 0; k < RL_BIAS; k++) bj[k] = kr_id_at(ids, k * RL_T + tid, nb);
    int mask = row.p.mask;
    if (mask < -1 || mask >= a.n_masks) {
        bad |= KR_BAD_LEN;
        mask = -1;
    }
    if (tid == 0) kr_report(fault, bad);
    if (ns > 0 || nb > 0) {
        for (int i = tid; i < RL_N / 4; i += RL_T) {
            if (ns > 0) ((int4 *)cnt)[i] = make_int4(0, 0, 0, 0);
            if (nb > 0) ((int4 *)last)[i] = make_int4(-1, -1, -1, -1);
        }
        __syncthreads();
        // ids below i0, negative ones among them, wrap past n: i0 + n <= 2^31
        auto count = [&](int id) {
            const unsigned t = (unsigned)id - (unsigned)i0;
            if (t < (unsigned)n) atomicAdd(&cnt[t], 1);
        };
        auto note = [&](int id, int j) {
            const unsigned t = (unsigned)id - (unsigned)i0;
            if (t < (unsigned)n) atomicMax(&last[t], j);
        };
#pragma unroll
        for (int k = 0; k < RL_SEEN; k++)
            if (k * RL_T + tid < ns) count(sj[k]);
#pragma unroll 4
        for (int j = RL_SEEN * RL_T + tid; j < ns; j += RL_T) count(seen[j]);
#pragma unroll
        for (int k = 0; k < RL_BIAS; k++)
            if (k * RL_T + tid < nb) note(bj[k], k * RL_T + tid);
        for (int j = RL_BIAS * RL_T + tid; j < nb; j += RL_T) note(ids[j], j);
        __syncthreads();
    }
    const unsigned *bits = a.masks + (mask >= 0 ? (size_t)mask * (((size_t)a.n + 31) / 32) : 0);
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int i = (k * RL_T + tid) * V;
        if (i >= n) break;
        const unsigned word = mask >= 0 ? bits[(i0 + i) >> 5] >> ((i0 + i) & 31) : ~0u;
#pragma unroll
        for (int c = 0; c < V; c++)
            x[k][c] = rl_apply(row, x[k][c], ns > 0 ? cnt[i + c] : 0, nb > 0 ? last[i + c] : -1, word >> c & 1);
        if constexpr (VEC) {
            if (i + 4 <= n) {
                *(float4 *)(out + i) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
                continue;
            }
        }
#pragma unroll
        for (int c = 0; c < V; c++)
            if (i + c < n) out[i + c] = x[k][c];
    }
}

}  // namespace

extern "C" void krh_logit_rules(float *out, size_t ldo, const float *logits, size_t ld, int n, int rows,
                                const krh_logit_rule *rule, const int *seen, size_t seen_ld, const int *n_seen,
                                const int *bias_id, const float *bias, size_t bias_ld, const int *n_bias,
                                const uint32_t *masks, int n_masks) {
    const bool sizes = n > 0 && rows >= 0 && rows <= KRH_ROWS_MAX && n_masks >= 0 && seen_ld <= INT32_MAX / 2 &&
                       bias_ld <= INT32_MAX / 2 &&
                       ldo >= (size_t)n && ld >= (size_t)n && (out != logits || ldo == ld);
    if (!sizes) {
        kr_fail(ML_E_SHAPE, "logit_rules sizes", hipSuccess);
        return;
    }
    if (rows == 0) return;
    if (!out || !logits || !rule || (seen && !n_seen) || (bias_id && (!bias || !n_bias)) || (n_masks > 0 && !masks)) {
        kr_fail(ML_E_SHAPE, "logit_rules: a missing array", hipSuccess);
        return;
    }
    if (!kr_fault_word()) {
        kr_fail(ML_E_ISA, "logit_rules before krh_init", hipSuccess);
        return;
    }
    // where there is no list, any readable words stand for its counts, so that a
    // launch asks for both without a branch
    const int *none = (const int *)rule;
    const RlArgs a = { out,    logits, ldo,     ld,      rule,  seen, seen ? n_seen : none, bias_id, bias_id ? n_bias : none,
                       bias,   seen_ld, bias_ld, masks, n,    n_masks };
    const bool vec = !(((uintptr_t)out | (uintptr_t)logits) & 15) && ldo % 4 == 0 && ld % 4 == 0;
    hipLaunchKernelGGL(vec ? k_logit_rules<true> : k_logit_rules<false>, dim3(((unsigned)n + RL_N - 1) / RL_N, rows), dim3(RL_T),
                       0, kr_stream(), a, kr_fault_word());
    kr_check_launch("logit_rules");
}
