// Rules on a batch of logit rows before the draw: penalties for the ids a
// sequence has seen, per-id biases and token masks, in one pass.
//
// A workgroup takes RL_N ids of one row: it counts the row's seen ids that
// fall among them in LDS (integer atomics: the order does not matter) and
// finds the last bias pair of each (a maximum of pair numbers), then passes
// over the logits once. Bound by HBM: 8 bytes a logit, when the seen ids are few.
#include "kr_internal.h"
#include "kr_numerics.h"
#include "kr_paged.h"

namespace {

constexpr int RL_T = 256, RL_N = 4096;

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

__global__ void __launch_bounds__(RL_T) k_logit_rules(const RlArgs a, int *fault) {
    __shared__ int cnt[RL_N];
    __shared__ int last[RL_N];
    const int tid = threadIdx.x, i0 = blockIdx.x * RL_N, n = min(RL_N, a.n - i0);
    const size_t r = blockIdx.y;
    const krh_logit_rule p = a.rule[r];
    int bad = 0;
    for (int i = tid; i < n; i += RL_T) {
        cnt[i] = 0;
        last[i] = -1;
    }
    __syncthreads();
    if (a.seen) {
        const int m = kr_page_len(a.n_seen[r], (int)a.seen_ld, bad);
        for (int j = tid; j < m; j += RL_T) {
            const int t = a.seen[r * a.seen_ld + j] - i0;
            if (t >= 0 && t < n) atomicAdd(&cnt[t], 1);
        }
    }
    if (a.bias_id) {
        const int m = kr_page_len(a.n_bias[r], (int)a.bias_ld, bad);
        for (int j = tid; j < m; j += RL_T) {
            const int t = a.bias_id[r * a.bias_ld + j] - i0;
            if (t >= 0 && t < n) atomicMax(&last[t], j);
        }
    }
    int mask = p.mask;
    if (mask < -1 || mask >= a.n_masks) {
        bad |= KR_BAD_LEN;
        mask = -1;
    }
    if (tid == 0) kr_report(fault, bad);
    __syncthreads();
    const unsigned *bits = mask >= 0 ? a.masks + (size_t)mask * (((size_t)a.n + 31) / 32) : nullptr;
    for (int i = tid; i < n; i += RL_T) {
        float x = a.logits[r * a.ld + i0 + i];
        const int c = cnt[i], b = last[i];
        if (c > 0) {
            x = x > 0.0f ? kr_fdiv(x, p.repeat) : kr_fmul(x, p.repeat);
            x = kr_fsub(kr_fsub(x, kr_fmul(p.frequency, (float)c)), p.presence);
        }
        if (b >= 0) x = kr_fadd(x, a.bias[r * a.bias_ld + b]);
        if (bits && !(bits[(i0 + i) >> 5] >> ((i0 + i) & 31) & 1)) x = -INFINITY;
        a.out[r * a.ldo + i0 + i] = x;
    }
}

}  // namespace

extern "C" void krh_logit_rules(float *out, size_t ldo, const float *logits, size_t ld, int n, int rows,
                                const krh_logit_rule *rule, const int *seen, size_t seen_ld, const int *n_seen,
                                const int *bias_id, const float *bias, size_t bias_ld, const int *n_bias,
                                const uint32_t *masks, int n_masks) {
    const bool sizes = n > 0 && rows >= 0 && rows <= KRH_ROWS_MAX && n_masks >= 0 && seen_ld <= INT32_MAX && bias_ld <= INT32_MAX &&
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
    const RlArgs a = { out, logits, ldo, ld, rule, seen, n_seen, bias_id, n_bias, bias, seen_ld, bias_ld, masks, n, n_masks };
    hipLaunchKernelGGL(k_logit_rules, dim3((n + RL_N - 1) / RL_N, rows), dim3(RL_T), 0, kr_stream(), a, kr_fault_word());
    kr_check_launch("logit_rules");
}
