// What stands between two blocks of a layer (krh_block_norm): the norm of a
// block's output, its gate, the residual add and the next block's norm, whose
// result leaves as floats or as 8-bit rows for krh_matmul_i8; and such rows
// back as floats.
//
// A row is one workgroup's, its values in registers from the one read to the
// one write: x' = x + alpha (gate (y / rms(y)) post), z = (x' / rms(x')) pre,
// q = z's 8-bit row. Three sums over the row at most (two of squares, in 64
// bits, and the largest |z|) are all that its threads wait for each other for.
//
// Bound by HBM with many rows, 16 bytes a value (13 with 8-bit rows): 2047 rows of
// 4096 29.0 us (4.6 TB/s), 8000 97 (5.4), 2047 of 2048 12.6 (5.3); the sums' 64-bit
// products, two a value, hide behind it. By the launch and three waits of a row with
// few: 16 rows of 4096 4.6 us, as long as any small launch takes here. One pass in place of
// the five calls that do the same in turn, whose values pass through memory each time.
#include "kr_internal.h"
#include "kr_numerics.h"

namespace {

// values a thread. With 8, twice the threads: 16 rows of 4096 as long, 8000 94.8 us instead of 97.4, 2047 of 8192 55.6
// instead of 53.8, and rows of 16,384 have no workgroup; with 4, 8000 rows 110.3
constexpr int BN_K = 4, BN_V = 4 * BN_K;
constexpr int BN_MAX = 1024 * BN_V;

struct BnArgs {
    float *xo, *z, *d;
    int8_t *q;
    const float *x, *y, *post, *gate, *pre;
    size_t ldxo, ldx, ldy, ldg, ldz, ldq;
    float alpha, eps;
    double inv_n;
    int n;
};

// 1 / sqrt(x) to a last bit or two of 64 by two steps from the instruction's estimate
__device__ __forceinline__ double bn_rsqrt(double x) {
    if (!(x > 0.0 && x < (double)INFINITY)) return 1.0 / sqrt(x);
    double r = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; i++) r = __builtin_fma(r * 0.5, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}

// over all threads of the workgroup, the same in each
template <int T, class V, class F> __device__ __forceinline__ V bn_reduce(V v, V *s, F f) {
    for (int o = 32; o >= 1; o >>= 1) v = f(v, __shfl_xor(v, o));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int i = 1; i < T / 64; i++) v = f(v, s[i]);
    }
    return v;
}

// Values k, c of a thread: four in a row with VEC, else T apart
template <int T, bool VEC> __device__ __forceinline__ int bn_at(int k, int c) {
    return VEC ? (k * T + (int)threadIdx.x) * 4 + c : (k * 4 + c) * T + (int)threadIdx.x;
}
template <int T, bool VEC> __device__ __forceinline__ void bn_get(float (&v)[BN_K][4], const float *p, int n) {
#pragma unroll
    for (int k = 0; k < BN_K; k++) {
        if constexpr (VEC) {
            const int i = bn_at<T, VEC>(k, 0);
            const float4 x = i < n ? *(const float4 *)(p + i) : make_float4(0, 0, 0, 0);
            v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = bn_at<T, VEC>(k, c);
                v[k][c] = i < n ? p[i] : 0.0f;
            }
        }
    }
}
template <int T, bool VEC> __device__ __forceinline__ void bn_put(float *p, const float (&v)[BN_K][4], int n) {
#pragma unroll
    for (int k = 0; k < BN_K; k++) {
        if constexpr (VEC) {
            const int i = bn_at<T, VEC>(k, 0);
            if (i < n) *(float4 *)(p + i) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = bn_at<T, VEC>(k, c);
                if (i < n) p[i] = v[k][c];
            }
        }
    }
}

// v = (v / rms) w
template <int T> __device__ __forceinline__ void bn_scale(float (&v)[BN_K][4], const float (&w)[BN_K][4], const BnArgs &a, double *s) {
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < BN_K; k++)
#pragma unroll
        for (int c = 0; c < 4; c++) ss = __builtin_fma((double)v[k][c], (double)v[k][c], ss);
    ss = bn_reduce<T>(ss, s, [](double x, double y) { return x + y; });
    const float inv = (float)bn_rsqrt(__builtin_fma(ss, a.inv_n, (double)a.eps));
#pragma unroll
    for (int k = 0; k < BN_K; k++)
#pragma unroll
        for (int c = 0; c < 4; c++) v[k][c] = kr_fmul(kr_fmul(v[k][c], inv), w[k][c]);
}

template <int T, bool VEC> __global__ void __launch_bounds__(T) k_block_norm(const BnArgs a) {
    __shared__ double s_sum[2][T / 64];
    __shared__ unsigned s_max[T / 64];
    const size_t r = blockIdx.x;
    const int n = a.n;
    float x[BN_K][4], w[BN_K][4];
    bn_get<T, VEC>(x, a.x + r * a.ldx, n);
    if (a.y) {
        float y[BN_K][4];
        bn_get<T, VEC>(y, a.y + r * a.ldy, n);
        if (a.post) {
            bn_get<T, VEC>(w, a.post, n);
            bn_scale<T>(y, w, a, s_sum[0]);
        }
        if (a.gate) {
            bn_get<T, VEC>(w, a.gate + r * a.ldg, n);
#pragma unroll
            for (int k = 0; k < BN_K; k++)
#pragma unroll
                for (int c = 0; c < 4; c++) y[k][c] = kr_fmul(y[k][c], w[k][c]);
        }
#pragma unroll
        for (int k = 0; k < BN_K; k++)
#pragma unroll
            for (int c = 0; c < 4; c++) x[k][c] = kr_fadd(x[k][c], kr_fmul(y[k][c], a.alpha));
    }
    if (a.xo) bn_put<T, VEC>(a.xo + r * a.ldxo, x, n);
    if (!a.pre) return;
    bn_get<T, VEC>(w, a.pre, n);
    bn_scale<T>(x, w, a, s_sum[1]);
    if (a.z) bn_put<T, VEC>(a.z + r * a.ldz, x, n);
    if (!a.q) return;
    // the largest |z| by its bits, in which a NaN is larger still: such a row's scale is NaN
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < BN_K; k++)
#pragma unroll
        for (int c = 0; c < 4; c++) m = max(m, __float_as_uint(x[k][c]) & 0x7fffffffu);
    const float amax = __uint_as_float(bn_reduce<T>(m, s_max, [](unsigned x, unsigned y) { return max(x, y); }));
    const bool zero = amax < KR_QUANT_TINY;
    const float id = zero ? 0.0f : kr_fdiv(127.0f, amax);
    if (threadIdx.x == 0) a.d[r] = zero ? 0.0f : kr_fdiv(amax, 127.0f);
    int8_t *q = a.q + r * a.ldq;
#pragma unroll
    for (int k = 0; k < BN_K; k++) {
        unsigned word = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const unsigned e = zero ? 0u : (unsigned)kr_q8_elem(x[k][c], id) & 255u;
            if constexpr (VEC) {
                word |= e << 8 * c;
            } else {
                const int i = bn_at<T, VEC>(k, c);
                if (i < n) q[i] = (int8_t)e;
            }
        }
        if constexpr (VEC) {
            const int i = bn_at<T, VEC>(k, 0);
            if (i < n) *(unsigned *)(q + i) = word;
        }
    }
}

// By HBM, 5 bytes a value: 2047 rows of 4096 8.1 us (5.2 TB/s)
constexpr int DQ_T = 256;
template <bool VEC>
__global__ void __launch_bounds__(DQ_T) k_dequantize_row(float *x, size_t ldx, const int8_t *q, size_t ldq, const float *d,
                                                         size_t ldd, int n) {
    const size_t r = blockIdx.y;
    const float s = d[r * ldd];
    x += r * ldx;
    q += r * ldq;
    if constexpr (VEC) {
        const unsigned i = (blockIdx.x * DQ_T + threadIdx.x) * 4;
        if (i >= (unsigned)n) return;
        const char4 c = *(const char4 *)(q + i);
        *(float4 *)(x + i) = make_float4(kr_fmul(c.x, s), kr_fmul(c.y, s), kr_fmul(c.z, s), kr_fmul(c.w, s));
    } else {
        const unsigned i = blockIdx.x * DQ_T + threadIdx.x;
        if (i < (unsigned)n) x[i] = kr_fmul((float)q[i], s);
    }
}

bool bn_refuse(bool ok, const char *what) {
    if (!ok) kr_fail(ML_E_SHAPE, what, hipSuccess);
    return !ok;
}
bool bn_not_ready(const char *what) {
    if (!kr_stream()) kr_fail(ML_E_ISA, what, hipSuccess);
    return !kr_stream();
}

}  // namespace

extern "C" void krh_block_norm(float *xo, size_t ldxo, const float *x, size_t ldx, const float *y, size_t ldy,
                               const float *post, const float *gate, size_t ldg, float alpha, const float *pre,
                               float eps, float *z, size_t ldz, int8_t *q, size_t ldq, float *d, int n, int rows) {
    if (bn_refuse(n > 0 && n <= BN_MAX && rows >= 0 && rows <= KRH_ROWS_MAX, "block_norm sizes")) return;
    if (rows == 0) return;
    if (bn_refuse(x && (xo || z || q) && (pre || (!z && !q)) && (y || (!post && !gate)) && !q == !d,
                  "block_norm: a missing array") ||
        bn_refuse(ldx >= (size_t)n && (!xo || ldxo >= (size_t)n) && (!y || ldy >= (size_t)n) &&
                      (!gate || ldg == 0 || ldg >= (size_t)n) && (!z || ldz >= (size_t)n) && (!q || ldq >= (size_t)n),
                  "block_norm: row strides") ||
        // rows pass in no order: with strides apart one's output would lie on another's input
        bn_refuse(rows == 1 || ((xo != x || ldxo == ldx) && (!xo || xo != y || ldxo == ldy) && (z != x || ldz == ldx) &&
                                (!z || z != y || ldz == ldy)),
                  "block_norm: a row in place with another stride") ||
        bn_not_ready("block_norm before krh_init"))
        return;
    BnArgs a = {};
    a.xo = xo, a.z = z, a.d = d, a.q = q, a.x = x, a.y = y, a.post = post, a.gate = gate, a.pre = pre;
    a.ldxo = ldxo, a.ldx = ldx, a.ldy = ldy, a.ldg = ldg, a.ldz = ldz, a.ldq = ldq;
    a.alpha = alpha, a.eps = eps, a.inv_n = 1.0 / n, a.n = n;
    auto quads = [](const void *p, size_t ld, int bytes) { return !p || (!((uintptr_t)p & (4 * bytes - 1)) && ld % 4 == 0); };
    const bool vec = n % 4 == 0 && quads(xo, ldxo, 4) && quads(x, ldx, 4) && quads(y, ldy, 4) && quads(post, 0, 4) &&
                     quads(gate, ldg, 4) && quads(pre, 0, 4) && quads(z, ldz, 4) && quads(q, ldq, 1);
    const auto launch = [&](auto f, int threads) {
        hipLaunchKernelGGL(f, dim3(rows), dim3(threads), 0, kr_stream(), a);
        kr_check_launch("block_norm");
    };
    // the fewest threads whose registers hold a row: 2047 rows of 2048 by 128 threads 12.6 us, by 256 14.4; of 8192 by
    // 512 53.8, by 1024 64.1
    if (n <= 64 * BN_V) {
        launch(vec ? k_block_norm<64, true> : k_block_norm<64, false>, 64);
    } else if (n <= 128 * BN_V) {
        launch(vec ? k_block_norm<128, true> : k_block_norm<128, false>, 128);
    } else if (n <= 256 * BN_V) {
        launch(vec ? k_block_norm<256, true> : k_block_norm<256, false>, 256);
    } else if (n <= 512 * BN_V) {
        launch(vec ? k_block_norm<512, true> : k_block_norm<512, false>, 512);
    } else {
        launch(vec ? k_block_norm<1024, true> : k_block_norm<1024, false>, 1024);
    }
}

extern "C" void krh_dequantize_row_rows(float *x, size_t ldx, const int8_t *q, size_t ldq, const float *d, size_t ldd,
                                        int n, int rows) {
    if (bn_refuse(n >= 0 && rows >= 0 && rows <= KRH_ROWS_MAX, "dequantize_row sizes")) return;
    if (n == 0 || rows == 0) return;
    if (bn_refuse(x && q && d, "dequantize_row: a missing array") ||
        bn_refuse(ldx >= (size_t)n || rows == 1, "dequantize_row: rows on each other") ||
        bn_not_ready("dequantize_row before krh_init"))
        return;
    const bool vec = n % 4 == 0 && !((uintptr_t)x & 15) && ldx % 4 == 0 && !((uintptr_t)q & 3) && ldq % 4 == 0;
    const unsigned per = vec ? DQ_T * 4 : DQ_T;
    hipLaunchKernelGGL(vec ? k_dequantize_row<true> : k_dequantize_row<false>, dim3(((unsigned)n + per - 1) / per, rows),
                       dim3(DQ_T), 0, kr_stream(), x, ldx, q, ldq, d, ldd, n);
    kr_check_launch("dequantize_row");
}
