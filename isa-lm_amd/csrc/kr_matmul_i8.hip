// Products of 8-bit integers with a scale a token and a scale an output
// (krh_matmul_i8, krh_matmul_i8_swiglu): Y[t][r] = (sum_k W[r][k] x[t][k]) xd[t] wd[r].
//
// The sums are exact in 32 bits whatever their order, so the reduction is split
// and its parts are joined freely, and every form gives the same bits: one
// float conversion and two products an output.
#include "kr_internal.h"
#include "kr_numerics.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int I8_COLS = (1 << 17) - 1;   // 2^14 * cols < 2^31

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

// 16 bytes of a row from k on; those past its end are zeros (the row's stride
// holds whole 16 bytes)
__device__ __forceinline__ v4i i8_get(const int8_t *row, int k, int cols) {
    v4i v = {};
    if (k < cols) v = *(const v4i *)(row + k);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = cols - k - 4 * i;
        if (left < 4) v[i] = left <= 0 ? 0 : v[i] & (int)((1u << 8 * left) - 1);
    }
    return v;
}

__device__ __forceinline__ float i8_scaled(int sum, float xd, float wd) { return kr_fmul(kr_fmul((float)sum, xd), wd); }
__device__ __forceinline__ float i8_silu_mul(float g, float u) {
    return kr_fmul(kr_fdiv(g, kr_fadd(1.0f, kr_expf(-g))), u);
}
// the output of token t and row r from its sums
template <bool GLU> __device__ __forceinline__ void i8_out(const I8Args &a, int t, int r, int s0, int s1) {
    float v = i8_scaled(s0, a.xd[t], a.wd[0][r]);
    float *y = a.y + (size_t)t * a.ldy + r;
    if constexpr (GLU) {
        *y = i8_silu_mul(v, i8_scaled(s1, a.xd[t], a.wd[1][r]));
    } else {
        if (a.bias) v = kr_fadd(v, a.bias[r]);
        *y = a.add ? kr_fadd(*y, v) : v;
    }
}

// Few tokens: a workgroup has 16 rows (of both matrices) and 16 NT tokens, its
// waves parts of the reduction, each read straight into operand registers; the
// parts' sums meet in LDS.
constexpr int FEW_W = 8, FEW_T = 64 * FEW_W;
template <int NT, bool GLU> __global__ void __launch_bounds__(FEW_T) k_i8_few(const I8Args a) {
    constexpr int M = GLU ? 2 : 1;
    __shared__ v4i s_sum[FEW_W][M][NT][64];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * NT;
    const int8_t *w[M], *x[NT];
#pragma unroll
    for (int m = 0; m < M; m++) w[m] = a.w[m] + (size_t)min(r0 + n, a.rows - 1) * a.ldw[m];
#pragma unroll
    for (int j = 0; j < NT; j++) x[j] = a.x + (size_t)min(t0 + 16 * j + n, a.ntok - 1) * a.ldx;
    v4i acc[M][NT] = {};
    // 64 values a step, steps in turn over the waves
    for (int k0 = wave * 64; k0 < a.cols; k0 += FEW_W * 64) {
        const int k = k0 + 16 * g;
        v4i xv[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) xv[j] = i8_get(x[j], k, a.cols);
#pragma unroll
        for (int m = 0; m < M; m++) {
            const v4i wv = i8_get(w[m], k, a.cols);
#pragma unroll
            for (int j = 0; j < NT; j++) acc[m][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv[j], acc[m][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int j = 0; j < NT; j++) s_sum[wave][m][j][lane] = acc[m][j];
    __syncthreads();
    // an output a thread: row r of the tile is component r % 4 of lane 16 (r / 4) + token
    for (int i = threadIdx.x; i < 256 * NT; i += FEW_T) {
        const int r = i & 15, t = i >> 4, l = 16 * (r >> 2) + (t & 15);
        int sum[2] = { 0, 0 };
#pragma unroll
        for (int v = 0; v < FEW_W; v++)
#pragma unroll
            for (int m = 0; m < M; m++) sum[m] += ((const int *)&s_sum[v][m][t >> 4][l])[r & 3];
        if (r0 + r < a.rows && t0 + t < a.ntok) i8_out<GLU>(a, t0 + t, r0 + r, sum[0], sum[1]);
    }
}

template <bool GLU> void i8_launch(const I8Args &a, const char *what) {
    const int nt = a.ntok <= 16 ? 1 : a.ntok <= 32 ? 2 : 4;
    const auto f = nt == 1 ? k_i8_few<1, GLU> : nt == 2 ? k_i8_few<2, GLU> : k_i8_few<4, GLU>;
    hipLaunchKernelGGL(f, dim3((a.rows + 15) / 16, (a.ntok + 16 * nt - 1) / (16 * nt)), dim3(FEW_T), 0, kr_stream(), a);
    kr_check_launch(what);
}

bool i8_refuse(bool ok, const char *what) {
    if (!ok) kr_fail(ML_E_SHAPE, what, hipSuccess);
    return !ok;
}
bool i8_not_ready(const char *what) {
    if (!kr_stream()) kr_fail(ML_E_ISA, what, hipSuccess);
    return !kr_stream();
}
bool i8_aligned(const void *p) { return !((uintptr_t)p & 15); }
bool i8_mat_ok(const krh_mat8 *w) {
    return w && w->q && w->d && i8_aligned(w->q) && w->rows > 0 && w->rows <= INT32_MAX - 1024 && w->cols > 0 &&
           w->cols <= I8_COLS && w->ld % 16 == 0 && w->ld >= (size_t)w->cols;
}
bool i8_args_ok(const krh_mat8 *w, const float *y, size_t ldy, const int8_t *xq, size_t ldx, const float *xd) {
    return y && xq && xd && i8_aligned(xq) && ldy >= (size_t)w->rows && ldx % 16 == 0 && ldx >= (size_t)w->cols;
}

}  // namespace

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
