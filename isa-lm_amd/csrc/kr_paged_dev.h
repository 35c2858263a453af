// What the paged operators' translation units share: the view of a pool and its
// sequences, and the checks of a call's arguments.
#pragma once
#include "kr_internal.h"
#include "kr_numerics.h"
#include "kr_paged.h"

enum { PG_F32 = ML_F32, PG_Q8 = ML_Q8_0, PG_F16 = ML_F16 };

// a pool and the view of its sequences
struct PgView {
    void *k, *v;
    float *kd, *vd;
    const int *table;
    int ld, n_seq, n_pages, shift, n_kv, hd;
};

__device__ __forceinline__ int pg_page(const PgView &p, int seq, int row, int &bad) {
    return kr_page_of(p.table + (size_t)seq * p.ld, p.ld, row, p.shift, p.n_pages, bad);
}

// Inclusive sums over the wave's lanes, in registers
template <int CTRL, int ROWS> __device__ __forceinline__ int pg_add_dpp(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int pg_scan(int v) {
    v = pg_add_dpp<0x111, 0xf>(v);   // from 1, 2, 4 and 8 lanes below in the row of 16
    v = pg_add_dpp<0x112, 0xf>(v);
    v = pg_add_dpp<0x114, 0xf>(v);
    v = pg_add_dpp<0x118, 0xf>(v);
    v = pg_add_dpp<0x142, 0xa>(v);   // the sums of rows 0 and 2 to rows 1 and 3
    return pg_add_dpp<0x143, 0xc>(v);   // of the lower half to the upper
}

inline int pg_log2(int v) {
    int l = 0;
    while ((1 << l) < v) l++;
    return l;
}

inline bool pg_pages_ok(const krh_pages *kv) {
    return kv && kv->k && kv->v && !(((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) && kv->n_pages > 0 &&
           kv->page_size >= KR_PAGE_MIN && kv->page_size <= KR_PAGE_MAX && !(kv->page_size & (kv->page_size - 1)) &&
           kv->n_kv_heads > 0 && kv->n_kv_heads <= KRH_ROWS_MAX && kv->head_dim >= 8 && kv->head_dim <= KR_PAGE_HD_MAX &&
           kv->head_dim % 8 == 0 &&
           (kv->kv_type == ML_F32 || kv->kv_type == ML_F16 || 
            (kv->kv_type == ML_Q8_0 && kv->kd && kv->vd && !(((uintptr_t)kv->kd | (uintptr_t)kv->vd) & 15)));
}

inline bool pg_aligned(const void *p) { return !((uintptr_t)p & 15); }

inline PgView pg_view(const krh_pages *kv, const int *table, int ld, int n_seq) {
    const bool q8 = kv->kv_type == ML_Q8_0;
    return { kv->k, kv->v, q8 ? kv->kd : nullptr, q8 ? kv->vd : nullptr, table, ld, n_seq, kv->n_pages,
             pg_log2(kv->page_size), kv->n_kv_heads, kv->head_dim };
}

inline bool pg_refuse(bool ok, const char *what) {
    if (!ok) kr_fail(ML_E_SHAPE, what, hipSuccess);
    return !ok;
}
// a kernel's reports need the fault words
inline bool pg_not_ready(const char *what) {
    if (!kr_fault_word()) kr_fail(ML_E_ISA, what, hipSuccess);
    return !kr_fault_word();
}

