// Where a row of a paged cache lies. The tables, lengths and row numbers are
// device data that the host cannot check, so every kernel takes them through
// these functions: an id, row or length out of range is never used as an
// address (page 0, row 0 or length 0 stands in for it) and is reported to the
// host's fault words, which krh_sync turns into an error. Plain C++, so that the
// bounds can be checked on the host.
#pragma once
#include <stddef.h>

#ifdef __HIPCC__
#define KR_HD __host__ __device__ __forceinline__
#else
#define KR_HD inline
#endif

enum { KR_PAGE_MIN = 16, KR_PAGE_MAX = 1024, KR_PAGE_HD_MAX = 256, KR_PAGE_GROUP_MAX = 16, KR_PAGE_LEN_MAX = 1 << 29 };

// what a kernel found: bit i goes to fault word i
enum { KR_BAD_PAGE = 1, KR_BAD_LEN = 2, KR_BAD_SEQ = 4, KR_BAD_POS = 8, KR_FAULT_WORDS = 4 };

// The page that holds `row` of a sequence: an id in [0, n_pages), n_pages >= 1,
// whatever the table holds and `row` is; only the table's ld entries are read.
KR_HD int kr_page_of(const int *table, int ld, int row, int shift, int n_pages, int &bad) {
    const unsigned i = (unsigned)row >> shift;   // a negative row is past every table
    if (i >= (unsigned)ld) {
        bad |= KR_BAD_PAGE;
        return 0;
    }
    const int id = table[i];
    if ((unsigned)id >= (unsigned)n_pages) {
        bad |= KR_BAD_PAGE;
        return 0;
    }
    return id;
}

// Row numbers within the pool of (page, KV head, slot): page * n_kv * page_size
// passes 32 bits from 2^31 rows on, and their element offsets far earlier.
KR_HD size_t kr_page_row(int page, int n_kv, int kvh, int shift, int row) {
    return (((size_t)page * n_kv + kvh) << shift) + (row & ((1 << shift) - 1));
}

// a sequence's length, 0 where it is not in [0, most]
KR_HD int kr_page_len(int len, int most, int &bad) {
    if (len < 0 || len > most) {
        bad |= KR_BAD_LEN;
        return 0;
    }
    return len;
}

// an index in [0, n), n >= 1: 0 where it is none
KR_HD int kr_page_in(int i, int n, int what, int &bad) {
    if ((unsigned)i >= (unsigned)n) {
        bad |= what;
        return 0;
    }
    return i;
}

// entry j of a list that counts n of them, -1 past those: what lies behind the
// counted ones, up to the row's stride, may belong to no allocation
KR_HD int kr_id_at(const int *ids, int j, int n) { return j < n ? ids[j] : -1; }

#ifdef __HIPCC__
// any thread that found something bad; a store a word, so that none is lost
__device__ __forceinline__ void kr_report(int *fault, int bad) {
    if (!bad) return;
    for (int i = 0; i < KR_FAULT_WORDS; i++)
        if (bad >> i & 1) __hip_atomic_store(fault + i, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
#endif
