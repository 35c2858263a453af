// The paged cache's lookups (isa-lm_amd/csrc/kr_paged.h) on the host: whatever
// the tables, lengths and rows hold, every row number that comes out lies in
// the pool, the table's own entries alone are read, and what was out of range
// is told.
#include "kr_paged.h"
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <sys/mman.h>
#include <unistd.h>

static unsigned long long st = 88172645463325252ull;
static unsigned rnd() {
    st ^= st << 13;
    st ^= st >> 7;
    st ^= st << 17;
    return (unsigned)(st >> 16);
}

int main(int argc, char **argv) {
    const int trials = argc > 1 ? atoi(argv[1]) : 100000;
    // a page with nothing behind it, nor before it: a read past a table that ends there faults
    const size_t ps = (size_t)sysconf(_SC_PAGESIZE);
    char *map = (char *)mmap(nullptr, 3 * ps, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (map == MAP_FAILED || mprotect(map + ps, ps, PROT_READ | PROT_WRITE)) return 9;
    const int odd[] = { INT_MIN, -1, 0, 1, INT_MAX, 1 << 30, 65536 };
    for (int i = 0; i < trials; i++) {
        const int shift = 4 + rnd() % 7, ld = 1 + rnd() % 9, n_pages = 1 + rnd() % 20, n_kv = 1 + rnd() % 8;
        int *table = (int *)(i & 1 ? map + ps : map + 2 * ps - ld * sizeof(int));
        for (int j = 0; j < ld; j++) table[j] = rnd() % 4 ? (int)(rnd() % n_pages) : rnd() % 3 ? odd[rnd() % 7] : n_pages + (int)(rnd() % 2);
        const int row = rnd() % 3 ? (int)(rnd() % (unsigned)((ld + 1) << shift)) : INT_MAX - (int)(rnd() % 100);
        int bad = 0;
        const int id = kr_page_of(table, ld, row, shift, n_pages, bad);
        const bool good = (row >> shift) < ld && table[row >> shift] >= 0 && table[row >> shift] < n_pages;
        const int kvh = rnd() % n_kv;
        const size_t at = kr_page_row(id, n_kv, kvh, shift, row), rows = ((size_t)n_pages * n_kv) << shift;
        if (id < 0 || id >= n_pages || at >= rows || good != (bad == 0) || (good && id != table[row >> shift]) ||
            (good && at != ((size_t)id * n_kv + kvh) * ((size_t)1 << shift) + (size_t)row % ((size_t)1 << shift))) {
            printf("page: trial %d: row %d id %d at %zu of %zu bad %d\n", i, row, id, at, rows, bad);
            return 1;
        }
        const int most = 1 + rnd() % 100, len = rnd() % 2 ? odd[rnd() % 7] : (int)(rnd() % 200) - 50;
        bad = 0;
        const int l = kr_page_len(len, most, bad);
        if (l < 0 || l > most || (bad != 0) != (len < 0 || len > most) || (!bad && l != len) || (bad && l != 0)) return 2;
        bad = 0;
        const int k = kr_page_in(len, most, KR_BAD_SEQ, bad);
        if (k < 0 || k >= most || (bad != 0) != (len < 0 || len >= most) || (!bad && k != len)) return 3;
    }
    // a pool past 32 bits: page 70,000 of 8 heads and 1024 slots
    if (kr_page_row(70000, 8, 7, 10, 1023) != (size_t)70000 * 8192 + 7 * 1024 + 1023) return 4;
    printf("ok %d\n", trials);
    return 0;
}
