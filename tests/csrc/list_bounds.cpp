// The logit rules' lists (isa-lm_amd/csrc/kr_paged.h) on the host: a row of ids
// that ends with its last counted one, at a page with nothing behind it, is
// read as far as its count and no further, whatever the row's stride is.
#include "kr_paged.h"
#include <cstdio>
#include <cstdlib>
#include <sys/mman.h>
#include <unistd.h>

int main(int argc, char **argv) {
    const int trials = argc > 1 ? atoi(argv[1]) : 1000;
    const size_t ps = (size_t)sysconf(_SC_PAGESIZE);
    char *map = (char *)mmap(nullptr, 4 * ps, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (map == MAP_FAILED || mprotect(map + ps, 2 * ps, PROT_READ | PROT_WRITE)) return 9;
    int *end = (int *)(map + 3 * ps);
    const int most = (int)(2 * ps / sizeof(int));
    unsigned st = 1;
    for (int i = 0; i < trials; i++) {
        st = st * 1664525u + 1013904223u;
        const int n = (int)((st >> 8) % (most + 1)), ld = n + (int)((st >> 4) % 3000);   // the stride passes the row
        int *ids = end - n, bad = 0;
        for (int j = 0; j < n; j++) ids[j] = j + 7;
        const int counted = kr_page_len(n, ld, bad);
        for (int j = 0; j < ld; j++)
            if (kr_id_at(ids, j, counted) != (j < n ? j + 7 : -1) || bad) return 1;
        // a count that the row cannot hold is none, and none is read
        bad = 0;
        if (kr_id_at(end, 0, kr_page_len(ld + 1, ld, bad)) != -1 || !bad) return 2;
        if (kr_id_at(nullptr, 0, 0) != -1) return 3;
    }
    printf("ok %d\n", trials);
    return 0;
}
