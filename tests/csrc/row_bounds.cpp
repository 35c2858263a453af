// The paged cache's lookup (isa-lm_amd/csrc/kr_paged.h) of any row at all, as a
// workspace that was overwritten could hold it: a negative one is out of range,
// and nothing before the table is read (a page with nothing before it).
#include "kr_paged.h"
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <sys/mman.h>
#include <unistd.h>

int main(int argc, char **argv) {
    const int trials = argc > 1 ? atoi(argv[1]) : 1000;
    const size_t ps = (size_t)sysconf(_SC_PAGESIZE);
    char *map = (char *)mmap(nullptr, 3 * ps, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (map == MAP_FAILED || mprotect(map + ps, ps, PROT_READ | PROT_WRITE)) return 9;
    int *table = (int *)(map + ps);
    for (int j = 0; j < 8; j++) table[j] = j;
    unsigned st = 7;
    for (int i = 0; i < trials; i++) {
        st = st * 1664525u + 1013904223u;
        const int row = i == 0 ? INT_MIN : i == 1 ? -1 : (int)st, shift = 4 + (int)((st >> 20) % 7);
        int bad = 0;
        const int id = kr_page_of(table, 8, row, shift, 8, bad);
        const bool good = row >= 0 && (row >> shift) < 8;
        if (good ? id != row >> shift || bad : id != 0 || bad != KR_BAD_PAGE) {
            printf("trial %d: row %d id %d bad %d\n", i, row, id, bad);
            return 1;
        }
        if (kr_page_row(id, 2, 1, shift, row) >= (size_t)8 * 2 << shift) return 2;
    }
    printf("ok %d\n", trials);
    return 0;
}
