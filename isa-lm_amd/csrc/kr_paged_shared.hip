// Attention of one token of each sequence over a paged cache in which groups of
// sequences begin with the same rows (krh_paged_attention_shared).
//
// With few sequences a shared row is read by each (krh_paged_attention); with
// many a group's shared rows are passed over once for all of its query heads
// (k_shared_rows), its sequences' own rows as krh_paged_attention passes over a
// window (kr_paged_wave.h), and a last launch joins the parts: with each part's
// maximum m (in log2), sum l and unscaled output o, out = sum 2^(m - M) o / sum 2^(m - M) l.
//
// The shared rows are a matrix product with as many columns as the group has
// query heads of the KV head. A workgroup's waves have 32 columns each and the
// same rows, 32 at a time, which pass through LDS: S^T = K Q^T has rows as rows, so
// the lane that holds a column's scores of rows 4 h + 8 j + (0..3), h its half of
// the wave, has them as the operand P^T of O^T = V^T P^T as they are, in the order
// of rows in which V is laid down transposed (F32: a float is an operand by itself,
// so V's rows lie as they are). All products are those of kr_paged_wave.h: a float operand
// is two halves, x = hi + lo, F32 caches take the 32-bit product.
//
// The tiles of all (group, column tile) pairs are cut into equal shares, one a
// workgroup and KV head, by the lengths that the device has; a share's sums of a
// column tile are a part.
//
// What bounds it (8B shape, halves): 64 sequences behind 32,000 rows 98 to 113 us by
// the card, of which the join's reads of the parts 9; the matrix cores and the
// softmax's instructions beside each other (busy 37 and 38% of the cycles), at the 1.6 to
// 2.0 GHz of 2.4 that power leaves (67 GFLOP with both halves, 54 us of a large
// product's rate). 16 behind 2048 19.9 us: four tiles a workgroup, 1.8 us each on
// their way (the matrix cores are busy 5% of the cycles), and the join's latency, 5.8. Each sequence
// reading its own (krh_paged_attention) takes 1069 us and 26.8 there. Floats of 256
// dims, 32 behind 8192 134 us: one wave a SIMD, the matrix cores busy 17%.
#include <cfloat>
#include <cmath>
#include "kr_paged_wave.h"

namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int SH_R = 32;   // rows a tile
constexpr int SH_FEW = 8;   // tiles a share up to which a compute unit has one workgroup
constexpr int SH_WC = 4, SH_CT = 32 * SH_WC;   // waves and columns of a workgroup
struct ShArgs : PaShared {
    float *spart, *spml;   // [n_kv][column tiles + shares][SH_CT][hd] and [2]: the shared rows' parts
    int wgs, own;    // workgroups of a KV head, and of these for the sequences' own rows at least
    float weigh;     // a wave's work on a tile of those, in a workgroup's on one of the shared rows, a wave
    int sfew, sleast, slots;
    int *fault;
};

// The groups, one a lane
struct ShGroups {
    int s0, s1, rows;   // sequences [s0, s1), which share `rows` rows
};
// Starts that do not ascend within the batch leave no group; a group of one sequence is none.
__device__ __forceinline__ ShGroups sh_groups(const PgView &p, const PaShared &a, int &bad) {
    const int g = (int)(threadIdx.x & 63), i = min(g, a.n_groups - 1);
    ShGroups r = { a.group[i], a.group[i + 1], kr_page_len(a.shared[i], a.max_shared, bad) };
    if (__any(r.s0 < 0 || r.s1 < r.s0 || r.s1 > p.n_seq)) {
        bad |= KR_BAD_SEQ;
        r.s0 = r.s1 = 0;
    }
    if (g >= a.n_groups || r.s1 - r.s0 < 2) r.rows = 0;
    return r;
}
__device__ __forceinline__ int pa_skip(const PgView &p, const PaShared &a, int i, int &bad) {
    const ShGroups r = sh_groups(p, a, bad);
    int skip = 0;
    for (int g = 0; g < a.n_groups; g++) {
        const int rows = __builtin_amdgcn_readlane(r.rows, g);
        if (i >= __builtin_amdgcn_readlane(r.s0, g) && i < __builtin_amdgcn_readlane(r.s1, g)) skip = rows;
    }
    return skip;
}

__device__ __forceinline__ int sh_rts(int rows, int begin) { return (rows - begin + SH_R - 1) / SH_R; }
__device__ __forceinline__ int sh_cts(int seqs, int group) { return (seqs * group + SH_CT - 1) / SH_CT; }
// The tiles of the groups, one group a lane: `cts` column tiles of the rows from
// `begin` on in `rts` row tiles; `sum`, `csum`: inclusive sums of all tiles and of
// the column tiles
struct ShTiles {
    ShGroups g;
    int begin, rts, cts, sum, csum;
    int tiles, own;   // of all groups, and workgroups of a KV head that have the sequences' own rows
};
__device__ __forceinline__ ShTiles sh_tiles(const PgView &p, const ShArgs &a, int &bad) {
    ShTiles r;
    const int lane = (int)(threadIdx.x & 63), group = a.nh / p.n_kv;
    r.g = sh_groups(p, a, bad);
    r.begin = 0;
    if (a.window > 0) {
        // of a window the first row that any sequence of the group attends
        for (int g = 0; g < a.n_groups; g++) {
            if (__builtin_amdgcn_readlane(r.g.rows, g) == 0) continue;
            const int s1 = __builtin_amdgcn_readlane(r.g.s1, g);
            int least = INT_MAX;
            for (int s = __builtin_amdgcn_readlane(r.g.s0, g) + lane; s < s1; s += 64) {
                const int len = kr_page_len(a.len[s], a.max_len, bad);
                if (len > 0) least = min(least, max(0, len - a.window));
            }
            for (int o = 32; o >= 1; o >>= 1) least = min(least, __shfl_xor(least, o));
            if (lane == g) r.begin = min(least, r.g.rows) & -SH_R;
        }
    }
    r.rts = sh_rts(r.g.rows, r.begin);
    r.cts = r.g.rows > 0 ? sh_cts(r.g.s1 - r.g.s0, group) : 0;
    r.sum = pg_scan(r.rts * r.cts);
    r.csum = pg_scan(r.cts);
    r.tiles = __builtin_amdgcn_readlane(r.sum, 63);
    r.own = a.own;
    if (a.weigh > 0.0f) {
        // what is attended but for the shared rows, in tiles of SH_R
        int own = -(r.cts > 0 ? r.g.s1 - r.g.s0 : 0) * r.rts;
        for (int i = lane; i < p.n_seq; i += 64) {
            const int len = kr_page_len(a.len[i], a.max_len, bad);
            own += ((a.window > 0 ? min(len, a.window) : len) + SH_R - 1) / SH_R;
        }
        // (sequences shorter than their group's shared rows may leave less than nothing)
        const float w = a.weigh * (float)max(__builtin_amdgcn_readlane(pg_scan(own), 63), 0);
        const int part = __builtin_amdgcn_readfirstlane((int)((float)a.wgs * (w / (w + (float)max(r.tiles, 1)))));
        r.own = r.tiles == 0 ? a.wgs : min(max(a.own, part), a.wgs - 1);
    }
    return r;
}
// how many shares they make: as many as there are compute units, the own rows' workgroups among them, where that gives
// each a few tiles only
__device__ __forceinline__ int sh_shares(const ShArgs &a, const ShTiles &r) {
    const int most = min(r.tiles <= SH_FEW * a.sfew ? a.sfew : a.wgs, a.wgs - r.own);
    return max(1, min(most, (r.tiles + a.sleast - 1) / a.sleast));
}

__device__ __forceinline__ float sh_other(float v) {   // the same column's value in the other half of the wave
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(threadIdx.x & 32 ? s[0] : s[1]);
}

template <int KT, int CL, bool WIN> struct ShLds {
    static constexpr int EB = KT == PG_F32 ? 4 : 2;
    alignas(16) char k[2][SH_R * CL * EB];
    alignas(16) char v[2][SH_R * CL * EB];
    alignas(16) float kd[2][KT == PG_Q8 ? SH_R : 4], vd[2][KT == PG_Q8 ? SH_R : 4];
    std::conditional_t<WIN, unsigned long long, int> range[2];
    int2 col[WIN ? SH_CT : 1];   // the rows that each column attends
    int4 group[64];              // the groups: sequences, rows, and the first row of their tiles
    int2 sums[64];               // sum, csum
};

// where 16 bytes of a K row lie (F32: of a V row too): 16 rows of one chunk in all banks
template <int NC> __device__ __forceinline__ int sh_at(int row, int c) {
    return (row * NC + (c ^ (NC >= 16 ? row & 15 : (row >> 1) & 7))) * 16;
}
// 4 rows (8 c16 + 4 h + 16 s + 0..3, quad = 4 s + 2 p + h) of one dim of V in halves
__device__ __forceinline__ int sh_vt(int dim, int chunk) { return dim * 64 + ((chunk ^ ((dim >> 2) & 3)) << 4); }

constexpr int sh_waves(int kt, int cl) { return cl > 128 || (kt == PG_F32 && cl > 64) ? 1 : 2; }   // a SIMD

// WIN: there is a window, and rows that no column attends may lie between those that some do. A kernel of its own has
// such calls, so that the others' registers hold what they work on (one kernel for both: 32 sequences behind 4096 rows of
// 256 floats 88 us instead of 84, 64 behind the 8B shape's 38.6 instead of 38.0).
template <int KT, int CL, bool WIN> struct ShWork {
    static constexpr bool HALF = KT != PG_F32;
    static constexpr int NTH = 64 * SH_WC, CT = SH_CT;
    static constexpr int KC = HALF ? CL / 8 : CL / 4;          // LDS chunks of 16 bytes a row
    static constexpr int KN = (SH_R * KC + NTH - 1) / NTH;     // K chunks a thread
    static constexpr int VU = HALF ? 8 * (CL / 4) : SH_R * KC; // V's pieces: 4 rows of 4 dims, or a chunk
    static constexpr int VN = (VU + NTH - 1) / NTH;
    static constexpr int KW = KT == PG_Q8 ? 2 : 4;             // words of a K chunk in the pool
    static constexpr int VW = KT == PG_F32 ? 4 : KT == PG_F16 ? 8 : 4;
    static constexpr int KS = HALF ? CL / 16 : CL / 8;         // K operands of a row
    static constexpr int EB = KT == PG_F32 ? 4 : KT == PG_F16 ? 2 : 1, KD = HALF ? 8 : 4, VC = CL / 4;
    static_assert(16 % (64 / (KC < 64 ? KC : 64)) == 0 && 16 % (64 * (HALF ? 4 : 1) / VC) == 0, "a wave's pieces in one half of a tile");
    // log2 of what the weights are over, and by how much (log2) one may pass the maximum that it is taken from before
    // that moves: 2^13 2^2 are within the halves, and a weight's lo a whole half down to 2^-15 of the largest
    static constexpr int UP = KT == PG_F16 ? 13 : 0, SLACK = 2;
    static constexpr int DT = CL / 32;

    const PgView &p;
    const ShArgs &a;
    ShLds<KT, CL, WIN> &lds;
    const int lane, h, wave, kvh, hd, group;
    int bad;
    // the piece: rows [row0, row1) in tiles; columns here attend rows of [vf, vl)
    int lead, vf, vl;
    bool live, busy;   // the lane's column, or any of the wave's, is a query head's
    int first, last, wf, wl;   // the column's rows; all columns of the wave have [wf, wl)
    int ids, ids_at;
    unsigned in;   // WIN: which rows of its half tile any column attends
    unsigned kr[KN][KW], vr[VN][VW];
    unsigned ko[KN], vo[VN];   // this thread's pieces of a tile, bytes from the row that its half of the tile starts at
    float sr, minus;   // minus: -1, which the compiler does not see, so that a lo is one instruction
    std::conditional_t<HALF, half8, float4v> qf[KS][HALF ? 2 : 1];
    float cs, m_run, l_run, v_run, v_end;
    int ev;
    float16v o[DT];

    __device__ __forceinline__ ShWork(const PgView &p_, const ShArgs &a_, ShLds<KT, CL, WIN> &l, int kvh_)
        : p(p_), a(a_), lds(l), lane(threadIdx.x & 63), h(lane >> 5),
          wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))), kvh(kvh_), hd(p_.hd), group(a_.nh / p_.n_kv), bad(0), sr(0.0f), minus(-1.0f) {
        asm("" : "+v"(minus));
        // past the head's dims its first ones, which meet zeros (K) or come to nothing (V)
#pragma unroll
        for (int j = 0; j < KN; j++) {
            const int u = j * NTH + (int)threadIdx.x, row = u / KC, d = u % KC * KD;
            ko[j] = ((row & 15) * hd + (d < hd ? d : 0)) * EB;
        }
#pragma unroll
        for (int j = 0; j < VN; j++) {
            const int u = j * NTH + (int)threadIdx.x, row = vrow(u), d = u % VC * 4;
            vo[j] = ((row & 15) * hd + (d < hd ? d : 0)) * EB;
        }
    }
    // the first row of a V piece, one of VC beside each other
    static __device__ __forceinline__ int vrow(int u) { return HALF ? u / VC * 4 : u / VC; }

    // this lane's column: head `head` of all, or none
    __device__ __forceinline__ void column(int s0, int s1, int rows, int ct, size_t &head) {
        const int c = ct * CT + wave * 32 + (lane & 31), s = s0 + c / group;
        live = s < s1;
        busy = __any(live);
        head = live ? (size_t)s * a.nh + kvh * group + c % group : (size_t)s0 * a.nh + kvh * group;
        const int len = live ? kr_page_len(a.len[s], a.max_len, bad) : 0;
        last = min(len, rows);
        first = a.window > 0 && len > a.window ? min(len - a.window, rows) : 0;
        const bool some = live && first < last;
        // the columns' least first row and largest end; WIN: below it, of those that begin or end there, the most rows
        using Key = std::conditional_t<WIN, unsigned long long, int>;
        constexpr int SH = WIN ? 32 : 0;
        Key f = (Key)(some ? first : INT_MAX) << SH, l = (Key)(some ? last : 0) << SH;
        if constexpr (WIN) {
            f |= INT_MAX - (some ? last : 0);
            l |= INT_MAX - (some ? first : INT_MAX);
        }
        wf = live ? first : 0;
        wl = live ? last : INT_MAX;
        for (int o = 16; o >= 1; o >>= 1) {
            f = min(f, __shfl_xor(f, o));
            l = max(l, __shfl_xor(l, o));
            wf = max(wf, __shfl_xor(wf, o));
            wl = min(wl, __shfl_xor(wl, o));
        }
        wf = __builtin_amdgcn_readfirstlane(wf);
        wl = __builtin_amdgcn_readfirstlane(wl);
        __syncthreads();   // the piece before has been read
        if (threadIdx.x == 0) lds.range[0] = (Key)INT_MAX << SH, lds.range[1] = 0;
        __syncthreads();
        if (lane == 0) {
            atomicMin(&lds.range[0], f);
            atomicMax(&lds.range[1], l);
        }
        if (WIN && h == 0) lds.col[wave * 32 + lane] = some ? make_int2(first, last) : make_int2(INT_MAX, 0);
        __syncthreads();
        vf = __builtin_amdgcn_readfirstlane((int)(lds.range[0] >> SH));
        vl = __builtin_amdgcn_readfirstlane((int)(lds.range[1] >> SH));
    }

    // The pages of the 64 half tiles from r0 on. Windows may leave rows within [vf, vl) to no column, between sequences
    // far apart: those may hold anything, and pages of such rows alone need not be in the table.
    __device__ __forceinline__ void find(int r0) {
        ids_at = r0;
        const int r = r0 + 16 * lane;
        if constexpr (WIN) {
            const auto rows = [&](int f, int l) {   // of the half tile, those of [f, l)
                const int b = max(f - r, 0), e = min(l - r, 16);
                return b < e ? (1u << e) - (1u << b) : 0u;
            };
            in = rows(vf, vl);
            // a column has all rows from vf to f, and another all from l to vl
            const int f = INT_MAX - __builtin_amdgcn_readfirstlane((int)(unsigned)lds.range[0]);
            const int l = INT_MAX - __builtin_amdgcn_readfirstlane((int)(unsigned)lds.range[1]);
            if (f < l && r0 < l && r0 + 64 * 16 > f) {
                in = 0;
#pragma unroll 1
                for (int c = 0; c < CT; c++) in |= rows(lds.col[c].x, lds.col[c].y);
            }
            ids = in ? pg_page(p, lead, r, bad) : -1;
        } else {
            ids = r + 16 > vf && r < vl ? pg_page(p, lead, r, bad) : -1;
        }
    }

    // asks for the rows of the tile at r0
    __device__ __forceinline__ void fetch(int r0) {
        if (r0 - ids_at >= 64 * 16) find(r0);
        const int i = (r0 - ids_at) >> 4;
        const int a0 = __builtin_amdgcn_readlane(ids, i), a1 = __builtin_amdgcn_readlane(ids, i + 1);
        const size_t lo = kr_page_row(max(a0 >= 0 ? a0 : a1, 0), p.n_kv, kvh, p.shift, r0);
        const size_t hi = kr_page_row(max(a1 >= 0 ? a1 : a0, 0), p.n_kv, kvh, p.shift, r0 + 16);
        const char *const k0 = (const char *)p.k + lo * hd * EB, *const k1 = (const char *)p.k + hi * hd * EB;
        const char *const v0 = (const char *)p.v + lo * hd * EB, *const v1 = (const char *)p.v + hi * hd * EB;
        const int first_u = wave * 64;   // of the wave, whose pieces lie in one half of the tile
#pragma unroll
        for (int j = 0; j < KN; j++) {
            const int row = (j * NTH + first_u) / KC;
            if (SH_R * KC % NTH == 0 || row < SH_R) pa_load(kr[j], (row < 16 ? k0 : k1) + ko[j]);
        }
#pragma unroll
        for (int j = 0; j < VN; j++) {
            if (VU % NTH != 0 && j * NTH + first_u >= VU) continue;
            const char *const at = (vrow(j * NTH + first_u) < 16 ? v0 : v1) + vo[j];
            if constexpr (HALF) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    unsigned x[VW / 4];
                    pa_load(x, at + r * hd * EB);
#pragma unroll
                    for (int w = 0; w < VW / 4; w++) vr[j][r * (VW / 4) + w] = x[w];
                }
            } else {
                pa_load(vr[j], at);
            }
        }
        if constexpr (KT == PG_Q8) {
            const int row = lane & 31;
            if (wave == 0) sr = (lane < 32 ? p.kd : p.vd)[row < 16 ? lo + row : hi + (row - 16)];
        }
    }

    // and lays them down; rows that no column attends may hold anything, so of V (or its scales) they are zeros
    __device__ __forceinline__ void put(int buf, int r0) {
        [[maybe_unused]] unsigned some = 0;   // which of its rows a column attends
        if constexpr (WIN) {
            const int at = (r0 - ids_at) >> 4;
            some = __builtin_amdgcn_readlane(in, at) | __builtin_amdgcn_readlane(in, at + 1) << 16;
        }
        const bool whole = WIN ? some == ~0u : r0 >= vf && r0 + SH_R <= vl;
        auto has = [&](int row) { return WIN ? (some >> row & 1) != 0 : r0 + row >= vf && r0 + row < vl; };
#pragma unroll
        for (int j = 0; j < KN; j++) {
            const int u = j * NTH + (int)threadIdx.x, row = u / KC, c = u % KC;
            if (SH_R * KC % NTH != 0 && row >= SH_R) continue;
            uint4v w;
            if constexpr (KT == PG_Q8) {
                const unsigned x = kr[j][0] ^ 0x80808080u, y = kr[j][1] ^ 0x80808080u;
                w = uint4v{ pa_h2(x, 0x04010400), pa_h2(x, 0x04030402), pa_h2(y, 0x04010400), pa_h2(y, 0x04030402) };
            } else {
                w = uint4v{ kr[j][0], kr[j][1], kr[j][2], kr[j][3] };
            }
            *(uint4v *)(lds.k[buf] + sh_at<KC>(row, c)) = w;
        }
#pragma unroll
        for (int j = 0; j < VN; j++) {
            const int u = j * NTH + (int)threadIdx.x;
            if (VU % NTH != 0 && u >= VU) continue;
            if (!whole && KT != PG_Q8) {
                [[maybe_unused]] const unsigned mine = some >> vrow(u);   // (each row's own shift would be kept in a register)
#pragma unroll
                for (int w = 0; w < VW; w++) {
                    const int i = HALF ? w / (VW / 4) : 0;
                    vr[j][w] = (WIN ? (mine >> i & 1) != 0 : has(vrow(u) + i)) ? vr[j][w] : 0u;
                }
            }
            if constexpr (HALF) {
                const int quad = u / VC, d = u % VC * 4;
                const int chunk = (quad >> 2) * 2 + (quad & 1), half = (quad >> 1) & 1;
                uint2v t[4];
                if constexpr (KT == PG_F16) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const unsigned sel = c & 1 ? 0x07060302u : 0x05040100u;
                        t[c] = uint2v{ __builtin_amdgcn_perm(vr[j][2 + c / 2], vr[j][c / 2], sel),
                                       __builtin_amdgcn_perm(vr[j][6 + c / 2], vr[j][4 + c / 2], sel) };
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const unsigned x = vr[j][2 * i] ^ 0x80808080u, y = vr[j][2 * i + 1] ^ 0x80808080u;
                        const unsigned lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
                        t[0][i] = pa_h2(lo, 0x04010400);
                        t[1][i] = pa_h2(lo, 0x04030402);
                        t[2][i] = pa_h2(hi, 0x04010400);
                        t[3][i] = pa_h2(hi, 0x04030402);
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) *(uint2v *)(lds.v[buf] + sh_vt(d + c, chunk) + 8 * half) = t[c];
            } else {
                const int row = u / KC, c = u % KC;
                // rows 4 apart, which the two halves of a wave read together, in different banks
                *(uint4v *)(lds.v[buf] + (row * KC + (c ^ ((row >> 2 & 1) << 3))) * 16) =
                    uint4v{ vr[j][0], vr[j][1], vr[j][2], vr[j][3] };
            }
        }
        if constexpr (KT == PG_Q8) {
            // 8-bit rows are numbers whatever they hold; their scales may be none
            if (wave == 0) (lane < 32 ? lds.kd : lds.vd)[buf][lane & 31] = whole || has(lane & 31) ? sr : 0.0f;
        }
    }

    __device__ __forceinline__ void queries(size_t head) {
        const float *q = a.q + head * hd;
        // the scores' factor is positive, so that the largest product is the largest score: its sign is the queries', and
        // of 0 so are the zeros
        const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : a.scale;
        int e = 0;
        if constexpr (HALF) {
            float x[KS][8], m = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = j * 16 + h * 8;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4v t = live && d < hd ? *(const float4v *)(q + d + i) : float4v{ 0, 0, 0, 0 };
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        x[j][i + c] = t[c] * sign;
                        m = fmaxf(m, fabsf(t[c]));
                    }
                }
            }
            m = fmaxf(m, sh_other(m));
            e = pa_power(m, a.scale);
#pragma unroll
            for (int j = 0; j < KS; j++) {
                half8 hi, lo;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = ldexpf(x[j][i], e);
                    hi[i] = (_Float16)y;
                    lo[i] = (_Float16)(y - (float)hi[i]);
                }
                qf[j][0] = hi;
                qf[j][1] = lo;
            }
        } else {
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = j * 8 + h * 4;
                qf[j][0] = live && d < hd ? *(const float4v *)(q + d) * sign : float4v{ 0, 0, 0, 0 };
            }
        }
        const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
        cs = ldexpf(a.cap > 0.0f ? scale : scale * 1.4426950408889634f, -e);
    }

    // the tile at row r0, in LDS. Waves at their scores' products go first, those that lay down rows last: the
    // scores are what a wave waits for longest (16 sequences behind 16,000 rows 37.5 -> 36.1 us, 8 bits of 64 dims 31.7 -> 30.1)
    __device__ __forceinline__ void tile(int buf, int r0) {
        __builtin_amdgcn_s_setprio(2);
        float16v s = {};
        // a float cache's products in two sums where registers hold them: at 128 dims 5.1e-7 of error against 64 bits
        // instead of 8.1e-7, and 1% of the time
        constexpr bool TWO = !HALF && CL < 256;
        [[maybe_unused]] float16v more = {};
        // eight operands are asked for at once: one by one their way from LDS would be most of a tile's time
        constexpr int G = 8;
#pragma unroll
        for (int j0 = 0; j0 < KS; j0 += G) {
            uint4v w[G];
#pragma unroll
            for (int j = 0; j < G && j0 + j < KS; j++) w[j] = *(const uint4v *)(lds.k[buf] + sh_at<KC>(lane & 31, 2 * (j0 + j) + h));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < G && j0 + j < KS; j++) {
                if constexpr (HALF) {
#pragma unroll
                    for (int x = 0; x < 2; x++)
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, w[j]), qf[j0 + j][x], s, 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float16v &sum = TWO && c & 1 ? more : s;
                        sum = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w[j][c]), qf[j0 + j][0][c], sum, 0, 0, 0);
                    }
                }
            }
        }
        if constexpr (TWO) s += more;
        __builtin_amdgcn_s_setprio(1);
        // V's first operands, on their way meanwhile
        constexpr int VG = HALF ? (DT < 4 ? DT : 4) : 0;
        half8 vf8[HALF ? VG : 1][2];
        auto v_read = [&](int t, int c) { return *(const half8 *)(lds.v[buf] + sh_vt(32 * t + (lane & 31), 2 * c + h)); };
        if constexpr (HALF) {
#pragma unroll
            for (int t = 0; t < VG; t++)
#pragma unroll
                for (int c = 0; c < 2; c++) vf8[t][c] = v_read(t, c);
            __builtin_amdgcn_sched_barrier(0);
        }
        // value i is row (i & 3) + 8 (i >> 2) + 4 h
        float ce = cs;   // a score's power of two is s ce, ce > 0: what is cut off stays -inf
        if constexpr (KT == PG_Q8) {
            // both factors first: either one alone may take the products out of the floats
            ce = 1.0f;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4v d = *(const float4v *)(lds.kd[buf] + 2 * i + 4 * h);
#pragma unroll
                for (int c = 0; c < 4; c++) s[i + c] *= cs * d[c];
            }
        }
        if (a.cap > 0.0f) {
            // one after the other: the product of both factors may lie below the normal floats
            const float inv_cap = 1.0f / a.cap;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = pa_tanh(s[i] * ce * inv_cap);
            ce = a.cap * 1.4426950408889634f;
        }
        if (r0 < wf || r0 + SH_R > wl) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int r = r0 + (i & 3) + 8 * (i >> 2) + 4 * h;
                s[i] = r >= first && r < last ? s[i] : -INFINITY;
            }
        }
        float m_tile = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) m_tile = fmaxf(m_tile, s[i]);
        m_tile *= ce;
        // what the weights are taken from moves where a score passes it by more than SLACK (and at the first)
        const bool moved = __any(m_tile > m_run + SLACK);
        float f = 1.0f;
        if (moved) {
            const float m_new = fmaxf(m_run, fmaxf(m_tile, sh_other(m_tile)));
            f = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= f;
        }
        // weights of no finite maximum: 0 for -inf, NaN for NaN
        const float base = UP - (m_run == -INFINITY ? 0.0f : m_run);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], ce, base));
            l_run += s[i];
        }
        if constexpr (KT == PG_Q8) {
            float v_tile = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4v d = *(const float4v *)(lds.vd[buf] + 2 * i + 4 * h);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    // a rounded product: hi and lo are of the same value
                    float x = s[i + c] * d[c];
                    asm("" : "+v"(x));
                    s[i + c] = x;
                    v_tile = fmaxf(v_tile, fabsf(x));
                }
            }
            // what the weights times their scales are over, as kr_paged_wave.h has it
            if (moved || __any(v_tile >= v_end)) {
                v_run = fmaxf(v_run * f, fmaxf(v_tile, sh_other(v_tile)));
                const int e = max(PA_EV, (int)(__float_as_uint(v_run) >> 23) - 126);
                f = ldexpf(f, ev - e);
                ev = e;
                v_end = ldexpf(1.0f, e);
#pragma unroll
                for (int t = 0; t < DT; t++) o[t] *= f;
            }
            const float up = ldexpf(1.0f, PA_UP - ev);
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] *= up;
        } else if (moved) {
#pragma unroll
            for (int t = 0; t < DT; t++) o[t] *= f;
        }
        if constexpr (HALF) {
            half8 w[2][2];   // [16 rows][hi, lo]
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                // as a pair that the compiler does not take apart again, so that it converts once
                unsigned pair = __builtin_bit_cast(unsigned, half2v{ (_Float16)s[i], (_Float16)s[i + 1] });
                asm("" : "+v"(pair));
                const half2v hi = __builtin_bit_cast(half2v, pair);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    w[i >> 3][0][(i & 7) + c] = hi[c];
                    w[i >> 3][1][(i & 7) + c] = (_Float16)__builtin_fmaf((float)hi[c], minus, s[i + c]);
                }
            }
#pragma unroll
            for (int t0 = 0; t0 < DT; t0 += VG) {
#pragma unroll
                for (int t = 0; t < VG; t++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
#pragma unroll
                        for (int x = 0; x < 2; x++)
                            o[t0 + t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf8[t][c], w[c][x], o[t0 + t], 0, 0, 0);
                        if (t0 + VG < DT) vf8[t][c] = v_read(t0 + VG + t, c);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int t = 0; t < DT; t++) {
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int row = (i & 3) + 8 * (i >> 2) + 4 * h, dim = 32 * t + (lane & 31);
                    v[i] = *(const float *)(lds.v[buf] + (row * KC + ((dim >> 2) ^ ((row >> 2 & 1) << 3))) * 16 + (dim & 3) * 4);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[i], s[i], o[t], 0, 0, 0);
            }
        }
    }

    // row tiles at rows [r0, r1) of a group's column tile ct, and the part's sums
    __device__ __forceinline__ void part(int s0, int s1, int rows, int ct, int r0, int r1, size_t slot) {
        size_t head;
        column(s0, s1, rows, ct, head);
        lead = s0;
        m_run = -INFINITY;
        l_run = 0.0f;
        ev = PA_EV;
        v_run = v_end = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) o[t] = float16v{};
        // tiles that no column here attends are passed over
        r0 = max(r0, vf & -SH_R);
        r1 = min(r1, vl);
        if (r0 < r1) {
            find(r0);
            fetch(r0);
            queries(head);
            put(0, r0);
            __syncthreads();
            for (int buf = 0; r0 < r1; r0 += SH_R, buf ^= 1) {
                const bool more = r0 + SH_R < r1;
                if (more) fetch(r0 + SH_R);
                if (busy) {
                    tile(buf, r0);
                    __builtin_amdgcn_s_setprio(0);
                }
                if (more) put(buf ^ 1, r0 + SH_R);
                __syncthreads();
            }
        }
        const float l = ldexpf(l_run + sh_other(l_run), -UP), f = ldexpf(1.0f, KT == PG_Q8 ? ev - PA_UP : -UP);
        if (!live) return;
        const size_t at = slot * CT + wave * 32 + (lane & 31);
        if (h == 0) *(float2v *)(a.spml + at * 2) = float2v{ m_run, l };
        float *out = a.spart + at * hd;
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * t + 2 * i + 4 * h;
                if (d < hd) *(float4v *)(out + d) = float4v{ o[t][i] * f, o[t][i + 1] * f, o[t][i + 2] * f, o[t][i + 3] * f };
            }
    }
};

// The first workgroups' waves have shares of the sequences' own rows, the others shares of the
// shared ones: the former wait for HBM, the latter for the matrix cores (and
// for power: 64 sequences behind 32,000 rows run at 1.6 to 2.0 GHz), so they are one launch.
template <int KT, int CL, bool WIN>
__global__ void __launch_bounds__(64 * SH_WC, sh_waves(KT, CL)) k_shared_rows(const PgView p, const ShArgs a) {
    __shared__ ShLds<KT, CL, WIN> lds;
    // KV heads in turn, so that a die has few of them (of eight one), whose rows its L2 holds for all columns
    const int kvh = (int)blockIdx.x % p.n_kv, block = (int)blockIdx.x / p.n_kv;
    int bad = 0;
    const ShTiles all = sh_tiles(p, a, bad);
    if (block < all.own) {
        const int u = block * SH_WC + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        PaWave<KT, CL, false, ShArgs, true> w(p, a, kvh);
        w.bad = bad;
        PaAll pa = pa_all(p, a, w.bad, SH_WC * all.own);
        if (u < pa.shares) {
            int left = pa_bound(pa, u + 1) - pa_bound(pa, u), t = pa_bound(pa, u);
            for (w.seq = pa_find(p, a, pa, t, w.bad); left > 0; w.seq++, t = 0) {
                w.sp = pa_of(p, a, pa, w.seq, w.bad);
                const int end = min(w.sp.tiles, t + left);
                w.part(t, end, (size_t)kvh * (p.n_seq + a.shares) + w.seq + u);
                left -= end - t;
            }
        }
        kr_report(a.fault, w.bad);
        return;
    }
    const int u = block - all.own, tiles = all.tiles, shares = sh_shares(a, all);
    ShWork<KT, CL, WIN> w(p, a, lds, kvh);
    w.bad = bad;
    if (u < shares && tiles > 0) {
        // what the later pieces are found by lies in LDS, as registers are short in between
        const int lane = (int)(threadIdx.x & 63);
        if (threadIdx.x < 64) {
            lds.group[lane] = make_int4(all.g.s0, all.g.s1, all.g.rows, all.begin);
            lds.sums[lane] = make_int2(all.sum, all.csum);
        }
        const auto at = [](int v, int g) { return __builtin_amdgcn_readlane(v, g); };
        const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        const int end = (int)((long long)tiles * (u + 1) / shares);
        int t = (int)((long long)tiles * u / shares), g = __popcll(__ballot(all.sum <= t));
        int s0 = at(all.g.s0, g), s1 = at(all.g.s1, g), rows = at(all.g.rows, g), begin = at(all.begin, g);
        int sum = at(all.sum, g), csum = at(all.csum, g);
        for (;;) {
            const int rts = sh_rts(rows, begin), cts = sh_cts(s1 - s0, w.group);
            const int i = t - (sum - rts * cts), ct = i / rts, r = i % rts, n = min(rts - r, end - t);
            w.part(s0, s1, rows, ct, begin + r * SH_R, min(rows, begin + (r + n) * SH_R),
                   (size_t)kvh * a.slots + csum - cts + ct + u);
            if ((t += n) >= end) break;
            g = __popcll(__ballot(lds.sums[lane].x <= t));
            const int4 of = lds.group[g];
            const int2 sums = lds.sums[g];
            s0 = one(of.x), s1 = one(of.y), rows = one(of.z), begin = one(of.w), sum = one(sums.x), csum = one(sums.y);
        }
    }
    kr_report(a.fault, w.bad);
}

// A head of a sequence a workgroup: its own rows' parts, then the shared ones'
// (2^dl lanes hold its dims four at a time, the workgroup's other factor the parts
// side by side). By latency, so the parts are asked for before their weights are known: 512
// heads of 17 parts of 128 dims 5.8 us (7.5 one after the other).
constexpr int SJ_N = 4;   // parts a thread asks for at once
template <int T> __global__ void __launch_bounds__(T) k_shared_join(const PgView p, const ShArgs a, int dl) {
    __shared__ float4v s_o[T];
    const int s = blockIdx.y, x = blockIdx.x, tid = threadIdx.x, group = a.nh / p.n_kv, kvh = x / group, col = x % group;
    int bad = 0;   // reported by the other launches
    PaSpan sp;
    const ShTiles all = sh_tiles(p, a, bad);
    const PaParts r = pa_parts(p, a, s, kvh, sp, SH_WC * all.own);
    const float *ml0 = a.pml + (r.slot * group + col) * 2, *part0 = a.part + (r.slot * group + col) * p.hd;
    const float *ml1 = nullptr, *part1 = nullptr;
    int n1 = 0;
    const unsigned long long in = __ballot(all.g.rows > 0 && s >= all.g.s0 && s < all.g.s1);
    if (in) {
        const int g = __builtin_ctzll(in), rts = __builtin_amdgcn_readlane(all.rts, g), cts = __builtin_amdgcn_readlane(all.cts, g);
        const int c = (s - __builtin_amdgcn_readlane(all.g.s0, g)) * group + col, ct = c / SH_CT;
        if (rts > 0) {
            const int tiles = all.tiles, shares = sh_shares(a, all);
            const int t0 = __builtin_amdgcn_readlane(all.sum, g) - rts * cts + ct * rts;
            const auto share = [&](int t) { return (int)((((long long)t + 1) * shares - 1) / tiles); };
            const int u0 = share(t0);
            n1 = share(t0 + rts - 1) - u0 + 1;
            const size_t slot = (size_t)kvh * a.slots + __builtin_amdgcn_readlane(all.csum, g) - cts + ct + u0;
            ml1 = a.spml + (slot * SH_CT + c % SH_CT) * 2;
            part1 = a.spart + (slot * SH_CT + c % SH_CT) * p.hd;
        }
    }
    const int n = r.n + n1;
    const auto get = [&](int i) {
        return *(const float2v *)(i < r.n ? ml0 + (size_t)i * group * 2 : ml1 + (size_t)(i - r.n) * SH_CT * 2);
    };
    const auto at = [&](int i) { return i < r.n ? part0 + (size_t)i * group * p.hd : part1 + (size_t)(i - r.n) * SH_CT * p.hd; };
    // the first parts are on their way while the weights are found
    const int lane = tid & 63, first = tid >> dl, lanes = T >> dl, q = tid & ((1 << dl) - 1), d = 4 * q < p.hd ? 4 * q : 0;
    float4v v[SJ_N];
    const auto fetch = [&](int i) {
#pragma unroll
        for (int k = 0; k < SJ_N; k++) v[k] = *(const float4v *)(at(min(i + k * lanes, n - 1)) + d);
    };
    const float2v mine = lane < n ? get(lane) : float2v{ -INFINITY, 0.0f };
    fetch(first);
    float m = mine.x;
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, get(i).x);
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const auto weight = [&](float v) { return v == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v - m); };
    const float w = weight(mine.x);
    float l = mine.y * w;
    for (int i = lane + 64; i < n; i += 64) {
        const float2v v = get(i);
        l += v.y * weight(v.x);
    }
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
    const float inv = 1.0f / l;
    float4v acc = { 0, 0, 0, 0 };
    for (int i0 = 0; i0 < n; i0 += SJ_N * lanes) {
        if (i0 > 0) fetch(i0 + first);
#pragma unroll
        for (int k = 0; k < SJ_N; k++) {
            const int i = i0 + first + k * lanes;
            const float x = __shfl(w, i & 63);
            if (i < n) acc += v[k] * (i < 64 ? x : weight(get(i).x));
        }
    }
    s_o[tid] = acc;
    for (int k = lanes >> 1; k >= 1; k >>= 1) {
        __syncthreads();
        if (first < k) s_o[tid] = acc = acc + s_o[tid + (k << dl)];
    }
    // (zeros for no rows: the shared ones' parts hold what their NaNs times 0 are)
    if (first == 0 && 4 * q < p.hd) *(float4v *)(a.o + ((size_t)s * a.nh + x) * p.hd + d) = sp.len == 0 ? float4v{} : acc * inv;
}

// ---- the host's side ----

constexpr int SH_CUS = 256;

struct ShSizes {
    int wgs, own, sfew, slots;
    size_t part, pml, spart, spml;   // floats
};
ShSizes sh_sizes(const krh_pages *kv, int n_seq, int nh, int n_groups, int max_shared) {
    ShSizes r;
    const int group = nh / kv->n_kv_heads;
    const long long cts = (long long)n_seq * group / SH_CT + n_groups, tiles = cts * ((max_shared + SH_R - 1) / SH_R);
    // as many workgroups as the chip holds at once
    const int most = SH_CUS * sh_waves(kv->kv_type, kv->head_dim) / kv->n_kv_heads;
    r.wgs = most < 2 ? 2 : most;
    r.own = r.wgs / 4 > 0 ? r.wgs / 4 : 1;
    const int shared = (int)(r.wgs - r.own < tiles ? r.wgs - r.own : tiles);
    // Where a compute unit holds two, one each while there are few tiles (8B shape, halves, in us, 128 / 256 / 384
    // workgroups for the shared rows: 16 sequences behind 2048 20.9 / 23.7 / -, 64 33.0 / 37.8 / 38.7, behind 4096 42.0 / - / 40.6)
    r.sfew = sh_waves(kv->kv_type, kv->head_dim) > 1 && r.own < shared ? r.own : shared;
    r.slots = (int)(cts + shared);
    const size_t own = (size_t)kv->n_kv_heads * (n_seq + SH_WC * r.wgs) * group;
    const size_t both = (size_t)kv->n_kv_heads * r.slots * SH_CT;
    r.part = own * kv->head_dim;
    r.pml = (own * 2 + 3) & ~(size_t)3;
    r.spart = both * kv->head_dim;
    r.spml = both * 2;
    return r;
}

// Tiles that a share is worth: two, whose parts are fewer to join (8B shape, halves, 16
// sequences behind 1024 rows in us, of 1 / 2 / 4: 20.8 / 18.4 / 19.7, 64 31.8 / 30.9 / 27.8); one of those
// that take long (floats of 256 dims, 32 behind 1024 rows 50.7 / 60 / 83.5, of 128 30.7 / 29.4 / 37.7;
// halves of 256 dims 27.3 / 27.9 / 35.7).
int sh_least(const krh_pages *kv) { return kv->kv_type == ML_F32 || kv->head_dim > 128 ? 1 : 2; }

// Column tiles of groups of as many sequences each
double sh_cols(const krh_pages *kv, int n_seq, int nh, int n_groups) {
    return n_groups * ceil(ceil((double)n_seq / n_groups) * (nh / kv->n_kv_heads) / SH_CT);
}

// What a wave does on SH_R own rows, in the work of a workgroup, a wave, on a tile of the shared ones: by it the device
// has as many workgroups for the own rows as their part of all work is. 0: they have a quarter, which needs no look at all
// lengths (0.5 to 0.9 us: 16 sequences of up to 1001 rows behind 2048 of the 8B shape 20.4 us instead of 19.6): where they
// are at most, by max_len, three fifths of the work, or two fifths of kernels that have one workgroup a compute unit, whose
// quarter is few waves. Measured, a quarter / by the work / each sequence by itself, 64 sequences of 4000 to 8000 own rows
// behind 1024: 8B shape, halves 349 / 287 / 282 us, floats 1150 / 535 / 547; 1B shape, 8 bits 178 / 95 / 96; floats of 256
// dims 1150 / 544 / 526, 8 bits 471 / 175 / 160. Behind 4096: 364 / 289 / 357, 1133 / 525 / 703, 184 / 102 / 120, 1145 / 560 /
// 714, 467 / 193 / 227.
float sh_weigh(const krh_pages *kv, int n_seq, int nh, int max_len, int n_groups, int max_shared, int window) {
    static const float weigh[3][3] = { { .12f, .19f, .06f }, { .11f, .12f, .08f }, { .12f, .15f, .06f } };   // F32, F16, Q8
    const float w = weigh[kv->kv_type == ML_F32 ? 0 : kv->kv_type == ML_F16 ? 1 : 2][kv->head_dim <= 64 ? 0 : kv->head_dim <= 128 ? 1 : 2];
    const double most = max_len - max_shared, own = n_seq * (window > 0 && window < most ? window : most);
    const double shared = sh_cols(kv, n_seq, nh, n_groups) * (window > 0 && window < max_shared ? window : max_shared);
    return w * own > (sh_waves(kv->kv_type, kv->head_dim) > 1 ? 1.5 : 0.7) * shared ? w : 0.0f;
}

// Whether the shared rows are better passed over once, by estimated times in us. Each
// sequence by itself (krh_paged_attention): 11.5, a group's shared rows at the rate of HBM, and at the rate at which dies
// read what others read too for its other sequences (TB/s: halves 4 and 10.5, floats 6.6, 8 bits 5). Once for
// all: 15, 2.5 for 1024 heads of 128 dims to join (by dims squared), a workgroup's tiles, `tile` each, and with a window
// 2.5 a group, whose first rows are looked for one after another. As many groups as do not leave a sequence alone; own
// rows are as long either way. Measured, each / once, 64 sequences of 75 to 150 own rows in 1 / 8 / 16 / 32 / 63 groups:
// 8B shape, halves, behind 1024 rows 39 / 24, 53 / 29, 54 / 35, 54 / 55, 65 / 87, behind 4096 90 / 36, 161 / 51, 160 / 81,
// 197 / 140, 196 / 243, floats behind 1024 76 / 40, 95 / 68, 95 / 122, 107 / 227, 117 / 238; 1B shape, 8 bits, behind 2048 36 / 24,
// 37 / 29, 37 / 41, 38 / 71, 39 / 77; floats of 256 dims behind 2048 124 / 79, 162 / 233, 166 / 422, 168 / 798, 197 / 428. Of 4242
// sizes (2 to 128 sequences, 1 to 64 groups of 128 to 8192 rows, 30 to 8000 own rows, windows) 4% take the slower way by more
// than 5%, 1% by more than 15, the worst by 48.
bool sh_pays(const krh_pages *kv, int n_seq, int nh, int n_groups, int max_shared, int window) {
    static const double first[3] = { 6.6e6, 4e6, 5e6 }, again[3] = { 6.6e6, 10.5e6, 5e6 };   // bytes a us: F32, F16, Q8
    static const double tile[3][3] = { { 2.5, 3.8, 25 }, { 1.1, 1.85, 6 }, { 1.45, 2.7, 10 } };
    if (n_seq <= n_groups) return false;
    const int t = kv->kv_type == ML_F32 ? 0 : kv->kv_type == ML_F16 ? 1 : 2, c = kv->head_dim <= 64 ? 0 : kv->head_dim <= 128 ? 1 : 2;
    const int groups = n_groups < n_seq - n_groups ? n_groups : n_seq - n_groups, seqs = n_seq - (n_groups - groups);
    const double rows = window > 0 && window < max_shared ? window : max_shared;
    const double row = (double)kv->n_kv_heads * kv->head_dim * (t == 0 ? 8 : t == 1 ? 4 : 2) + (t == 2 ? 8 * kv->n_kv_heads : 0);
    const double tiles = ceil(sh_cols(kv, seqs, nh, groups) * ceil(rows / SH_R) * kv->n_kv_heads /
                              (SH_CUS * sh_waves(kv->kv_type, kv->head_dim) * 3 / 4));
    const double heads = (double)n_seq * nh / 1024, dims = kv->head_dim / 128.0;
    return 11.5 + rows * row * (groups / first[t] + (seqs - groups) / again[t]) >
           15 + 2.5 * heads * dims * dims + tiles * tile[t][c] + (window > 0 ? 2.5 * n_groups : 0);
}
bool sh_shared(const krh_pages *kv, int n_seq, int nh, int n_groups, int max_shared, int window) {
    return n_groups > 0 && max_shared > 0 && sh_pays(kv, n_seq, nh, n_groups, max_shared, window);
}

bool sh_args_ok(const krh_pages *kv, int n_seq, int n_heads, int max_len, int n_groups, int max_shared) {
    return pg_pages_ok(kv) && n_seq > 0 && n_seq <= KRH_ROWS_MAX && max_len > 0 && max_len <= KR_PAGE_LEN_MAX &&
           n_heads > 0 && n_heads % kv->n_kv_heads == 0 && n_heads / kv->n_kv_heads <= KR_PAGE_GROUP_MAX &&
           (long long)n_seq * (max_len / 16 + 1) <= INT32_MAX / 2 && n_groups >= 0 && n_groups <= PA_GROUPS &&
           max_shared >= 0 && max_shared <= max_len &&
           // tiles of all column tiles
           ((long long)n_seq * (n_heads / kv->n_kv_heads) / 32 + n_groups) * (max_shared / SH_R + 1) <= INT32_MAX / 2;
}

using ShRows = void (*)(const PgView, const ShArgs);
template <int KT, bool WIN> ShRows sh_rows(int hd) {
    return hd <= 64 ? k_shared_rows<KT, 64, WIN> : hd <= 128 ? k_shared_rows<KT, 128, WIN> : k_shared_rows<KT, 256, WIN>;
}
template <int KT> ShRows sh_rows(int hd, bool win) { return win ? sh_rows<KT, true>(hd) : sh_rows<KT, false>(hd); }

}  // namespace

extern "C" int krh_paged_attention_shared_form(const krh_pages *kv, int n_seq, int n_heads, int max_len, int n_groups,
                                               int max_shared, int window) {
    if (!sh_args_ok(kv, n_seq, n_heads, max_len, n_groups, max_shared) || window < 0) return -1;
    return sh_shared(kv, n_seq, n_heads, n_groups, max_shared, window);
}

extern "C" size_t krh_paged_attention_shared_ws(const krh_pages *kv, int n_seq, int n_heads, int max_len, int n_groups,
                                                int max_shared) {
    if (!sh_args_ok(kv, n_seq, n_heads, max_len, n_groups, max_shared)) return 0;
    const size_t base = krh_paged_attention_ws(kv, n_seq, n_heads, max_len, 0);
    if (n_groups == 0 || max_shared == 0) return base;
    // for both ways, whichever pays: fewer sequences may pay where more do not, and a window where none does
    const ShSizes r = sh_sizes(kv, n_seq, n_heads, n_groups, max_shared);
    const size_t b = sizeof(float) * (r.part + r.pml + r.spart + r.spml + 4);
    return b > base ? b : base;
}

extern "C" void krh_paged_attention_shared(float *o, const krh_pages *kv, const int *table, int table_ld, const int *len,
                                           int n_seq, const int *group, const int *shared, int n_groups, int max_shared,
                                           const float *q, int n_heads, int max_len, int window, float scale,
                                           float softcap, void *ws) {
    if (n_seq == 0) return;
    if (pg_refuse(sh_args_ok(kv, n_seq, n_heads, max_len, n_groups, max_shared), "paged_attention_shared sizes") ||
        pg_refuse(o && table && table_ld > 0 && len && q && ws && pg_aligned(o) && pg_aligned(q) && pg_aligned(ws) &&
                      (n_groups == 0 || (group && shared)),
                  "paged_attention_shared: a missing or unaligned array") ||
        pg_refuse(window >= 0 && (softcap == 0.0f || (softcap >= FLT_MIN && softcap <= 0x1p126f)),
                  "paged_attention_shared: window or soft-cap"))
        return;
    if (!sh_shared(kv, n_seq, n_heads, n_groups, max_shared, window)) {
        kr_paged_attention(true, o, kv, table, table_ld, len, n_seq, q, n_heads, max_len, window, scale, softcap, nullptr, 0, ws);
        return;
    }
    if (pg_not_ready("paged_attention_shared before krh_init")) return;
    const ShSizes r = sh_sizes(kv, n_seq, n_heads, n_groups, max_shared);
    float *w = (float *)ws;
    ShArgs a = {};
    a.o = o, a.q = q, a.len = len;
    a.part = w, a.pml = w + r.part, a.spart = a.pml + r.pml, a.spml = a.spart + r.spart;
    a.nh = n_heads, a.max_len = max_len, a.window = window, a.shares = SH_WC * r.wgs, a.tl = pg_log2(pa_tile(kv->head_dim));
    a.least = 1;
    a.scale = scale, a.cap = softcap;
    a.group = group, a.shared = shared, a.n_groups = n_groups, a.max_shared = max_shared;
    a.wgs = r.wgs, a.own = r.own, a.weigh = sh_weigh(kv, n_seq, n_heads, max_len, n_groups, max_shared, window);
    a.sfew = r.sfew, a.sleast = sh_least(kv), a.slots = r.slots, a.fault = kr_fault_word();
    const PgView p = pg_view(kv, table, table_ld, n_seq);
    const int hd = kv->head_dim;
    const bool win = window > 0;
    const ShRows f = kv->kv_type == ML_F32   ? sh_rows<PG_F32>(hd, win)
                     : kv->kv_type == ML_F16 ? sh_rows<PG_F16>(hd, win)
                                             : sh_rows<PG_Q8>(hd, win);
    hipLaunchKernelGGL(f, dim3(r.wgs * kv->n_kv_heads), dim3(64 * SH_WC), 0, kr_stream(), p, a);
    kr_check_launch("paged_attention_shared");
    // Threads a head: with few heads the parts are asked for side by side, with many each wave's search for its parts
    // is what takes the time (a call of 512 heads of 128 dims by 256 / 128 / 64 20.1 / 20.5 / 21.1 us, 1024 of 64 36.2 / 35.2 /
    // 35.8, 1536 of 64 30.0 / 28.1 / 27.3, 2048 of 64 46.2 / 43.0 / 43.0)
    const long long heads = (long long)n_heads * n_seq;
    const int threads = heads <= 512 ? 256 : heads <= 1024 ? 128 : 64;
    hipLaunchKernelGGL(threads == 256 ? k_shared_join<256> : threads == 128 ? k_shared_join<128> : k_shared_join<64>,
                       dim3(n_heads, n_seq), dim3(threads), 0, kr_stream(), p, a, pg_log2(hd / 4));
    kr_check_launch("paged_attention_shared");
}
