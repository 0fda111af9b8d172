/* Checks cpg_paged_sched.h against counting one tile and key at a time: the units before each tile,
 * and that the workgroups' walks over their shares meet every unit of every item once, with the
 * owners that the merge of an item's pieces counts on. Prints the first difference and returns 1. */
#include "cpg_paged_sched.h"

#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <tuple>
#include <vector>

static uint32_t rng_state = 12345;
static int below(int n) {
    rng_state = rng_state * 1664525u + 1013904223u;
    return (int)((rng_state >> 8) % (uint32_t)n);
}

/* units of tile i, by the keys that its rows see */
static int count_units(const pg_batch &b, const pg_seq &s, int i, int *lo_unit) {
    const int tl = b.tl, window = b.window, unit = 1 << b.ul;
    int lo = -1, hi = -1;
    for (int t = i << tl; t < s.n && t < (i + 1) << tl; t++) {
        const int pos = s.p0 + t;
        if (pos < 0) continue;
        const int first = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
        if (lo < 0 || first < lo) lo = first;
        if (pos > hi) hi = pos;
    }
    if (hi < 0) { *lo_unit = 0; return 1; }
    *lo_unit = lo / unit;
    return hi / unit - lo / unit + 1;
}

static int check(const std::vector<int> &off, const std::vector<int> &len, int T, int KV, int parts, int tl,
                 int ul, int extra, int window, int plog, int max_pages, int grid) {
    const int S = (int)len.size();
    const pg_batch b = {off.data(), len.data(), S, T, KV, max_pages, plog, window, parts, tl, ul, extra};
    int64_t U = 0;
    std::vector<int64_t> before(S);
    for (int s = 0; s < S; s++) {
        const pg_seq q = pg_get_seq(b.q_off, b.len, s, T, max_pages, plog);
        if (q.lo < 0 || q.n < 0 || q.lo + q.n > T || q.len < 0) { printf("bad rows of %d\n", s); return 1; }
        int64_t sum = 0;
        for (int i = 0; i <= pg_tiles(q, tl); i++) {
            if (q.n && pg_units_before(b, q, i) != sum) {
                printf("units before tile %d of n=%d len=%d tl=%d window=%d: %lld, counted %lld\n", i, q.n,
                       q.len, tl, window, (long long)pg_units_before(b, q, i), (long long)sum);
                return 1;
            }
            if (i == pg_tiles(q, tl)) break;
            int lo;
            const int c = count_units(b, q, i, &lo);
            if (q.p0 + q.n > 0 && q.p0 + ((i + 1) << tl) > 0 && q.len > 0 && lo != pg_unit_lo(b, q, i)) {
                printf("first unit of tile %d\n", i);
                return 1;
            }
            sum += c + extra;
        }
        if (pg_seq_units(b, q) != sum * KV * parts) { printf("units of %d\n", s); return 1; }
        before[s] = U;
        U += sum * KV * parts;
    }
    /* the walks */
    std::map<std::tuple<int, int, int, int>, std::vector<int>> met;   /* item -> owner of each unit */
    std::map<std::tuple<int, int, int, int>, uint32_t> firsts;
    int64_t next = 0;
    for (int w = 0; w < grid && U; w++) {
        pg_share r;
        int block = 0;                           /* the block that takes share w */
        for (; block < grid; block++) {
            r = pg_deal((uint32_t)U, block, grid);
            if (r.w == w) break;
        }
        if (block == grid) { printf("no block for share %d of %d\n", w, grid); return 1; }
        if (r.w >= r.W) {
            if (r.u0 != r.u1) { printf("a share beyond W\n"); return 1; }
            continue;
        }
        if (r.u0 != next || r.u1 <= r.u0) { printf("share %d: %lld..%lld after %lld\n", w, (long long)r.u0, (long long)r.u1, (long long)next); return 1; }
        next = r.u1;
        int s = S - 1;
        while (before[s] > r.u0) s--;
        int64_t rem = r.u0 - before[s];
        for (uint32_t u = r.u0; u < r.u1;) {
            pg_seq q = pg_get_seq(b.q_off, b.len, s, T, max_pages, plog);
            while (rem >= pg_seq_units(b, q)) {
                q = pg_get_seq(b.q_off, b.len, ++s, T, max_pages, plog);
                rem = 0;
            }
            const pg_item it = pg_find_item(b, q, u, r.u1, (uint32_t)rem);
            rem += it.step;
            if (it.step <= 0 || it.off < 0 || it.off + it.cnt > it.all || u + it.step > r.u1) { printf("bad item\n"); return 1; }
            u += it.step;
            if (it.cnt <= 0) continue;
            auto key = std::make_tuple(s, it.kv, it.part, it.tile);
            if (!met.count(key)) firsts[key] = it.first;
            if (firsts[key] != it.first || (int)met[key].size() != it.off) { printf("pieces out of order\n"); return 1; }
            for (int i = 0; i < it.cnt; i++) met[key].push_back(w);
            if ((int)met[key].size() == it.all) {
                const int wf = pg_owner(it.first, (uint32_t)U, r.W), wl = pg_owner(it.first + it.all - 1, (uint32_t)U, r.W);
                int pieces = 1;
                for (int i = 1; i < it.all; i++) pieces += met[key][i] != met[key][i - 1];
                if (wf != met[key][0] || wl != w || wl - wf + 1 != pieces) { printf("owners %d..%d, met %d..%d\n", wf, wl, met[key][0], w); return 1; }
            }
        }
    }
    if (next != U) { printf("%lld of %lld units dealt\n", (long long)next, (long long)U); return 1; }
    for (int s = 0; s < S; s++) {
        const pg_seq q = pg_get_seq(b.q_off, b.len, s, T, max_pages, plog);
        for (int kv = 0; kv < KV; kv++)
            for (int p = 0; p < parts; p++)
                for (int i = 0; i < pg_tiles(q, tl); i++) {
                    int lo;
                    if ((int)met[std::make_tuple(s, kv, p, i)].size() != count_units(b, q, i, &lo)) {
                        printf("item (%d, %d, %d, %d) not whole\n", s, kv, p, i);
                        return 1;
                    }
                }
    }
    return 0;
}

int main() {
    const int grids[] = {1, 3, 8, 16, 64, 256, 512};
    for (int c = 0; c < 4000; c++) {
        const int S = 1 + below(c % 7 == 0 ? 40 : 5), tl = below(8), plog = below(8);
        std::vector<int> off(1, below(3) == 0 ? below(4) : 0), len;
        const int longest = c % 3 == 0 ? 2000 : 300;
        int need = 1;
        for (int s = 0; s < S; s++) {
            const int n = below(4) == 0 ? 0 : 1 + below(below(3) == 0 ? 200 : 3);
            int L = below(5) == 0 ? below(n + 1) : n + below(longest);   /* some rows without a key */
            off.push_back(off.back() + n);
            len.push_back(L);
            need = L > need ? L : need;
        }
        int T = off.back() + below(3);
        int max_pages = (need >> plog) + 1;
        if (c % 11 == 0) {                       /* data that a batch may not have */
            const int s = below(S);
            if (below(3) == 0) len[s] = -1 - below(5);
            else if (below(2)) len[s] = (max_pages << plog) + 1 + below(1 << 28);
            else off[s + 1] = below(2) ? -5 : T + 7;
        }
        const int window = below(2) ? 0 : 1 + below(below(2) ? 20 : 500);
        if (check(off, len, T, 1 + below(4), 1 + below(2), tl, tl + below(9 - tl), below(2) ? 0 : below(5), window, plog, max_pages, grids[below(7)])) {
            printf("case %d\n", c);
            return 1;
        }
    }
    /* the largest positions: a sum that leaves 32 bits, differences that do not */
    const pg_seq big = {0, 1 << 10, PG_MAX_LEN, PG_MAX_LEN - (1 << 10), false, false};
    const pg_batch b = {nullptr, nullptr, 1, 1 << 10, 1, 0, 0, 0, 1, 0, 12, 1};
    uint32_t sum = 0;
    for (int i = 0; i < 1 << 10; i++) {
        int lo;
        if (pg_units_before(b, big, i) != sum) return 1;
        sum += count_units(b, big, i, &lo) + 1;
    }
    printf("ok\n");
    return 0;
}
