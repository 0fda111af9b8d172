/* cpg_paged_sched.h — how the work of an attention call over the paged cache is divided. Integer
 * arithmetic alone, for the kernels and, compiled as plain C++, for the tests.
 *
 * Work. The rows of a sequence are taken in tiles of TB = 2^tl tokens (times the query heads of one
 * kv head), and a tile's visible keys in units of UNIT. An item is one tile of one kv head (and of
 * one part of its query heads, where they are more than a tile's rows). The units of all items,
 * U of them in the order (sequence, kv head and part, tile, key), are dealt to W workgroups in equal
 * shares of neighbours: workgroup w takes units [w U / W, (w + 1) U / W). So a batch of one long
 * and many short sequences keeps every workgroup as busy as one of equal lengths, with the lengths
 * known on the device alone. The price is a scan over the sequences ahead of the work, and items
 * cut by a border, whose pieces are merged by the last workgroup to arrive. */
#ifndef CPG_PAGED_SCHED_H
#define CPG_PAGED_SCHED_H
#include <stdint.h>

#ifdef __HIPCC__
#define PG_FN __host__ __device__ static inline
#else
#define PG_FN static inline
#endif

#define PG_UL 7             /* log2 of the keys per unit of work */
#define PG_UNIT (1 << PG_UL)
#define PG_MAX_LEN (1 << 30) /* tokens of a sequence: positions and their sums stay in 32 bits */

/* the batch and its division: S sequences, T rows; parts of a kv head's query heads, log2 of a
   tile's tokens, log2 of a page's */
struct pg_batch {
    const int *q_off, *len;
    int S, T, KV, max_pages, plog, window, parts, tl;
};

PG_FN int pg_min(int a, int b) { return a < b ? a : b; }
PG_FN int pg_max(int a, int b) { return a > b ? a : b; }

struct pg_seq {
    int lo, n, len, p0;     /* first row, new rows, tokens in the cache, position of the first row */
    bool cut, bad;          /* rows outside 0 .. T; or a length that the pages cannot hold */
};

PG_FN pg_seq pg_get_seq(const int *q_off, const int *len,
                                           int s, int T, int max_pages, int plog) {
    const int a = q_off[s], b = q_off[s + 1], L = len[s];
    pg_seq r;
    r.lo = pg_min(pg_max(a, 0), T);
    const int hi = pg_min(pg_max(b, r.lo), T);
    r.n = hi - r.lo;
    r.cut = a != r.lo || b != hi;
    r.bad = r.cut || L < 0 || L > PG_MAX_LEN || (int64_t)L > ((int64_t)max_pages << plog);
    r.len = r.bad ? 0 : L;
    r.p0 = r.len - r.n;
    return r;
}

/* sum of floor(y / 2^k) over y < z */
PG_FN int64_t pg_floor_sum(int z, int k) {
    const int64_t q = z >> k, r = z & ((1 << k) - 1);
    return ((q * (q - 1)) << k >> 1) + r * q;
}

PG_FN int pg_tiles(const pg_seq &s, int tl) { return (s.n + (1 << tl) - 1) >> tl; }

/* first and past-the-last unit of the keys that tile i sees; one empty unit where it sees none */
PG_FN int pg_unit_lo(const pg_seq &s, int tl, int window, int i) {
    return window > 0 ? pg_max(0, s.p0 + (i << tl) - window + 1) >> PG_UL : 0;
}

/* units of the tiles before tile x of a sequence (every tile has one at least, so that the rows
   without a key are written too): with the position of a tile's last row a_i = p0 + (i + 1) TB - 1,
   the sum of floor(a_i / UNIT) + 1 - floor(b_i / UNIT) over the tiles with a key, b_i the first key
   that the tile's first row sees, in closed form since TB divides UNIT */
PG_FN int64_t pg_units_before(const pg_seq &s, int tl, int window, int x) {
    const int nt = pg_tiles(s, tl);
    const int i0 = s.len <= 0 ? nt : s.p0 >= 0 ? 0 : (-s.p0) >> tl;   /* first tile with a key */
    if (x <= i0) return x;
    const int c = x - i0, k = PG_UL - tl;
    const int A = (s.p0 + ((i0 + 1) << tl) - 1) >> tl;
    int64_t sum = x + pg_floor_sum(A + c, k) - pg_floor_sum(A, k);
    if (x == nt)                                 /* the last tile may be short */
        sum += ((s.p0 + s.n - 1) >> PG_UL) - ((A + c - 1) >> k);
    if (window > 0) {
        const int64_t need = (int64_t)window - 1 - s.p0;              /* b_i >= 0 from here on */
        const int64_t i1 = need <= 0 ? 0 : (need + (1 << tl) - 1) >> tl;
        const int j = i1 > i0 ? (int)(i1 < x ? i1 : x) : i0;
        if (j < x) {
            const int B = (s.p0 + (j << tl) - window + 1) >> tl;
            sum -= pg_floor_sum(B + x - j, k) - pg_floor_sum(B, k);
        }
    }
    return sum;
}

/* The share of a workgroup. Workgroups
   beyond the number of units have none, so that between two that share an item every one has a
   piece of it. Neighbours in the order of units are on one XCD where every workgroup has a share
   (their tiles read the same keys; workgroup i of a launch runs on XCD i % 8), and spread over the
   XCDs where not. */
struct pg_share {
    int w, W;               /* this workgroup, of those that have a share */
    int64_t U, u0, u1;      /* all units, and this workgroup's */
    int s;                  /* the sequence of u0, and the units before u0 in it */
    int64_t rem;
};

PG_FN void pg_deal(pg_share &r, int block, int grid) {
    r.W = r.U < grid ? (int)r.U : grid;
    r.w = r.W < grid || grid % 8 ? block : block % 8 * (grid / 8) + block / 8;
    const bool some = r.w < r.W;
    r.u0 = some ? r.w * r.U / r.W : 0;
    r.u1 = some ? (r.w + 1) * r.U / r.W : 0;
}

/* the workgroup that has unit u */
PG_FN int pg_owner(int64_t u, int64_t U, int W) { return (int)(((u + 1) * W - 1) / U); }

/* a walk over a share's items */
struct pg_item {
    pg_seq q;
    int s, kv, part, tile;  /* the item */
    int off, cnt;           /* its units from `off` on, cnt of them, are this workgroup's */
    int all;                /* its units */
    int64_t first;          /* the number of its first unit among all */
};

/* the item at unit u (u0 <= u < u1) of the share; s and rem are moved on past it */
PG_FN pg_item pg_next_item(const pg_batch &b, int64_t u, int64_t u1, int &s,
                                              int64_t &rem) {
    pg_item it;
    int64_t per;
    for (;;) {
        it.q = pg_get_seq(b.q_off, b.len, s, b.T, b.max_pages, b.plog);
        per = it.q.n ? pg_units_before(it.q, b.tl, b.window, pg_tiles(it.q, b.tl)) : 0;
        if (rem < per * b.KV * b.parts || s + 1 >= b.S) break;
        s++;
        rem = 0;
    }
    it.s = s;
    const uint32_t kp = (uint32_t)(rem / per);
    const int64_t in = rem - kp * per;
    it.kv = kp / b.parts;
    it.part = kp % b.parts;
    int lo = 0, hi = pg_tiles(it.q, b.tl);       /* the tile: units_before(lo) <= in < units_before(hi) */
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pg_units_before(it.q, b.tl, b.window, mid) <= in) lo = mid;
        else hi = mid;
    }
    it.tile = lo;
    const int64_t ahead = pg_units_before(it.q, b.tl, b.window, lo);
    it.all = (int)(pg_units_before(it.q, b.tl, b.window, lo + 1) - ahead);
    it.off = (int)(in - ahead);
    it.first = u - it.off;
    const int64_t left = u1 - u;
    it.cnt = it.all - it.off < left ? it.all - it.off : (int)left;
    rem += it.cnt;
    return it;
}

#endif
