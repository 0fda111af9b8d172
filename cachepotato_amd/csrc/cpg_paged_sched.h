/* cpg_paged_sched.h — how the work of an attention call over the paged cache is divided. Integer
 * arithmetic alone, for the kernels and, compiled as plain C++, for the tests.
 *
 * Work. The rows of a sequence are taken in tiles of TB = 2^tl tokens (times the query heads of one
 * kv head), and a tile's visible keys in units of UNIT. An item is one tile of one kv head (and of
 * one part of its query heads, where they are more than a tile's rows). The units of all items,
 * U of them in the order (sequence, kv head and part, tile, key), are dealt to W workgroups in equal
 * shares of neighbours. So a batch of one long and many short sequences keeps
 * every workgroup as busy as one of equal lengths, with the lengths known on the device alone. The
 * price is a scan over the sequences ahead of the work (0.7 us), and items cut by a border, whose
 * pieces are merged by the last workgroups to arrive (3 us with the arrival). */
#ifndef CPG_PAGED_SCHED_H
#define CPG_PAGED_SCHED_H
#include <stdint.h>

#ifdef __HIPCC__
#define PG_FN __host__ __device__ static inline
#else
#define PG_FN static inline
#endif

#define PG_MAX_LEN (1 << 30) /* tokens of a sequence: positions and their sums stay in 32 bits */

/* the batch and its division: S sequences, T rows; parts of a kv head's query heads; log2 of the
   tokens of a page, of those of a tile and of the keys of a unit (tl <= ul); the units that an item
   counts for ahead of its keys (its start and its end take the time of some) */
struct pg_batch {
    const int *q_off, *len;
    int S, T, KV, max_pages, plog, window, parts, tl, ul, extra;
};

PG_FN int pg_min(int a, int b) { return a < b ? a : b; }
PG_FN int pg_max(int a, int b) { return a > b ? a : b; }

struct pg_seq {
    int lo, n, len, p0;     /* first row, new rows, tokens in the cache, position of the first row */
    bool cut, bad;          /* rows outside 0 .. T; or a length that the pages cannot hold */
};

PG_FN pg_seq pg_get_seq(const int *q_off, const int *len, int s, int T, int max_pages, int plog) {
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

/* sum of floor(y / 2^k) over y < z, modulo 2^32 (differences of it are used) */
PG_FN uint32_t pg_floor_sum(uint32_t z, int k) {
    const uint32_t q = z >> k, r = z & ((1u << k) - 1);
    return ((q & 1 ? q * ((q - 1) >> 1) : (q >> 1) * (q - 1)) << k) + r * q;
}

PG_FN int pg_tiles(const pg_seq &s, int tl) { return (int)(((uint32_t)s.n + (1u << tl) - 1) >> tl); }

/* first unit of the keys that tile i sees */
PG_FN int pg_unit_lo(const pg_batch &b, const pg_seq &s, int i) {
    return b.window > 0 ? pg_max(0, s.p0 + (i << b.tl) - b.window + 1) >> b.ul : 0;
}

/* units of the tiles before tile x of a sequence (every tile has one at least, so that the rows
   without a key are written too): with the position of a tile's last row a_i = p0 + (i + 1) TB - 1,
   the sum of floor(a_i / UNIT) + 1 - floor(b_i / UNIT) over the tiles with a key, b_i the first key
   that the tile's first row sees, in closed form since TB divides UNIT; and `extra` for each tile */
PG_FN uint32_t pg_units_before(const pg_batch &b, const pg_seq &s, int x) {
    const int nt = pg_tiles(s, b.tl), tl = b.tl;
    const int i0 = s.len <= 0 ? nt : s.p0 >= 0 ? 0 : (-s.p0) >> tl;   /* first tile with a key */
    const uint32_t more = (uint32_t)x * (uint32_t)b.extra;
    if (x <= i0) return (uint32_t)x + more;
    const int c = x - i0, k = b.ul - tl;
    const int A = (s.p0 + ((i0 + 1) << tl) - 1) >> tl;
    uint32_t sum = (uint32_t)x + more + pg_floor_sum(A + c, k) - pg_floor_sum(A, k);
    if (x == nt)                                 /* the last tile may be short */
        sum += (uint32_t)(((s.p0 + s.n - 1) >> b.ul) - ((A + c - 1) >> k));
    if (b.window > 0) {
        const int need = b.window - 1 - s.p0;    /* b_i >= 0 from tile i1 on */
        const int i1 = need <= 0 ? 0 : (int)(((uint32_t)need + (1u << tl) - 1) >> tl);
        const int j = i1 > i0 ? pg_min(i1, x) : i0;
        if (j < x) {
            const int B = (s.p0 + (j << tl) - b.window + 1) >> tl;
            sum -= pg_floor_sum(B + x - j, k) - pg_floor_sum(B, k);
        }
    }
    return sum;
}

/* the units of a whole sequence, of all its kv heads and parts */
PG_FN uint32_t pg_seq_units(const pg_batch &b, const pg_seq &s) {
    return s.n ? pg_units_before(b, s, pg_tiles(s, b.tl)) * (uint32_t)(b.KV * b.parts) : 0;
}

/* The share of a workgroup: U / W units, one more for the first U % W. Workgroups beyond the number
   of units have none, so that between two that share an item every one has a piece of it. Neighbours
   in the order of units are on one XCD where every workgroup has a share (their tiles read the same
   keys; workgroup i of a launch runs on XCD i % 8), and spread over the XCDs where not. */
struct pg_share {
    int w, W;               /* this workgroup, of those that have a share */
    uint32_t U, u0, u1;     /* all units, and this workgroup's */
};

PG_FN pg_share pg_deal(uint32_t U, int block, int grid) {
    pg_share r;
    r.U = U;
    r.W = U < (uint32_t)grid ? (int)U : grid;
    r.w = r.W < grid || grid % 8 ? block : block % 8 * (grid / 8) + block / 8;
    r.u0 = r.u1 = 0;
    if (r.w < r.W) {
        const uint32_t per = U / (uint32_t)r.W, more = U - per * r.W, w = (uint32_t)r.w;
        r.u0 = w * per + (w < more ? w : more);
        r.u1 = r.u0 + per + (w < more);
    }
    return r;
}

/* the workgroup that has unit u */
PG_FN int pg_owner(uint32_t u, uint32_t U, int W) {
    const uint32_t per = U / (uint32_t)W, more = U - per * W, wide = more * (per + 1);
    return (int)(u < wide ? u / (per + 1) : more + (u - wide) / per);
}

/* a walk over a share's items */
struct pg_item {
    int kv, part, tile;     /* the item */
    int step;               /* units to go on by */
    int off, cnt;           /* its units of keys from `off` on, cnt of them, are this workgroup's; none
                               where the share ends in the units ahead of the keys */
    int all;                /* its units of keys */
    uint32_t first;         /* the number of its first unit of keys among all units */
};

/* the item of sequence q at unit u (below u1, `rem` units into the sequence) */
PG_FN pg_item pg_find_item(const pg_batch &b, const pg_seq &q, uint32_t u, uint32_t u1, uint32_t rem) {
    pg_item it;
    const int nt = pg_tiles(q, b.tl);
    const uint32_t per = pg_units_before(b, q, nt), kp = rem / per, in = rem - kp * per;
    it.kv = b.parts == 1 ? (int)kp : (int)(kp / (uint32_t)b.parts);
    it.part = (int)kp - it.kv * b.parts;
    uint32_t ahead = 0, upto = per;
    int lo = 0, hi = nt;                         /* units_before(lo) <= in < units_before(hi) */
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const uint32_t x = pg_units_before(b, q, mid);
        if (x <= in) { lo = mid; ahead = x; }
        else { hi = mid; upto = x; }
    }
    it.tile = lo;
    const int at = (int)(in - ahead);            /* of the item's units, those ahead of the keys first */
    it.step = pg_min((int)(upto - ahead) - at, (int)(u1 - u));
    it.all = (int)(upto - ahead) - b.extra;
    it.off = pg_max(at - b.extra, 0);
    it.cnt = at + it.step - b.extra - it.off;
    it.first = u - at + b.extra;
    return it;
}

#endif
