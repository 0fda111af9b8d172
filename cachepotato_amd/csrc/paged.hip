/* paged.hip — the paged key/value cache: the new tokens' heads into it (cpg_paged_append), and the
 * host side of the attention over it (cpg_paged_attn, whose kernels are in paged_few.hip).
 */
#include "cpg_paged.h"

#include <math.h>
#include <stdlib.h>

/* ---------------------------------------------------------------- append */

/* k_paged_append: heads a lane, from APPEND_NI_ROWS rows on (below, one: a launch of few rows is
   shorter with more workgroups). us for 1, 2, 3 and 4: prompts of 9 k rows, 32 heads on 8, bf16
   57.0, 53.6, 48.7 (4.8 TB/s in and out, a copy's rate), 49.2; 512 rows, 32 on 4, f32 7.9, 8.4, 8.9,
   9.3 */
#define APPEND_NI 3
#define APPEND_NI_ROWS 2048

struct pg_append {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    const int *pages, *q_off, *len;
    int64_t ldq, ldk, ldv, ldqo, page_stride, slot_stride, head_stride;
    const float *table, *q_norm, *k_norm;
    int H, KV, HD, S, T, max_pages, n_pages, plog, max_pos, rot, adjacent, *stat;
    float eps;
};

/* The last sequence s with q_off[s] <= t (-1: none), for ascending q_off: 64 probes a step, so one
   step up to 64 sequences and two up to 4096. Whole wavefront. */
__device__ static inline int pg_row_seq(const int *__restrict__ q_off, int S, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = S;                           /* the answer is lo - 1 or in [lo, lo + n) */
    while (n > 0) {
        const int step = (n + 63) >> 6, i = lo + lane * step;
        const bool yes = i < lo + n && q_off[i] <= t;
        const int c = __popcll(__ballot(yes));
        if (c == 0) return lo - 1;
        const int end = lo + n;
        lo += (c - 1) * step + 1;                /* probe c - 1 said yes, probe c no */
        n = min(step - 1, end - lo);
    }
    return lo - 1;
}

/* grid (T, parts of the H + 2 KV heads), 256 threads: row t, 2^gl lanes to a head, eight elements a
   lane (HD = 96 and 192 leave a quarter of the lanes idle), NI heads a lane, 256 >> gl apart. A query or
   key head is normed (its sum of squares over the lanes in fp32), turned, and rounded once where it
   is stored; a value head is only stored. The partner of a lane's elements in the rotation is a
   lane's whole eight, since rot is a multiple of 16: rot / 16 lanes away, or its own. A lane's place in
   its heads is the same, so the row's search, page and rotation pairs serve all of them.
   Bound by the bytes of the heads in and out (APPEND_NI); for a few rows by the chain of launch,
   row's sequence, page id, store: 3.3 us for one row. */
template <int AT, int CT, int NI>
__global__ __launch_bounds__(256) void k_paged_append(const pg_append a, int gl) {
    const int t = blockIdx.x, tid = threadIdx.x, li = tid & ((1 << gl) - 1), hpw = 256 >> gl;
    const int head0 = blockIdx.y * NI * hpw + (tid >> gl), heads = a.H + 2 * a.KV;
    const bool in = li * 8 < a.HD;
    const int lc = min(li, a.HD / 8 - 1);
    typedef typename pg_elem<AT>::t at;
    constexpr int NR = AT == CPG_T_F32 ? 2 : 1;
    uint4 raw[NI][NR];
#pragma unroll
    for (int i = 0; i < NI; i++) {               /* unconditional, a head past the last the last */
        const int hc = min(head0 + i * hpw, heads - 1);
        const bool isq = hc < a.H, isv = hc >= a.H + a.KV;
        const int hh = isq ? hc : isv ? hc - a.H - a.KV : hc - a.H;
        const at *src = (const at *)(isq ? a.q : isv ? a.v : a.k) +
                        (size_t)t * (isq ? a.ldq : isv ? a.ldv : a.ldk) + (size_t)hh * a.HD + 8 * lc;
#pragma unroll
        for (int j = 0; j < NR; j++) raw[i][j] = ((const uint4 *)src)[j];
    }
    const int s = pg_row_seq(a.q_off, a.S, t);
    if (s < 0) return;
    const pg_seq sq = pg_get_seq(a.q_off, a.len, s, a.T, a.max_pages, a.plog);
    if (t < sq.lo || t >= sq.lo + sq.n) {        /* a row of no sequence */
        if (sq.bad && tid == 0) *a.stat = 1;
        return;
    }
    const int pos = sq.p0 + t - sq.lo;
    const bool bad = sq.bad || pos < 0 || (a.rot > 0 && pos >= a.max_pos);
    const int pc = bad ? 0 : pos;
    const int page = bad ? -1 : a.pages[(size_t)s * a.max_pages + (pc >> a.plog)];
    const bool miss = page < 0 || page >= a.n_pages;
    if (miss && tid == 0) *a.stat = 1;
    /* the lane's rotation: pairs of its elements and of another lane's (halves), or among its own */
    const bool turn = 8 * li < a.rot;
    const int hl = a.rot / 16;                   /* lanes of half the rotated elements */
    const bool upper = li >= hl;
    const int lane = tid & 63, other = turn ? (upper ? lane - hl : lane + hl) : lane;
    float cs[8], sn[8];
    if (a.rot > 0) {
        const float4 *row = (const float4 *)(a.table + (size_t)pc * a.rot);
#pragma unroll
        for (int i = 0; i < 4; i++) {            /* two pairs to a float4 */
            const float4 r = row[a.adjacent ? (turn ? 2 * li + (i >> 1) : 0)
                                            : (turn ? 4 * (upper ? li - hl : li) : 0) + i];
            cs[2 * i] = r.x; sn[2 * i] = r.y; cs[2 * i + 1] = r.z; sn[2 * i + 1] = r.w;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int head = head0 + i * hpw, hc = min(head, heads - 1);
        const bool isq = hc < a.H, isv = hc >= a.H + a.KV;
        const int hh = isq ? hc : isv ? hc - a.H - a.KV : hc - a.H;
        float x[8];
        if constexpr (AT == CPG_T_F32) {
            const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                                   raw[i][NR - 1].x, raw[i][NR - 1].y, raw[i][NR - 1].z, raw[i][NR - 1].w};
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = __uint_as_float(w[j]);
        } else {
            const uint32_t w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = pg_unpack2<AT>(w[j]);
                x[2 * j] = f.x;
                x[2 * j + 1] = f.y;
            }
        }
        const float *gain = isq ? a.q_norm : a.k_norm;
        if (a.q_norm || a.k_norm) {              /* shuffles: every lane takes part */
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) ss = fmaf(x[j], x[j], ss);
            ss = in ? ss : 0.0f;
            for (int o = 1; o < 1 << gl; o <<= 1) ss += __shfl_xor(ss, o);
            if (gain && !isv) {
                const float inv = __fdiv_rn(1.0f, cpg_sqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.HD), a.eps)));
                const float4 g0 = ((const float4 *)gain)[2 * lc], g1 = ((const float4 *)gain)[2 * lc + 1];
                const float g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = __fmul_rn(__fmul_rn(x[j], inv), g[j]);
            }
        }
        if (a.rot > 0 && a.adjacent) {
            if (turn && !isv)
#pragma unroll
                for (int j = 0; j < 4; j++) {    /* pair j of the lane: read as pairs 2 (j / 2) + j % 2 */
                    const int c = 4 * (j >> 1) + (j & 1);
                    const float u = x[2 * j], w = x[2 * j + 1];
                    x[2 * j] = __fsub_rn(__fmul_rn(u, cs[c]), __fmul_rn(w, sn[c]));
                    x[2 * j + 1] = __fadd_rn(__fmul_rn(w, cs[c]), __fmul_rn(u, sn[c]));
                }
        } else if (a.rot > 0) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = __shfl(x[j], other);
                const float down = __fsub_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y, sn[j]));
                const float up = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y, sn[j]));
                x[j] = turn && !isv ? (upper ? up : down) : x[j];
            }
        }
        if (!in || head >= heads) continue;
        if (isq) {
            if (bad)
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = __int_as_float(0x7fc00000);
            pg_put8<AT>(a.q_out, (size_t)t * a.ldqo + (size_t)hh * a.HD + 8 * li, x);
        } else if (!miss) {
            pg_put8<CT>(isv ? a.vc : a.kc,
                        (size_t)page * a.page_stride + (size_t)(pos & ((1 << a.plog) - 1)) * a.slot_stride +
                            (size_t)hh * a.head_stride + 8 * li, x);
        }
    }
}

/* ---------------------------------------------------------------- host side */

static int elem_bytes(int type) { return type == CPG_T_F32 ? 4 : 2; }

static bool types_ok(int type, int cache) {
    return (type == CPG_T_F32 && cache >= CPG_T_F32 && cache <= CPG_T_BF16) ||
           ((type == CPG_T_F16 || type == CPG_T_BF16) && cache == type);
}

static bool head_dim_ok(int HD) { return HD == 64 || HD == 96 || HD == 128 || HD == 192 || HD == 256; }

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

/* rows of `heads` heads, `ld` elements apart, at p */
static bool rows_ok(const void *p, int64_t ld, int heads, int HD, int type) {
    return p && aligned16(p) && ld >= (int64_t)heads * HD && ld * elem_bytes(type) % 16 == 0;
}

/* log2 of the largest power of two of bytes that divides both strides of a slot's offset in the pool */
static int row_shift(const cpg_paged_cache *C) {
    const int64_t all = (C->n_pages > 1 ? C->page_stride : 0) | (C->page > 1 ? C->slot_stride : 0);
    int s = 4;
    while (s < 20 && !(all * elem_bytes(C->type) >> s & 1)) s++;
    return s;
}

/* the checks that both entry points make, of the arguments and then of the workspace; 0, or -1
   with the reason set */
static int check_call(const char *who, const cpg_paged_cache *C, const cpg_paged_batch *B, int type) {
    if (!C || !B || !C->k || !C->v) {
        cpg_set_error("%s: null argument", who);
        return -1;
    }
    if (!types_ok(type, C->type)) {
        cpg_set_error("%s: activations of type %d with a cache of type %d", who, type, C->type);
        return -1;
    }
    if (!head_dim_ok(C->HD) || C->KV <= 0) {
        cpg_set_error("%s: KV=%d, HD=%d (64, 96, 128, 192 or 256)", who, C->KV, C->HD);
        return -1;
    }
    if (C->page <= 0 || C->page > 1024 || (C->page & (C->page - 1)) || C->n_pages <= 0) {
        cpg_set_error("%s: %d pages of %d tokens (a power of two up to 1024)", who, C->n_pages, C->page);
        return -1;
    }
    const int eb = elem_bytes(C->type);
    const int64_t st[3] = {C->page_stride, C->slot_stride, C->head_stride};
    const int64_t n[3] = {C->n_pages, C->page, C->KV};
    for (int i = 0; i < 3; i++) {
        if (st[i] * eb % 16 || (n[i] > 1 && st[i] < C->HD) || st[i] < 0 ||
            (n[i] > 1 && st[i] > ((int64_t)1 << 56) / n[i])) {
            cpg_set_error("%s: stride %lld (at least HD elements, a multiple of 16 bytes)", who,
                          (long long)st[i]);
            return -1;
        }
    }
    /* slots are found at 32-bit offsets in units of row_shift: at least 64 GiB, 1 TiB for strides of
       256 bytes */
    const double last = ((double)(C->n_pages - 1) * (n[0] > 1 ? st[0] : 0) + (double)(C->page - 1) * (n[1] > 1 ? st[1] : 0)) * eb;
    if (ldexp(last, -row_shift(C)) >= 4294967040.0) {
        cpg_set_error("%s: a pool of %.0f bytes is too large for its strides", who, last);
        return -1;
    }
    if (!aligned16(C->k) || !aligned16(C->v)) {
        cpg_set_error("%s: the pool is not aligned to 16 bytes", who);
        return -1;
    }
    if (B->S < 0 || B->S > PG_MAX_LEN || B->T < 0 || B->T > PG_MAX_LEN || B->max_pages < 0 ||
        (B->S > 0 && B->T > 0 && (!B->q_off || !B->len || !B->pages || B->max_pages == 0))) {
        cpg_set_error("%s: bad batch S=%d T=%d max_pages=%d", who, B->S, B->T, B->max_pages);
        return -1;
    }
    return 0;
}

static int check_ws(const char *who, const cpg_paged_ws *ws, int H, const cpg_paged_cache *C) {
    if (!ws) {
        cpg_set_error("%s: null workspace", who);
        return -1;
    }
    if (H != ws->H || C->KV != ws->KV || C->HD != ws->HD) {
        cpg_set_error("%s: H=%d KV=%d HD=%d, the workspace's H=%d KV=%d HD=%d", who, H, C->KV, C->HD,
                      ws->H, ws->KV, ws->HD);
        return -1;
    }
    return 0;
}

static int log2_of(int x) {
    int l = 0;
    while ((1 << l) < x) l++;
    return l;
}

/* tiles of `rows` query rows of a kv head: query heads of a row's token, parts that a kv head's make,
   tokens, and the most tiles that the batch can have (of each part) */
struct pg_tiling {
    int hpp, parts, log2_tokens;
    double tiles;
};

static pg_tiling tiling(const cpg_paged_batch *B, int G, int rows) {
    pg_tiling t = {G < rows ? G : rows, 0, 0, 0.0};
    t.parts = (G + t.hpp - 1) / t.hpp;
    while ((2 << t.log2_tokens) * t.hpp <= rows) t.log2_tokens++;
    t.tiles = (double)(B->T >> t.log2_tokens) + (B->S < B->T ? B->S : B->T);
    return t;
}

extern "C" cpg_paged_ws *cpg_paged_ws_create(int H, int KV, int HD) {
    if (!g_cpg.ready) { cpg_set_error("cpg_init has not been called"); return nullptr; }
    if (H <= 0 || KV <= 0 || H % KV || !head_dim_ok(HD) || H > 65536) {
        cpg_set_error("cpg_paged_ws_create: bad geometry H=%d KV=%d HD=%d", H, KV, HD);
        return nullptr;
    }
    cpg_paged_ws *ws = (cpg_paged_ws *)calloc(1, sizeof *ws);
    if (!ws) { cpg_set_error("out of host memory"); return nullptr; }
    ws->H = H;
    ws->KV = KV;
    ws->HD = HD;
    ws->rows = (size_t)2 * PG_MANY_WGS * PG_MANY_ROWS;     /* k_paged_few needs an eighth */
    const size_t sz[5] = {ws->rows * HD * 4, ws->rows * 8, (size_t)3 * PG_MANY_WGS * 4, 4, 2048};
    size_t total = 0;
    for (int i = 0; i < 5; i++) total += cpg_round256(sz[i]);
    uint8_t *p = (uint8_t *)cpg_malloc(total);
    if (!p) { free(ws); return nullptr; }
    ws->block = p;
    void **dst[5] = {(void **)&ws->pacc, (void **)&ws->pml, (void **)&ws->ctr, (void **)&ws->stat,
                     (void **)&ws->blank};
    for (int i = 0; i < 5; i++) {
        *dst[i] = p;
        p += cpg_round256(sz[i]);
    }
    /* every bit set is a NaN in all three element types */
    if (cpg_memset(ws->ctr, 0, sz[2]) || cpg_memset(ws->stat, 0, 4) ||
        cpg_memset(ws->blank, 0, 1024) || cpg_memset(ws->blank + 1024, 255, 1024)) {
        cpg_paged_ws_destroy(ws);
        return nullptr;
    }
    return ws;
}

extern "C" void cpg_paged_ws_destroy(cpg_paged_ws *ws) {
    if (!ws) return;
    cpg_free(ws->block);
    free(ws);
}

extern "C" int cpg_paged_ws_status(cpg_paged_ws *ws) {
    CPG_REQUIRE_INIT();
    if (!ws) { cpg_set_error("cpg_paged_ws_status: null workspace"); return -1; }
    int v = 0;
    if (cpg_sync() || cpg_d2h(&v, ws->stat, sizeof v)) return -7;
    if (v && cpg_memset(ws->stat, 0, sizeof v)) return -7;
    return v;
}

template <int NI> static int launch_append(const pg_append &a, int type, int cache) {
    const int gl = log2_of(a.HD / 8), hpw = (256 >> gl) * NI;
    const dim3 grid(a.T, (a.H + 2 * a.KV + hpw - 1) / hpw);
    auto kernel = type == CPG_T_F16    ? k_paged_append<CPG_T_F16, CPG_T_F16, NI>
                  : type == CPG_T_BF16 ? k_paged_append<CPG_T_BF16, CPG_T_BF16, NI>
                  : cache == CPG_T_F32 ? k_paged_append<CPG_T_F32, CPG_T_F32, NI>
                  : cache == CPG_T_F16 ? k_paged_append<CPG_T_F32, CPG_T_F16, NI>
                                       : k_paged_append<CPG_T_F32, CPG_T_BF16, NI>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, g_cpg.stream, a, gl);
    CPG_LAUNCH_CHECK("k_paged_append");
    return 0;
}

extern "C" int cpg_paged_append(const cpg_paged_cache *C, const cpg_paged_batch *B,
                                const cpg_paged_rope *R, int type, int H, const void *q, int64_t ldq,
                                const void *k, int64_t ldk, const void *v, int64_t ldv, void *q_out,
                                int64_t ldqo, cpg_paged_ws *ws) {
    if (check_call("cpg_paged_append", C, B, type)) return -1;
    if (H < 0 || H > 65536) { cpg_set_error("cpg_paged_append: %d query heads", H); return -1; }
    if (!rows_ok(k, ldk, C->KV, C->HD, type) || !rows_ok(v, ldv, C->KV, C->HD, type) ||
        (H && (!rows_ok(q, ldq, H, C->HD, type) || !rows_ok(q_out, ldqo, H, C->HD, type)))) {
        cpg_set_error("cpg_paged_append: rows of heads must not be null or overlap, and start on 16 bytes");
        return -1;
    }
    pg_append a = {};
    if (R) {
        if (R->rot < 0 || R->rot > C->HD || R->rot % 16 ||
            (R->rot && (!R->table || !aligned16(R->table) || R->max_pos <= 0)) ||
            (R->pairs != CPG_ROPE_HALVES && R->pairs != CPG_ROPE_ADJACENT)) {
            cpg_set_error("cpg_paged_append: bad rotation (rot=%d, a multiple of 16 up to HD=%d; "
                          "max_pos=%d; pairs=%d)", R->rot, C->HD, R->max_pos, R->pairs);
            return -1;
        }
        if ((R->q_norm && !aligned16(R->q_norm)) || (R->k_norm && !aligned16(R->k_norm)) ||
            ((R->q_norm || R->k_norm) && !(R->eps >= 0.0f && R->eps < INFINITY))) {
            cpg_set_error("cpg_paged_append: bad head norm (gains on 16 bytes, eps=%g)", R->eps);
            return -1;
        }
        a.table = R->table;
        a.max_pos = R->max_pos;
        a.rot = R->rot;
        a.adjacent = R->pairs == CPG_ROPE_ADJACENT;
        a.q_norm = R->q_norm;
        a.k_norm = R->k_norm;
        a.eps = R->eps;
    }
    if (check_ws("cpg_paged_append", ws, H ? H : ws ? ws->H : 0, C)) return -1;
    CPG_REQUIRE_INIT();
    if (B->S == 0 || B->T == 0) return 0;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kc = C->k; a.vc = C->v;
    a.pages = B->pages; a.q_off = B->q_off; a.len = B->len;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldqo = ldqo;
    a.page_stride = C->page_stride; a.slot_stride = C->slot_stride; a.head_stride = C->head_stride;
    a.H = H; a.KV = C->KV; a.HD = C->HD; a.S = B->S; a.T = B->T;
    a.max_pages = B->max_pages; a.n_pages = C->n_pages; a.plog = log2_of(C->page);
    a.stat = ws->stat;
    return B->T < APPEND_NI_ROWS ? launch_append<1>(a, type, C->type) : launch_append<APPEND_NI>(a, type, C->type);
}

static int g_paged_mode = CPG_PAGED_AUTO;

extern "C" int cpg_paged_attn_mode(int mode) {
    if (mode != CPG_PAGED_AUTO && mode != CPG_PAGED_FEW && mode != CPG_PAGED_MANY) {
        cpg_set_error("cpg_paged_attn_mode: unknown mode %d", mode);
        return -1;
    }
    g_paged_mode = mode;
    return 0;
}

extern "C" int cpg_paged_attn(const cpg_paged_cache *C, const cpg_paged_batch *B, int type, int H,
                              const void *q, int64_t ldq, float scale, int window, void *out,
                              int64_t ldo, float *lse, cpg_paged_ws *ws) {
    if (check_call("cpg_paged_attn", C, B, type)) return -1;
    if (H <= 0 || H % C->KV) { cpg_set_error("cpg_paged_attn: H=%d, KV=%d", H, C->KV); return -1; }
    if (!(scale >= 0.0f && scale < INFINITY) || window < 0) {
        cpg_set_error("cpg_paged_attn: scale %g, window %d (neither negative)", scale, window);
        return -1;
    }
    if (!rows_ok(q, ldq, H, C->HD, type) || !rows_ok(out, ldo, H, C->HD, type)) {
        cpg_set_error("cpg_paged_attn: rows of heads must not be null or overlap, and start on 16 bytes");
        return -1;
    }
    if (check_ws("cpg_paged_attn", ws, H, C)) return -1;
    CPG_REQUIRE_INIT();
    if (B->S == 0 || B->T == 0) return 0;
    pg_args a = {};
    const int eb = elem_bytes(C->type);
    a.q = q; a.out = out; a.lse = lse; a.pages = B->pages;
    a.k = (const uint8_t *)C->k; a.v = (const uint8_t *)C->v;
    a.ldq = ldq; a.ldo = ldo; a.head_bytes = C->head_stride * eb;
    a.H = H; a.G = H / C->KV; a.n_pages = C->n_pages;
    a.ush = row_shift(C);
    a.page_units = (uint32_t)(C->page_stride * eb >> a.ush);
    a.slot_units = (uint32_t)(C->slot_stride * eb >> a.ush);
    a.scale2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)C->HD)) * 1.4426950408889634f;
    a.blank = ws->blank;
    a.pacc = ws->pacc; a.pml = ws->pml; a.ctr = ws->ctr; a.stat = ws->stat;
    /* k_paged_few reads a sequence's keys again for each 16 query rows of a kv head, k_paged_many for
       each 128: it is ahead where that is the same, and where the items (tiles of 16 rows) are so
       few that the time is the length of the launch. us, few and many: f32, 32 heads on 4, one
       sequence over 3000, 44 items 28.6 and 31.4, 96 items 44.4 and 43.2; 8 over 700, 64 items 20.8 and
       22.9, 128 items 25.7 and 24.1; bf16, 32 heads on 8, 8 over 3000, 128 items 27.8 and 32.2, 384
       items 60.7 and 37.4. (One sequence over 12000, f32, 44 items 66.3 and 53.9.) */
    const pg_tiling t16 = tiling(B, a.G, PG_FEW_ROWS);
    const bool few = g_paged_mode != CPG_PAGED_AUTO
                         ? g_paged_mode == CPG_PAGED_FEW
                         : (int64_t)B->max_new * a.G <= PG_FEW_ROWS ||
                               t16.tiles * C->KV * t16.parts <= (C->type == CPG_T_F32 ? 64 : 128);
    const int rows = few ? PG_FEW_ROWS : PG_MANY_ROWS;
    const pg_tiling tl = few ? t16 : tiling(B, a.G, rows);
    a.hpp = tl.hpp;
    a.hinv = (65536 + a.hpp - 1) / a.hpp;
    /* a unit is 128 keys: one step of the four wavefronts of k_paged_few for a 16-bit cache (half
       as many for an f32 one), two or four steps of k_paged_many; more where the units of the
       largest batch there can be would not fit 31 bits. What an item counts for beside its keys,
       us for 0, 1, 2 and 3 units: prompts of 1500-4500, bf16 295, 260, 251, 253; 512 tokens over 3584,
       f32 132, 129, 135, 135; one token each, 16 conversations, f32 20.8, 19.0, 17.1; 96 sequences,
       bf16 202, 207 */
    a.b = pg_batch{B->q_off, B->len, B->S, B->T, C->KV, B->max_pages, log2_of(C->page),
                   window < PG_MAX_LEN ? window : 0, tl.parts, tl.log2_tokens,
                   few && C->type == CPG_T_F32 ? 6 : 7, few ? (C->type == CPG_T_F32 ? 2 : 0) : C->type == CPG_T_F32 ? 1 : 2};
    /* no more workgroups than units there can be: tiles of the rows, and keys of a full page row */
    double units;
    for (;; a.b.ul++) {
        units = tl.tiles * C->KV * a.b.parts * (a.b.extra + ceil(ldexp((double)B->max_pages, a.b.plog - a.b.ul)));
        if (units < 2147483648.0 || a.b.ul >= 30) break;
    }
    if (units >= 2147483648.0) {
        cpg_set_error("cpg_paged_attn: a batch of %d rows and %d sequences of %d heads is too large", B->T, B->S, H);
        return -1;
    }
    const int most = few ? PG_FEW_WGS : C->HD <= 128 ? PG_MANY_WGS : PG_MANY_WGS / 2;
    const int grid = units < most ? (int)units : most;
    if (!few) return pg_launch_many(a, type, C->type, C->HD, grid);
    return pg_launch_few(a, type, C->type, C->HD, grid);
}
