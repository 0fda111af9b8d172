/* paged_many.hip — attention of many new tokens per sequence over the paged cache: prompts' chunks.
 *
 * The mathematics of k_paged_few (scores, running maximum, weights, sums). A tile is 128 query rows
 * of one sequence and kv head: TB tokens times the kv head's query heads, 32 rows to each of four
 * wavefronts, which share the keys and values that the workgroup stages in LDS, KT keys a time in two
 * buffers: while one is computed on, the other is filled.
 *
 * Layouts. S^T = K Q^T and O^T = V^T P^T on the 32x32x16 matrix instruction: a lane holds one query
 * (l % 32) throughout, so the maximum, the sum and the rescaling are a lane's own affair but for
 * one exchange between the wavefront's halves. In S^T it holds the keys 8 b + 4 (l / 32) + i; taken
 * in that order (blocks b in pairs) they are the operand P^T of the second product without a move, and
 * V^T's operand, eight keys of one element, comes from rows of values through LDS's transposing read
 * (ds_read_b64_tr_b16: of a 4 x 16 block of 16-bit elements, lane i of 16 gets column i).
 * LDS rows are 2 HDP bytes in chunks of 16, chunk c of row r at c ^ f(r): the 16 rows that a key
 * read takes at once, and the 8 rows by 2 chunk pairs of a transposing read, then lie in different
 * banks.
 *
 * 16-bit caches are copied into LDS by the memory pipe itself (global_load_lds_dwordx4); the
 * exchange of chunks is made by permuting the addresses a lane reads from. f32 caches pass
 * through registers, where each element becomes two f16 (hi and lo, 22 bits): products of K and Q,
 * V and P are then three (hi hi + hi lo + lo hi). So that f16's exponents reach, the keys and the
 * values that a wavefront stages (a quarter of the step's, eight tokens) go by powers of two where
 * their largest element is not within 2^-3 .. 2^15: the scores take the keys' back, the weights and
 * the accumulators the values' (3 % of the time; without it, values of 1e-4 were off by 3e-5 of
 * the largest, and what passed 65504 became NaN). f32 queries over 16-bit caches are two f16 or
 * three bf16 pieces (rows of queries scaled by a power of two into f16's range), and so are the
 * weights.
 *
 * The running maximum that the weights refer to is renewed only where a score passes it by 2^8: until
 * then weights above one are as good (their sum and the accumulators are fp32), and most of the
 * rescaling of the accumulators falls away.
 *
 * What bounds it: the matrix products and the softmax's vector work (exp2, maximum, sum, rounding:
 * about as many cycles as the products of 16-bit operands), the two workgroups of a CU in turn.
 * Prompts of 1500 - 4500 tokens, bf16, 32 heads of 128 on 8: 240 us, 830 TFLOP/s (a large library
 * product: 1136), matrix units busy 38 % of the cycles; 512 tokens over 3584, f32, 32 heads on 4: 120
 * us, 270 TFLOP/s, 810 with the three products of each, matrix units busy 35 %.
 */
#include "cpg_paged.h"

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

template <int CT, int AT, int HD> struct pg_many_t {
    static constexpr bool F32 = CT == CPG_T_F32;
    static constexpr int NQ = AT != CPG_T_F32 ? 1 : CT == CPG_T_BF16 ? 3 : 2;    /* pieces of q and p */
    static constexpr int NC = F32 ? 2 : 1;                       /* planes of keys and of values */
    static constexpr int OT = CT == CPG_T_BF16 ? CPG_T_BF16 : CPG_T_F16;         /* operand type */
    static constexpr int KT = F32 || NQ == 3 ? 32 : 64;          /* keys per step */
    static constexpr int HDP = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;
    static constexpr int RB = 2 * HDP, CPR = RB / 16;            /* an LDS row: bytes, chunks */
    static constexpr int PLANE = KT * RB, BUF = 2 * NC * PLANE;  /* K planes, V planes */
    static constexpr int NB = KT / 32, NS = HD / 16, ND = HD / 32;
    /* a wavefront stages RW consecutive rows. 16-bit: E copies of 1 KiB, RPE rows each; f32: E chunks
       of eight elements to a lane, of CHUNKS */
    static constexpr int RW = KT / 4, CHUNKS = RW * (HD / 8);
    static constexpr int E = F32 ? (CHUNKS + 63) / 64 : PLANE / 4096, RPE = 64 / CPR;
    static constexpr size_t SLOT = (size_t)PG_MANY_ROWS * HD * 4;  /* bytes of a piece */
    static constexpr float LIFT = OT == CPG_T_F16 ? 4.0f : 0.0f;
    __host__ __device__ static constexpr int kswz(int r) { return CPR == 8 ? (r >> 1) & 7 : r & 15; }
    __host__ __device__ static constexpr int vswz(int r) { return CPR == 8 ? ((r >> 1) & 3) << 1 : (r & 7) << 1; }
};
#define PG_NO_SCALE (-300)  /* of values that are all zero: below any other's */
#define PG_SLACK 8.0f       /* log2 of how far a score may pass the maximum that weights refer to */

template <int OT>
__device__ static inline f32x16_t pg_mfma32(uint4 a, uint4 b, f32x16_t c) {
    if constexpr (OT == CPG_T_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a),
                                                      __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

/* the maximum and the sum of a value and the other half's */
__device__ static inline float pg_half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ static inline float pg_half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

/* one global_load_lds_dwordx4: 16 bytes from each lane's address into LDS at byte lds + 16 * lane
   (lds the same for the wavefront); waits are the caller's */
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"     /* m0 is written on purpose */
__device__ static inline void pg_dma16(uint64_t p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :: "v"(p), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

typedef __attribute__((address_space(3))) uint8_t lds_u8;

template <int CT, int AT, int HD>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void k_paged_many(const pg_args a) {
    typedef pg_many_t<CT, AT, HD> P;
    constexpr bool F32 = P::F32;
    constexpr int NQ = P::NQ, NC = P::NC, OT = P::OT, KT = P::KT, RB = P::RB, CPR = P::CPR, NB = P::NB,
                  NS = P::NS, ND = P::ND, E = P::E;
    extern __shared__ __align__(16) uint8_t lds[];       /* two buffers: K planes, V planes each */
    __shared__ int flag, wild_s[4];          /* wild_s, scale_s: of a step, by its number among all steps */
    __shared__ __align__(16) int scale_s[4][4];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    pg_start at;
    const pg_share sh = pg_find_share(a.b, at, a.stat);
    const int W = sh.W, me = sh.w;
    int s = at.s;
    uint32_t rem = at.rem;
    if (tid < 4) wild_s[tid] = 0;
    __syncthreads();
    int turn = 0;                                /* steps so far */
    pg_seq sq = pg_get_seq(a.b.q_off, a.b.len, s, a.b.T, a.b.max_pages, a.b.plog);
    for (uint32_t u = sh.u0; u < sh.u1;) {
        if (rem >= pg_seq_units(a.b, sq)) {      /* the sequence is done, or brings nothing */
            s++;
            rem = 0;
            sq = pg_get_seq(a.b.q_off, a.b.len, s, a.b.T, a.b.max_pages, a.b.plog);
            continue;
        }
        const pg_item it = pg_find_item(a.b, sq, u, sh.u1, rem);
        u += it.step;
        rem += it.step;
        if (it.cnt <= 0) continue;               /* its keys are all the next workgroups' */
        /* opaque, as in k_paged_few: nothing that follows from it is held over the walk */
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int c = lane & 31, h = lane >> 5;
        /* the lane's query: row 32 w + c of the tile */
        const int t0 = it.tile << a.b.tl, tb = min(1 << a.b.tl, sq.n - t0);
        const int row = 32 * w + c, tok = row * a.hinv >> 16, hq = it.part * a.hpp + row - tok * a.hpp;
        const bool row_ok = tok < tb && hq < a.G;
        const int pos = row_ok ? sq.p0 + t0 + tok : -1;              /* keys pos_lo .. pos */
        const int pos_lo = a.b.window > 0 ? max(0, pos - a.b.window + 1) : 0;
        const size_t qrow = (size_t)(sq.lo + t0 + min(tok, tb - 1));
        const int qh = it.kv * a.G + min(hq, a.G - 1);
        /* positions of the tile, and of the wavefront's rows */
        const int first = sq.p0 + t0, last = first + tb - 1;
        const int klo = a.b.window > 0 ? max(0, first - a.b.window + 1) : 0, khi = last + 1;
        const int wt0 = 32 * w * a.hinv >> 16, wt1 = min((32 * w + 31) * a.hinv >> 16, tb - 1);
        const bool active = wt0 < tb;
        const int wfirst = first + wt0, wlast = first + wt1;
        const int wklo = a.b.window > 0 ? max(0, wfirst - a.b.window + 1) : 0;
        const int wfull = a.b.window > 0 ? max(0, wlast - a.b.window + 1) : 0;
        const int j0 = (pg_unit_lo(a.b, sq, it.tile) + it.off) << a.b.ul;
        const int jend = (int)min((int64_t)j0 + ((int64_t)it.cnt << a.b.ul), (int64_t)khi);
        const int steps = jend > j0 ? (jend - j0 + KT - 1) / KT : 0;
        const int *ids = a.pages + (size_t)s * a.b.max_pages;
        const int pmask = (1 << a.b.plog) - 1;
        const uint8_t *kb = a.k + (size_t)it.kv * a.head_bytes;
        const uint8_t *vb = a.v + (size_t)it.kv * a.head_bytes;

        /* ---- staging. Copy (16-bit) or chunk (f32) e of a step: its row among the wavefront's, and
           the place of its 16 bytes (32 of an f32 cache) in rows of keys and of values */
        auto chunk_e = [&](int e) { return min(lane + 64 * e, P::CHUNKS - 1); };
        auto row_e = [&](int e) { return F32 ? chunk_e(e) / (HD / 8) : e * P::RPE + lane / CPR; };
        auto kcol = [&](int e) {
            return F32 ? 32 * (chunk_e(e) % (HD / 8)) : 16 * min((lane % CPR) ^ P::kswz(P::RW * w + row_e(e)), HD / 8 - 1);
        };
        auto vcol = [&](int e) {
            return F32 ? 32 * (chunk_e(e) % (HD / 8)) : 16 * min((lane % CPR) ^ P::vswz(P::RW * w + row_e(e)), HD / 8 - 1);
        };
        /* A key that no row sees stands for one that does (its score is masked; should its value be no
           number, that is noted below). Where a wavefront's rows lie in one page (`flat`), its id is
           one number and the rows' places in it are the same in every step. */
        const bool flat = (1 << a.b.plog) >= P::RW && (uint64_t)a.slot_units << a.ush < (uint64_t)1 << 26;
        auto key_of = [&](int n) {
            return max(min(max(j0 + KT * n + P::RW * w + (flat ? 0 : lane % P::RW), klo), khi - 1), 0);
        };
        auto load_id = [&](int n) { return ids[key_of(n) >> a.b.plog]; };
        uint32_t koff[E], voff[E];
        {
            const uint32_t slot_bytes = a.slot_units << a.ush;
#pragma unroll
            for (int e = 0; e < E; e++) {
                koff[e] = row_e(e) * slot_bytes + kcol(e);
                voff[e] = row_e(e) * slot_bytes + vcol(e);
            }
        }
        /* put(e, key's base, its offset, value's base, its offset) for the wavefront's rows of step n */
        auto stage = [&](int n, int id, auto put) __attribute__((always_inline)) {
            const int one = __builtin_amdgcn_readfirstlane(id);
            if (flat && (uint32_t)one < (uint32_t)a.n_pages) {
                const int j = j0 + KT * n + P::RW * w;
                const uint64_t off = (uint64_t)((uint32_t)one * a.page_units + (uint32_t)(j & pmask) * a.slot_units) << a.ush;
#pragma unroll
                for (int e = 0; e < E; e++) put(e, kb + off, koff[e], vb + off, voff[e]);
                return;
            }
            const int j = flat ? j0 + KT * n + P::RW * w + lane % P::RW : key_of(n);
            const bool miss = (uint32_t)id >= (uint32_t)a.n_pages;       /* the key NaN, and its scores */
            if (__any(miss) && lane == 0 && khi > 0) *pg_late_args()->stat = 1;    /* no key: no page is needed */
            const uint32_t ro = miss ? PG_BAD_ROW : (uint32_t)id * a.page_units + (uint32_t)(j & pmask) * a.slot_units;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t r = __shfl(ro, row_e(e));
                put(e, nullptr, pg_row_ptr(kb, r, a.ush, a.blank, true) + kcol(e), nullptr,
                    pg_row_ptr(vb, r, a.ush, a.blank, false) + vcol(e));
            }
        };
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8 *)lds;
        auto copy = [&](int n, int id, int buf) __attribute__((always_inline)) {
            const uint32_t to = lds0 + buf * P::BUF + w * E * 1024;
            stage(n, id, [&](int e, const uint8_t *kp, auto ko, const uint8_t *vp, auto vo) __attribute__((always_inline)) {
                if constexpr (sizeof(ko) == 4) {
                    lds_dma16(kp, ko, to + e * 1024);
                    lds_dma16(vp, vo, to + e * 1024 + P::PLANE);
                } else {
                    pg_dma16(ko, to + e * 1024);
                    pg_dma16(vo, to + e * 1024 + P::PLANE);
                }
            });
        };
        constexpr int EF = F32 ? E : 1;
        u32x4_t kraw[EF][2], vraw[EF][2];
        auto fetch = [&](int n, int id) __attribute__((always_inline)) {
            stage(n, id, [&](int e, const uint8_t *kp, auto ko, const uint8_t *vp, auto vo) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    kraw[e][i] = pg_load<u32x4_t>((uint64_t)kp + ko + 16 * i);
                    vraw[e][i] = pg_load<u32x4_t>((uint64_t)vp + vo + 16 * i);
                }
            });
        };
        auto split_to = [&](uint8_t *dst, const u32x4_t (&x)[2]) __attribute__((always_inline)) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f16pair2 p = split_f16x2(__uint_as_float(x[i >> 1][2 * (i & 1)]),
                                               __uint_as_float(x[i >> 1][2 * (i & 1) + 1]));
                hi[i] = p.hi;
                lo[i] = p.lo;
            }
            *(uint4 *)dst = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *(uint4 *)(dst + P::PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        };
        auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < EF; e++) {
                /* past the last chunk: the last one again, the same bytes */
                const int r = P::RW * w + row_e(e), ch = chunk_e(e) % (HD / 8);
                uint8_t *b = lds + buf * P::BUF + r * RB;
                split_to(b + ((ch ^ P::kswz(r)) << 4), kraw[e]);
                split_to(b + NC * P::PLANE + ((ch ^ P::vswz(r)) << 4), vraw[e]);
            }
        };
        /* whether step n lies across the border of what the tile's rows see */
        auto crosses = [&](int n) { return j0 + KT * n < (a.b.window > 0 ? max(0, last - a.b.window + 1) : 0) || j0 + KT * n + KT - 1 > first; };
        /* Infinities and NaNs among the values of a step of which some row does not see some key: a weight
           of zero would not keep them out of that row's sums. They are taken out of LDS by the
           wavefronts that staged them, and added where they are seen (below). */
        auto note = [&](int n, int buf, int turn) __attribute__((always_inline)) {
            if (!crosses(n)) return;
            uint32_t any = 0;
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < EF; e++) {
                    /* what no row sees has no say in the scale either */
                    const int j = j0 + KT * n + P::RW * w + row_e(e);
                    const uint32_t seen = j >= klo && j < khi ? ~0u : 0u;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        kraw[e][i >> 2][i & 3] &= seen;
                        vraw[e][i >> 2][i & 3] &= seen;
                        any |= pg_wild<CPG_T_F32>(vraw[e][i >> 2][i & 3]);
                        vraw[e][i >> 2][i & 3] = pg_tame<CPG_T_F32>(vraw[e][i >> 2][i & 3]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    uint4 *p = (uint4 *)(lds + buf * P::BUF + P::PLANE + (w * E + e) * 1024 + 16 * lane);
                    const uint4 x = *p;
                    any |= pg_wild<CT>(x.x) | pg_wild<CT>(x.y) | pg_wild<CT>(x.z) | pg_wild<CT>(x.w);
                    *p = make_uint4(pg_tame<CT>(x.x), pg_tame<CT>(x.y), pg_tame<CT>(x.z), pg_tame<CT>(x.w));
                }
            }
            if (__any(any != 0)) wild_s[turn & 3] = 1;
        };

        /* f32 caches: the wavefront's rows by powers of two 2^-ek and 2^-ev that bring their largest key
           and value element within f16's range and its precision, 2^-3 .. 2^15: where it is within,
           none. The scores take ek back, and the sums of values ev. */
        auto scale = [&](int turn) __attribute__((always_inline)) {
            float tk = 0.0f, tv = 0.0f;
#pragma unroll
            for (int e = 0; e < EF; e++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    tk = fmaxf(tk, fabsf(__uint_as_float(kraw[e][i >> 2][i & 3])));
                    tv = fmaxf(tv, fabsf(__uint_as_float(vraw[e][i >> 2][i & 3])));
                }
            const bool kin = __any(tk >= 0.125f) && !__any(tk > 32768.0f);
            const bool vin = __any(tv >= 0.125f) && !__any(tv > 32768.0f);
            int ek = 0, ev = 0;
            if (!kin || !vin) {
#pragma nounroll
                for (int o = 1; o < 64; o <<= 1) {
                    tk = fmaxf(tk, __shfl_xor(tk, o));
                    tv = fmaxf(tv, __shfl_xor(tv, o));
                }
                if (!kin && tk > 0.0f && tk < INFINITY) ek = __builtin_amdgcn_frexp_expf(tk) - 8;
                if (!vin && tv < INFINITY) ev = tv > 0.0f ? __builtin_amdgcn_frexp_expf(tv) - 8 : PG_NO_SCALE;
#pragma unroll
                for (int e = 0; e < EF; e++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        kraw[e][i >> 2][i & 3] = __float_as_uint(ldexpf(__uint_as_float(kraw[e][i >> 2][i & 3]), -ek));
                        vraw[e][i >> 2][i & 3] = __float_as_uint(ldexpf(__uint_as_float(vraw[e][i >> 2][i & 3]), -ev));
                    }
            }
            if (lane == 0) scale_s[turn & 3][w] = (ek & 0xFFFF) | (int)((uint32_t)ev << 16);
        };

        f32x16_t o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = f32x16_t{};
        int Ev = PG_NO_SCALE;                    /* f32 caches: o counts in 2^Ev */
        float M = -INFINITY, l = 0.0f;           /* what the weights refer to, in log2; -inf: nothing yet */

        int id = load_id(0);
        /* the first step into buffer 0, and the queries behind its loads */
        if constexpr (F32) fetch(0, id);
        else copy(0, id, 0);
        id = load_id(1);
        /* ---- the queries */
        uint4 qf[NQ][NS];
        float cs = a.scale2;
        {
            const uint8_t *qp = (const uint8_t *)a.q + (qrow * a.ldq + (size_t)qh * HD + 8 * h) * (AT == CPG_T_F32 ? 4 : 2);
            if constexpr (AT != CPG_T_F32) {
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const uint4 x = *(const uint4 *)(qp + 32 * i);
                    qf[0][i] = row_ok ? x : make_uint4(0, 0, 0, 0);
                }
            } else {
                float top = 0.0f;
                float4 x[NS][2];
#pragma unroll
                for (int i = 0; i < NS; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        x[i][j] = *(const float4 *)(qp + 64 * i + 16 * j);
                        top = fmaxf(fmaxf(fmaxf(top, fabsf(x[i][j].x)), fmaxf(fabsf(x[i][j].y), fabsf(x[i][j].z))), fabsf(x[i][j].w));
                    }
                top = pg_half_max(top);
                /* the row by 2^-ex, its largest element in [0.5, 1), and the scores by 2^ex */
                const int ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
                cs = ldexpf(cs, ex);
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    uint32_t wd[4][NQ];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        pg_pieces2<OT, NQ>(ldexpf(x[i][j].x, -ex), ldexpf(x[i][j].y, -ex), wd[2 * j]);
                        pg_pieces2<OT, NQ>(ldexpf(x[i][j].z, -ex), ldexpf(x[i][j].w, -ex), wd[2 * j + 1]);
                    }
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        qf[n][i] = row_ok ? make_uint4(wd[0][n], wd[1][n], wd[2][n], wd[3][n]) : make_uint4(0, 0, 0, 0);
                }
            }
        }
        if constexpr (F32) {
            note(0, 0, turn);
            scale(turn);
            store(0);
        } else {
            wait_vm_lgkm<0>();
            note(0, 0, turn);
        }
        __syncthreads();

        /* where the lane reads a buffer: keys row c, chunk 2 i + h; values (transposing) */
        const int tr = lane & 15, trow = 4 * h + (tr >> 2);
        const int kread = c * RB + ((h ^ P::kswz(c)) << 4);
        const int vread = NC * P::PLANE + trow * RB +
                          (((2 * (lane >> 4 & 1) + (tr >> 1 & 1)) ^ P::vswz(trow)) << 4) + 8 * (tr & 1);
        for (int n = 0; n < steps; n++) {
            const int jb = j0 + KT * n, buf = n & 1;
            const bool more = n + 1 < steps;
            if (more) {
                if constexpr (F32) fetch(n + 1, id);
                else copy(n + 1, id, buf ^ 1);
                id = load_id(n + 2);
            }
            if (active && jb <= wlast && jb + KT > wklo) {
                const uint8_t *base = lds + buf * P::BUF;
                /* scores: st[b][i] of key jb + 32 b + 8 (i / 4) + 4 h + i % 4 */
                /* The matrix phases have the priority over the other workgroup's vector phases (2 %). The
                   order of reads and products is fenced throughout: left alone the compiler reads an
                   operand and waits for it at once. Operand t of the keys: block t % NB, elements
                   16 (t / NB) ..; PD of them are read ahead of the products. */
                __builtin_amdgcn_s_setprio(1);
                f32x16_t st[NB];
                {
                    constexpr int NT = NS * NB, PD = NQ > 1 ? 2 : 4;
                    uint4 kf[PD][NC];
                    auto read = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                        for (int p = 0; p < NC; p++)
                            kf[t % PD][p] = *(const uint4 *)(base + p * P::PLANE + 32 * (t % NB) * RB + (kread ^ (t / NB << 5)));
                    };
#pragma unroll
                    for (int t = 0; t < PD; t++) read(t);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const uint4 (&k)[NC] = kf[t % PD];
                        f32x16_t &x = st[t % NB];
                        if (t < NB) x = f32x16_t{};
                        if constexpr (F32) x = pg_mfma32<OT>(k[1], qf[0][t / NB], x);
#pragma unroll
                        for (int p = NQ - 1; p >= 0; p--) x = pg_mfma32<OT>(k[0], qf[p][t / NB], x);
                        if (t + PD < NT) read(t + PD);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                float vsc[4];                    /* of the weights of each wavefront's keys: 2^(ev - Ev) */
                if constexpr (F32) {
                    int ev[4], any = Ev, top = Ev;
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int x = __builtin_amdgcn_readfirstlane(scale_s[turn & 3][g]);
                        any |= x;
                        ev[g] = x >> 16;
                        top = max(top, ev[g]);
                    }
                    if (any) {
#pragma unroll
                        for (int i = 0; i < 16; i++) st[0][i] = ldexpf(st[0][i], (int16_t)scale_s[turn & 3][i >> 2]);
#pragma unroll
                        for (int d = 0; d < ND; d++)
#pragma unroll
                            for (int i = 0; i < 16; i++) o[d][i] = ldexpf(o[d][i], Ev - top);
                    }
                    Ev = top;
#pragma unroll
                    for (int g = 0; g < 4; g++) vsc[g] = __int_as_float((127 + max(ev[g] - top, -127)) << 23);
                }
                const bool edge = jb < wfull || jb + KT - 1 > wfirst;
                if (edge)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int j = jb + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3);
                            st[b][i] = j <= pos && j >= pos_lo ? st[b][i] : -INFINITY;
                        }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) mx = fmaxf(mx, st[b][i]);
                mx = cs * pg_half_max(mx);
                const bool renew = mx > M + PG_SLACK;
                if (__any(renew)) {              /* each row by itself: not by what others see */
                    const float Mn = renew ? mx : M;
                    const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
                    M = Mn;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[d][i] *= f;
                }
                const float off = P::LIFT - (M == -INFINITY ? 0.0f : M);
                const bool wild = crosses(n) && wild_s[turn & 3] != 0;
                /* The weights of 16 keys are an operand, computed among the products of the 16 before.
                   Operand t of the values: keys 16 (t / ND) .., elements 32 (t % ND) .. */
                {
                    constexpr int NT = 2 * NB * ND, PD = NQ > 1 ? 2 : 4;
                    uint4 vf[PD][NC], pf[2][NQ];
                    auto read = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                        for (int p = 0; p < NC; p++) {
                            const uint8_t *vp = base + p * P::PLANE + 16 * (t / ND) * RB + (vread ^ (t % ND << 6));
                            const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) s16x4_t *)(lds_u8 *)vp));
                            const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) s16x4_t *)(lds_u8 *)(vp + 8 * RB)));
                            vf[t % PD][p] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                        }
                    };
                    /* word i (of 4) of the weights of keys 16 k .. */
                    auto weight = [&](int k, int i) __attribute__((always_inline)) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(st[k >> 1][8 * (k & 1) + 2 * i], cs, off));
                        const float y = __builtin_amdgcn_exp2f(fmaf(st[k >> 1][8 * (k & 1) + 2 * i + 1], cs, off));
                        l += x;
                        l += y;
                        uint32_t wd[NQ];
                        if constexpr (F32) {
                            const float f = vsc[2 * (k & 1) + (i >> 1)];
                            pg_pieces2<OT, NQ>(x * f, y * f, wd);
                        } else {
                            pg_pieces2<OT, NQ>(x, y, wd);
                        }
#pragma unroll
                        for (int p = 0; p < NQ; p++) {
                            if (i == 0) pf[k & 1][p].x = wd[p];
                            if (i == 1) pf[k & 1][p].y = wd[p];
                            if (i == 2) pf[k & 1][p].z = wd[p];
                            if (i == 3) pf[k & 1][p].w = wd[p];
                        }
                    };
#pragma unroll
                    for (int t = 0; t < PD; t++) read(t);
#pragma unroll
                    for (int i = 0; i < 4; i++) weight(0, i);
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_setprio(1);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const int k = t / ND, d = t % ND;
                        const uint4 (&v)[NC] = vf[t % PD];
                        if constexpr (F32) o[d] = pg_mfma32<OT>(v[1], pf[k & 1][0], o[d]);
#pragma unroll
                        for (int p = NQ - 1; p >= 0; p--) o[d] = pg_mfma32<OT>(v[0], pf[k & 1][p], o[d]);
                        if (t + PD < NT) read(t + PD);
                        if (k + 1 < 2 * NB)
#pragma unroll
                            for (int i = 4 * d / ND; i < 4 * (d + 1) / ND; i++) weight(k + 1, i);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                if (wild) {
                    /* The rest, for the rows that see it (their weights taken as above zero), from the
                       pages again: in memory, in the place that the item's piece may take when it is
                       done, so that this seldom path holds no registers */
                    const pg_args *la = pg_late_args();
                    uint8_t *mine = (uint8_t *)la->pacc +
                                    ((size_t)2 * me + (me == pg_owner(it.first, sh.U, W))) * P::SLOT +
                                    (size_t)w * (ND * 4096);
                    /* stored and loaded as pieces are, since another XCD may write there later */
#pragma unroll
                    for (int i = 0; i < 4 * ND; i++)
                        pg_st_agent16(mine, 1024 * i + 16 * lane,
                                      make_float4(o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1],
                                                  o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]));
                    mem_done();
#pragma nounroll
                    for (int i = 0; i < 4 * ND; i++) {
                        const v4i_t r = ld_agent16(mine, 1024 * i + 16 * lane);
                        float x[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) x[k] = __int_as_float(r[k]);
#pragma nounroll
                        for (int j = max(jb, klo); j < min(jb + KT, khi); j++) {
                            const uint32_t vid = (uint32_t)ids[j >> a.b.plog];
                            if (vid >= (uint32_t)a.n_pages || j > pos || j < pos_lo) continue;
                            const uint64_t vp = (uint64_t)vb + ((uint64_t)(vid * a.page_units + (uint32_t)(j & pmask) * a.slot_units) << a.ush);
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int e = 8 * i + 4 * h + k;
                                float y;
                                if constexpr (F32) y = pg_load<float>(vp + 4 * e);
                                else y = pg_unpack2<CT>(pg_load<uint16_t>(vp + 2 * e)).x;
                                x[k] += fabsf(y) < INFINITY ? 0.0f : y;
                            }
                        }
                        pg_st_agent16(mine, 1024 * i + 16 * lane, make_float4(x[0], x[1], x[2], x[3]));
                    }
                    mem_done();
#pragma unroll
                    for (int i = 0; i < 4 * ND; i++) {
                        const v4i_t x = ld_agent16(mine, 1024 * i + 16 * lane);
#pragma unroll
                        for (int k = 0; k < 4; k++) o[i >> 2][4 * (i & 3) + k] = __int_as_float(x[k]);
                    }
                    /* waited for here: where the paths join it would be in every step, and for the
                       copies in flight too */
#pragma unroll
                    for (int d = 0; d < ND; d++) asm volatile("" : "+v"(o[d]));
                }
            }
            if (more) {
                if constexpr (F32) {
                    note(n + 1, buf ^ 1, turn + 1);
                    scale(turn + 1);
                    store(buf ^ 1);
                } else {
                    wait_vm_lgkm<0>();
                    note(n + 1, buf ^ 1, turn + 1);
                }
            }
            __syncthreads();
            if (tid == 0) wild_s[turn & 3] = 0;  /* noted again four steps on, with barriers between */
            turn++;
        }
        if (steps == 0) {                        /* the step that was staged for nothing */
            if (tid == 0) wild_s[turn & 3] = 0;
            turn++;
        }
        l = pg_half_sum(l);
        if (F32 && Ev != 0)
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] = ldexpf(o[d][i], Ev);

        /* ---- the rows: written, or left as a piece. A lane's elements 8 e + 4 h .. + 3 of its row */
        const pg_args *late = pg_late_args();
        const bool whole = it.cnt == it.all;
        const int wf = pg_owner(it.first, sh.U, W);
        auto place = [&](int x) { return (size_t)2 * x + (x == wf); };
        auto finish = [&](float top, float L) __attribute__((always_inline)) {
            if (!row_ok) return;
            const float nan = __int_as_float(0x7fc00000), inv = __fdiv_rn(1.0f, L);
            float e = (top + __builtin_amdgcn_logf(ldexpf(L, -(int)P::LIFT))) * 0.69314718055994531f;
            const bool none = sq.p0 + t0 + tok < 0;
            if (sq.bad) e = nan;
            else if (none) e = -INFINITY;
            if (late->lse && h == 0) late->lse[qrow * late->H + qh] = e;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    float4 y = make_float4(o[d][4 * b] * inv, o[d][4 * b + 1] * inv, o[d][4 * b + 2] * inv, o[d][4 * b + 3] * inv);
                    if (sq.bad) y = make_float4(nan, nan, nan, nan);
                    else if (none) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    pg_put4<AT>(late->out, qrow * late->ldo + (size_t)qh * HD + 32 * d + 8 * b + 4 * h, y);
                }
        };
        if (whole) {
            if (active) finish(M, l);
            continue;
        }
        /* a piece: per slot the four wavefronts' blocks of 4 ND x 64 lanes x 16 bytes */
        auto put = [&](size_t slot, float top, float L) __attribute__((always_inline)) {
            uint8_t *pa = (uint8_t *)late->pacc + slot * P::SLOT + (size_t)w * (ND * 4096);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int b = 0; b < 4; b++)
                    pg_st_agent16(pa, (4 * d + b) * 1024 + 16 * lane,
                                  make_float4(o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]));
            if (h == 0) {
                float *pm = (float *)(late->pml + slot * PG_MANY_ROWS + 32 * w + c);
                st_agent(pm, top);
                st_agent(pm + 1, L);
            }
        };
        /* pieces x0, x0 + step, ... (n of them) into o; returns (M, l) */
        auto merge = [&](int x0, int n, int step, float &top, float &L) __attribute__((always_inline)) {
            top = -INFINITY;
            L = 0.0f;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] = f32x16_t{};
#pragma nounroll
            for (int k = 0; k < n; k++) {
                const size_t slot = place(x0 + k * step);
                const uint8_t *pa = (const uint8_t *)late->pacc + slot * P::SLOT + (size_t)w * (ND * 4096);
                const unsigned long long mb = ld_agent((const unsigned long long *)(late->pml + slot * PG_MANY_ROWS + 32 * w + c));
                v4i_t y[ND][4];
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++) y[d][b] = ld_agent16(pa, (4 * d + b) * 1024 + 16 * lane);
                const float pm = __uint_as_float((uint32_t)mb), pl = __uint_as_float((uint32_t)(mb >> 32));
                const float t2 = fmaxf(top, pm);
                const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t2);
                const float e = pm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm - t2);
                top = t2;
                L = fmaf(e, pl, L * f);
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] = fmaf(e, __int_as_float(y[d][i >> 2][i & 3]), o[d][i] * f);
            }
        };
        if (active) put(place(me), M, l);
        constexpr int MG = 8;                    /* as in k_paged_few, in groups of eight */
        const int wl = pg_owner(it.first + it.all - 1, sh.U, W);
        const int gx = wf + (me - wf) / MG * MG, groups = (wl - wf) / MG + 1;
        float top, L;
        bool mine = true;
        if (groups > 1) {
            const int cnt = min(MG, wl - gx + 1);
            mine = last_arriver(&late->ctr[2 * gx + (gx == wf)], cnt - 1, &flag);
            if (mine && active) {
                merge(gx, cnt, 1, top, L);
                put(place(gx), top, L);          /* each lane what it has read itself: but for (M, l) */
            }
        }
        if (mine && last_arriver(&late->ctr[2 * W + wf], groups > 1 ? groups - 1 : wl - wf, &flag) && active) {
            merge(wf, groups > 1 ? groups : wl - wf + 1, groups > 1 ? MG : 1, top, L);
            finish(top, L);
        }
        __syncthreads();
    }
}

template <int CT, int AT, int HD> static int launch_one(const pg_args &a, int grid) {
    const int bytes = 2 * pg_many_t<CT, AT, HD>::BUF;
    CPG_HIP(hipFuncSetAttribute((const void *)k_paged_many<CT, AT, HD>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    hipLaunchKernelGGL((k_paged_many<CT, AT, HD>), dim3(grid), dim3(256), bytes, g_cpg.stream, a);
    CPG_LAUNCH_CHECK("k_paged_many");
    return 0;
}

template <int CT, int AT> static int launch(const pg_args &a, int HD, int grid) {
    return HD == 64    ? launch_one<CT, AT, 64>(a, grid)
           : HD == 96  ? launch_one<CT, AT, 96>(a, grid)
           : HD == 128 ? launch_one<CT, AT, 128>(a, grid)
           : HD == 192 ? launch_one<CT, AT, 192>(a, grid)
                       : launch_one<CT, AT, 256>(a, grid);
}

int pg_launch_many(const pg_args &a, int type, int cache, int HD, int grid) {
    if (type == CPG_T_F16) return launch<CPG_T_F16, CPG_T_F16>(a, HD, grid);
    if (type == CPG_T_BF16) return launch<CPG_T_BF16, CPG_T_BF16>(a, HD, grid);
    if (cache == CPG_T_F32) return launch<CPG_T_F32, CPG_T_F32>(a, HD, grid);
    if (cache == CPG_T_F16) return launch<CPG_T_F16, CPG_T_F32>(a, HD, grid);
    return launch<CPG_T_BF16, CPG_T_F32>(a, HD, grid);
}
