/* paged_few.hip — attention of few new tokens per sequence over the paged cache: decode steps.
 *
 * s_j = scale q . k_j, p_j = exp(s_j - M), out = sum p_j v_j / sum p_j with the running maximum M.
 * A tile is the (up to 16) query rows of one sequence that share a kv head: TB tokens times the
 * kv head's query heads. The keys stream through the four wavefronts of a workgroup, KT a time each,
 * straight from the pages into the registers that the matrix instructions read, with no staging
 * in LDS: the next keys are loaded once the scores are taken, the next values once they are summed,
 * and with the waves of a CU in turn that keeps enough bytes in flight.
 *
 * Layouts. S^T = K Q^T: a lane brings the key row l % 16 and the queries' column l % 16, and the sum
 * over the head may run in any order that both sides share, so a lane's pieces of a key row are 16
 * consecutive bytes. In the product S^T a lane holds one query (l % 16) and the keys 4 (l / 16) + i.
 * O^T = V^T P^T sums over keys, in any order: the one that S^T is held in makes P an operand where it
 * stands, one query to a lane, as the maximum and the sum of the softmax want it. V^T's rows are
 * the head's elements, and which element is row r of which product is free too: a lane loads HD /
 * 16 consecutive elements of the four (eight) keys whose weights it holds, and element j of them
 * belongs to product j. For 16-bit caches the pairs of keys are packed by byte permutes.
 *
 * f32 caches run on the f32 matrix instruction (16x16x4, 157 TFLOP/s): nothing is rounded, and
 * 8 FLOP for each byte read need 64 TFLOP/s at 8 TB/s. 16-bit caches run on 16x16x32 (2.5
 * PFLOP/s); f32 queries and weights go in as two f16 pieces (a row of queries scaled by a power of
 * two first, the weights lifted by 2^12, so that f16's exponents reach) or three bf16 pieces (which
 * have fp32's exponents), 16-bit activations as one piece, the weights rounded once.
 *
 * What bounds it: the bytes of the visible keys and values. 96 sequences of 500 - 8000 tokens, bf16,
 * 8 kv heads of 128: 1.08 GB in 200 us, 5.4 TB/s, where a plain read of 1 - 2 GB reaches 6.2; one
 * sequence of 32768 over a bf16 cache: 67 MB in 21.6 us. For short contexts it is the chain of one
 * workgroup, of the 10.2 us for one token over 200: launch 2, scan 0.7, item 1.0, page ids to
 * keys 1.6, steps 1.9, wavefronts' merge 1.0, arrival 1.0, workgroups' merge 2.
 */
#include "cpg_paged.h"

template <int CT, int AT> struct pg_few_t {
    /* pieces of queries and of weights */
    static constexpr int NP = CT == CPG_T_F32 || AT != CPG_T_F32 ? 1 : CT == CPG_T_F16 ? 2 : 3;
    static constexpr int KT = CT == CPG_T_F32 ? 16 : 32;        /* keys per wavefront and step */
    /* f16 weights are lifted by 2^12: a weight of 2^-26 is then still a normal number */
    static constexpr float LIFT = CT == CPG_T_F16 ? 12.0f : 0.0f;
};

/* 16-bit operands: eight elements in four words */
template <int CT>
__device__ static inline f32x4_t pg_mfma16(uint4 a, uint4 b, f32x4_t c) {
    if constexpr (CT == CPG_T_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                      __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

/* the registers of one step: KT key rows and value rows */
template <int CT, int HD> struct pg_buf {
    static constexpr bool F32 = CT == CPG_T_F32;
    static constexpr int DPL = HD / 16;          /* value elements of a row in a lane */
    static constexpr int NK = F32 ? HD / 16 : 2 * (HD / 32);
    static constexpr int NR = F32 ? 4 : 8;       /* value rows in a lane */
    static constexpr int NW = F32 ? DPL : DPL / 2;
    uint4 k[NK];
    uint32_t v[NR][NW];
};

template <int NW> __device__ static inline void pg_load_words(uint64_t p, uint32_t (&w)[NW]) {
    /* the lane's part of a row starts on a multiple of 4 NW bytes of it */
    if constexpr (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 4; i++) {
            const u32x4_t u = pg_load<u32x4_t>(p + 16 * i);
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
    } else if constexpr (NW % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 2; i++) {
            const u32x2_t u = pg_load<u32x2_t>(p + 8 * i);
            w[2 * i] = u.x; w[2 * i + 1] = u.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NW; i++) w[i] = pg_load<uint32_t>(p + 4 * i);
    }
}

/* grid W workgroups of 256 threads, each with its share of the units (cpg_paged.h) */
template <int CT, int AT, int HD>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void k_paged_few(const pg_args a) {
    typedef pg_few_t<CT, AT> P;
    typedef pg_buf<CT, HD> buf;
    constexpr bool F32 = CT == CPG_T_F32;
    constexpr int KT = P::KT, NP = P::NP, DPL = buf::DPL, NR = buf::NR, NW = buf::NW;
    constexpr int EB = F32 ? 4 : 2, NS = F32 ? HD / 16 : HD / 32, LD = HD + 4;
    __shared__ __align__(16) float o_s[4][16][LD];
    __shared__ float m_s[4][16], l_s[4][16];
    __shared__ int flag;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    pg_start at;
    const pg_share sh = pg_find_share(a.b, at, a.stat);
    const int W = sh.W, me = sh.w;
    int s = at.s;
    uint32_t rem = at.rem;
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
        /* the thread's number is made opaque, here and behind the loop: what follows from it would
           else be computed ahead of the walk and held, or spilled, over everything */
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int c = lane & 15, g = lane >> 4;
        /* the lane's query: row c of the tile */
        const int t0 = it.tile << a.b.tl, tb = min(1 << a.b.tl, sq.n - t0);
        const int tok = c * a.hinv >> 16, hq = it.part * a.hpp + c - tok * a.hpp;
        const bool row_ok = tok < tb && hq < a.G;
        const int pos = row_ok ? sq.p0 + t0 + tok : -1;           /* keys pos_lo .. pos */
        const int pos_lo = a.b.window > 0 ? max(0, pos - a.b.window + 1) : 0;
        const size_t qrow = (size_t)(sq.lo + t0 + min(tok, tb - 1));
        const int qh = it.kv * a.G + min(hq, a.G - 1);
        const int first = sq.p0 + t0, last = first + tb - 1;      /* positions of the tile */
        const int klo = a.b.window > 0 ? max(0, first - a.b.window + 1) : 0, khi = last + 1;
        const int full_lo = a.b.window > 0 ? max(0, last - a.b.window + 1) : 0;
        /* the units' keys */
        const int j0 = (pg_unit_lo(a.b, sq, it.tile) + it.off) << a.b.ul;
        const int jend = (int)min((int64_t)j0 + ((int64_t)it.cnt << a.b.ul), (int64_t)khi);
        f32x4_t o[DPL];
#pragma unroll
        for (int j = 0; j < DPL; j++) o[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, M = 0.0f, l = 0.0f;
        /* no branch around the loads, also where the tile sees no key: what its two sides bring would
           be joined in registers of their own */
        const int *ids = a.pages + (size_t)s * a.b.max_pages;
        const int pmask = (1 << a.b.plog) - 1;
        const uint8_t *kb = a.k + (size_t)it.kv * a.head_bytes;
        const uint8_t *vb = a.v + (size_t)it.kv * a.head_bytes;
        /* step n of this wavefront: keys jw + 4 KT n .. + KT - 1 */
        const int jw = j0 + KT * w;
        const int steps = jend > jw ? (jend - jw + 4 * KT - 1) / (4 * KT) : 0;
        /* the page of the step's key lane % KT (of a key that no row sees: any that one does) */
        auto page_of = [&](int n) __attribute__((always_inline)) {
            const int j = jw + 4 * KT * n + lane % KT;
            return ids[max(min(max(j, klo), khi - 1), 0) >> a.b.plog];
        };
        /* its row's offset. A key that no row sees reads zeros; a page id that is none makes the
           key NaN, and with it every score of it */
        auto row_of = [&](int n, int id) __attribute__((always_inline)) {
            const int j = jw + 4 * KT * n + lane % KT;
            const bool out = j < klo || j >= khi, miss = (uint32_t)id >= (uint32_t)a.n_pages;
            if (__any(miss && !out) && lane == 0) *pg_late_args()->stat = 1;
            const uint32_t r = (uint32_t)id * a.page_units + (uint32_t)(j & pmask) * a.slot_units;
            return out ? PG_NO_ROW : miss ? PG_BAD_ROW : r;
        };
        auto row_ptr = [&](const uint8_t *base, uint32_t r, bool key) __attribute__((always_inline)) {
            return pg_row_ptr(base, r, a.ush, a.blank, key);
        };
        buf b;
        auto load_k = [&](uint32_t ro) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < KT / 16; t++) {
                const uint64_t p = row_ptr(kb, __shfl(ro, 16 * t + c), true) + 16 * g;
#pragma unroll
                for (int i = 0; i < NS; i++) b.k[t * NS + i] = __builtin_bit_cast(uint4, pg_load<u32x4_t>(p + 64 * i));
            }
        };
        auto load_v = [&](uint32_t ro) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < NR; r++)
                pg_load_words<NW>(row_ptr(vb, __shfl(ro, 16 * (r >> 2) + 4 * g + (r & 3)), false) + c * DPL * EB, b.v[r]);
        };
        int id = page_of(0);
        /* ---- the queries, in the order the key rows are loaded in; issued between the first
           page ids and the first keys, and put into pieces while those fly */
        constexpr int QN = F32 || AT != CPG_T_F32 ? NS : 2 * NS;
        const uint8_t *qp = (const uint8_t *)a.q +
                            (qrow * a.ldq + (size_t)qh * HD) * (AT == CPG_T_F32 ? 4 : 2) +
                            g * (QN == 2 * NS ? 32 : 16);
        uint4 qraw[QN];
#pragma unroll
        for (int i = 0; i < QN; i++)
            qraw[i] = *(const uint4 *)(qp + (QN == NS ? 64 * i : 128 * (i >> 1) + 16 * (i & 1)));
        __builtin_amdgcn_sched_barrier(0);
        uint32_t ro = row_of(0, id);
        id = page_of(1);                     /* ahead of the loads, so that it is there with them */
        load_k(ro);
        load_v(ro);
        __builtin_amdgcn_sched_barrier(0);
        uint4 qf[NP][NS];
        float cs = a.scale2;
        if constexpr (QN == NS) {
#pragma unroll
            for (int i = 0; i < NS; i++) qf[0][i] = row_ok ? qraw[i] : make_uint4(0, 0, 0, 0);
        } else {
            int ex = 0;
            if constexpr (CT == CPG_T_F16) {     /* bf16 has fp32's exponents */
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < QN; i++) {
                    const uint32_t x[4] = {qraw[i].x, qraw[i].y, qraw[i].z, qraw[i].w};
#pragma unroll
                    for (int j = 0; j < 4; j++) top = fmaxf(top, fabsf(__uint_as_float(x[j])));
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                /* the row by 2^-ex, its largest element in [0.5, 1), and the scores by 2^ex */
                ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
                cs = ldexpf(cs, ex);
            }
            auto scaled = [&](uint32_t x) {
                return CT == CPG_T_F16 ? ldexpf(__uint_as_float(x), -ex) : __uint_as_float(x);
            };
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint4 r0 = qraw[2 * i], r1 = qraw[2 * i + 1];
                const uint32_t x[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
                uint32_t wd[4][NP];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    pg_pieces2<CT, NP>(scaled(x[2 * j]), scaled(x[2 * j + 1]), wd[j]);
#pragma unroll
                for (int n = 0; n < NP; n++)
                    qf[n][i] = row_ok ? make_uint4(wd[0][n], wd[1][n], wd[2][n], wd[3][n]) : make_uint4(0, 0, 0, 0);
            }
        }
        for (int n = 0; n < steps; n++) {
            const int jb = jw + 4 * KT * n;
            /* scores: st[t][i] of key jb + 16 t + 4 g + i */
            f32x4_t st[KT / 16];
#pragma unroll
            for (int t = 0; t < KT / 16; t++) {
                st[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const uint4 kf = b.k[t * NS + i];
                    if constexpr (F32) {
                        const uint4 qv = qf[0][i];
                        st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf.x), __uint_as_float(qv.x), st[t], 0, 0, 0);
                        st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf.y), __uint_as_float(qv.y), st[t], 0, 0, 0);
                        st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf.z), __uint_as_float(qv.z), st[t], 0, 0, 0);
                        st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf.w), __uint_as_float(qv.w), st[t], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int p = NP - 1; p >= 0; p--) st[t] = pg_mfma16<CT>(kf, qf[p][i], st[t]);
                    }
                }
            }
            /* the key registers are free: without the fence the loads would be moved ahead of
               the scores, into registers of their own */
            __builtin_amdgcn_sched_barrier(0);
            ro = row_of(n + 1, id);          /* past the last step: zeros */
            id = page_of(n + 2);
            load_k(ro);
            __builtin_amdgcn_sched_barrier(0);
            const bool edge = jb < full_lo || jb + KT - 1 > first;
            if (edge)                        /* some row does not see some key */
#pragma unroll
                for (int t = 0; t < KT / 16; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = jb + 16 * t + 4 * g + i;
                        st[t][i] = j <= pos && j >= pos_lo ? st[t][i] : -INFINITY;
                    }
            float mn = m;
#pragma unroll
            for (int t = 0; t < KT / 16; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) mn = fmaxf(mn, st[t][i]);
            mn = fmaxf(mn, __shfl_xor(mn, 16));
            mn = fmaxf(mn, __shfl_xor(mn, 32));
            if (__any(mn > m)) {
                const float Mn = mn == -INFINITY ? 0.0f : cs * mn;
                const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
                m = mn;
                M = Mn;
                l *= f;
#pragma unroll
                for (int j = 0; j < DPL; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[j][i] *= f;
            }
            float p[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(st[r >> 2][r & 3], cs, P::LIFT - M));
                l += p[r];
            }
            /* values that are no numbers in a step of which some row does not see some key: a
               weight of zero would not keep them out, so the tokens are taken one by one */
            bool wild = false;
            if (edge && tb > 1) {
                uint32_t any = 0;
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int i = 0; i < NW; i++) any |= pg_wild<CT>(b.v[r][i]);
                wild = __any(any != 0);
            }
            uint4 pf[NP];                    /* 16-bit caches: the weights' pieces */
            if constexpr (!F32) {
                uint32_t wd[4][NP];
#pragma unroll
                for (int r = 0; r < 4; r++) pg_pieces2<CT, NP>(p[2 * r], p[2 * r + 1], wd[r]);
#pragma unroll
                for (int n = 0; n < NP; n++) pf[n] = make_uint4(wd[0][n], wd[1][n], wd[2][n], wd[3][n]);
            }
            /* x plus element j's sum over the keys of the step that `mask` leaves */
            auto weigh = [&](int j, f32x4_t x, const uint32_t (&mask)[4]) __attribute__((always_inline)) {
                if constexpr (F32) {
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.v[r][j] & mask[r]), p[r], x, 0, 0, 0);
                } else {
                    uint32_t vw[4];          /* element j of the eight keys */
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        vw[r] = mask[r] & __builtin_amdgcn_perm(b.v[2 * r + 1][j >> 1], b.v[2 * r][j >> 1],
                                                                j & 1 ? 0x07060302u : 0x05040100u);
                    const uint4 vf = make_uint4(vw[0], vw[1], vw[2], vw[3]);
#pragma unroll
                    for (int n = NP - 1; n >= 0; n--) x = pg_mfma16<CT>(vf, pf[n], x);
                }
                return x;
            };
            if (!wild) {
                const uint32_t all[4] = {~0u, ~0u, ~0u, ~0u};
#pragma unroll
                for (int j = 0; j < DPL; j++) o[j] = weigh(j, o[j], all);
            } else {                         /* a lane's rows are one token's: taken in its turn */
#pragma nounroll
                for (int z = 0; z < tb; z++) {
                    const int ph = first + z, pl = a.b.window > 0 ? ph - a.b.window + 1 : 0;
                    auto seen = [&](int i) { return jb + i <= ph && jb + i >= pl; };
                    uint32_t mask[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (F32) {
                            mask[r] = seen(4 * g + r) ? ~0u : 0u;
                        } else {
                            const int i = 16 * (r >> 1) + 4 * g + 2 * (r & 1);
                            mask[r] = (seen(i) ? 0xFFFFu : 0u) | (seen(i + 1) ? 0xFFFF0000u : 0u);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < DPL; j++) {
                        const f32x4_t x = weigh(j, o[j], mask);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[j][i] = tok == z ? x[i] : o[j][i];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(ro);
            __builtin_amdgcn_sched_barrier(0);
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        /* ---- the four wavefronts' results in one: row r of the tile, element d. */
        int te = tid;
        asm volatile("" : "+v"(te));
        const int ce = te & 15, ge = te >> 4 & 3;
        if (ge == 0) {
            m_s[w][ce] = m == -INFINITY ? -INFINITY : M;
            l_s[w][ce] = l;
        }
        __syncthreads();
        {
            float top = fmaxf(fmaxf(m_s[0][ce], m_s[1][ce]), fmaxf(m_s[2][ce], m_s[3][ce]));
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < DPL; j++) o_s[w][ce][DPL * (4 * ge + i) + j] = o[j][i] * f;
        }
        __syncthreads();
        const pg_args *late = pg_late_args();
        const int rows = tb * a.hpp;
        const bool whole = it.cnt == it.all;
        const int wf = pg_owner(it.first, sh.U, W);
        const size_t slot = ((size_t)2 * me + (me == wf)) * PG_FEW_ROWS;
        /* the finished row: divided, or zeros where it has no key, or NaN where the batch is bad */
        auto finish = [&](int r, int d, float4 v, float top, float L) __attribute__((always_inline)) {
            const int rt = r * a.hinv >> 16, rh = it.part * a.hpp + r - rt * a.hpp;
            if (rh >= a.G) return;
            const int rp = sq.p0 + t0 + rt, h = it.kv * a.G + rh;
            const size_t row = (size_t)(sq.lo + t0 + rt);
            const float nan = __int_as_float(0x7fc00000);
            float4 y = make_float4(v.x / L, v.y / L, v.z / L, v.w / L);
            /* the lift taken back ahead of the logarithm, exactly */
            float e = (top + __builtin_amdgcn_logf(ldexpf(L, -(int)P::LIFT))) * 0.69314718055994531f;
            if (sq.bad) {
                y = make_float4(nan, nan, nan, nan);
                e = nan;
            } else if (rp < 0) {
                y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                e = -INFINITY;
            }
            pg_put4<AT>(late->out, row * late->ldo + (size_t)h * HD + d, y);
            if (late->lse && d == 0) late->lse[row * late->H + h] = e;
        };
        auto put = [&](size_t slot, int r, int d, float4 v, float top, float L) __attribute__((always_inline)) {
            float *pa = late->pacc + (slot + r) * HD + d;
            st_agent(pa + 0, v.x);
            st_agent(pa + 1, v.y);
            st_agent(pa + 2, v.z);
            st_agent(pa + 3, v.w);
            if (d == 0) {
                st_agent((float *)(late->pml + slot + r), top);
                st_agent((float *)(late->pml + slot + r) + 1, L);
            }
        };
        for (int i = te; i < rows * (HD / 4); i += 256) {
            const int r = i / (HD / 4), d = i % (HD / 4) * 4;
            float4 v = *(const float4 *)&o_s[0][r][d];
            const float top = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
            float L = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float mx = m_s[x][r];
                L = fmaf(mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - top), l_s[x][r], L);
                if (x == 0) continue;
                const float4 y = *(const float4 *)&o_s[x][r][d];
                v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
            }
            if (whole) {
                finish(r, d, v, top, L);
            } else {
                put(slot, r, d, v, top, L);
            }
        }
        if (!whole) {
            /* The pieces of workgroups wf .. wl. Up to MG of them: the last to arrive merges them.
               More: the last of each MG merges those into the first one's place, and the last of
               these merges theirs, so that each round of loads flies at once. A workgroup is the
               first of an item's pieces, or of a later group of an item's, with a counter for each. */
            constexpr int MG = 16;
            const int wl = pg_owner(it.first + it.all - 1, sh.U, W);
            const int gx = wf + (me - wf) / MG * MG, groups = (wl - wf) / MG + 1;
            auto place = [&](int x) { return ((size_t)2 * x + (x == wf)) * PG_FEW_ROWS; };
            /* pieces x0, x0 + step, ... (n of them, at most 2 MG) of row r, element d */
            auto merge = [&](int x0, int n, int step, int r, int d, float4 &v, float &top, float &L)
                             __attribute__((always_inline)) {
                v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                top = -INFINITY;
                L = 0.0f;
                for (int k0 = 0; k0 < n; k0 += MG) {
                    f32x2_t ml[MG];
                    float4 y[MG];
#pragma unroll
                    for (int k = 0; k < MG; k++) {
                        const size_t sl = place(x0 + min(k0 + k, n - 1) * step) + r;
                        const unsigned long long b = ld_agent((const unsigned long long *)(late->pml + sl));
                        ml[k] = f32x2_t{__uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))};
                        const v4i_t z = ld_agent16(late->pacc, (uint32_t)((sl * HD + d) * 4));
                        y[k] = make_float4(__int_as_float(z.x), __int_as_float(z.y),
                                           __int_as_float(z.z), __int_as_float(z.w));
                    }
                    float t2 = top;
#pragma unroll
                    for (int k = 0; k < MG; k++) t2 = fmaxf(t2, ml[k].x);
                    const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t2);
                    top = t2;
                    L *= f;
                    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
#pragma unroll
                    for (int k = 0; k < MG; k++) {
                        if (k0 + k < n) {
                        const float e = ml[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - top);
                        L = fmaf(e, ml[k].y, L);
                        v = make_float4(fmaf(e, y[k].x, v.x), fmaf(e, y[k].y, v.y),
                                        fmaf(e, y[k].z, v.z), fmaf(e, y[k].w, v.w));
                        }
                    }
                }
            };
            bool mine = true;
            if (groups > 1) {
                const int n = min(MG, wl - gx + 1);
                mine = last_arriver(&late->ctr[2 * gx + (gx == wf)], n - 1, &flag);
                if (mine) {
                    /* whole rows a pass: a row's (M, l) is replaced once all of the row has it */
                    constexpr int PASS = 256 / (HD / 4) * (HD / 4);
                    for (int i0 = 0; i0 < rows * (HD / 4); i0 += PASS) {
                        const int end = min(i0 + PASS, rows * (HD / 4)), i = i0 + te, ic = min(i, end - 1);
                        const int r = ic / (HD / 4), d = ic % (HD / 4) * 4;
                        float4 v;
                        float top, L;
                        merge(gx, n, 1, r, d, v, top, L);
                        __syncthreads();         /* every thread of the row has read its (M, l) */
                        if (i < end) put(place(gx), r, d, v, top, L);
                    }
                }
            }
            if (mine && last_arriver(&late->ctr[2 * W + wf], groups > 1 ? groups - 1 : wl - wf, &flag))
                for (int i = te; i < rows * (HD / 4); i += 256) {
                    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
                    float4 v;
                    float top, L;
                    merge(wf, groups > 1 ? groups : wl - wf + 1, groups > 1 ? MG : 1, r, d, v, top, L);
                    finish(r, d, v, top, L);
                }
        }
        __syncthreads();                         /* LDS is free for the next item */
    }
}

template <int CT, int AT> static int launch(const pg_args &a, int HD, int grid) {
    auto kernel = HD == 64    ? k_paged_few<CT, AT, 64>
                  : HD == 96  ? k_paged_few<CT, AT, 96>
                  : HD == 128 ? k_paged_few<CT, AT, 128>
                  : HD == 192 ? k_paged_few<CT, AT, 192>
                              : k_paged_few<CT, AT, 256>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, g_cpg.stream, a);
    CPG_LAUNCH_CHECK("k_paged_few");
    return 0;
}

int pg_launch_few(const pg_args &a, int type, int cache, int HD, int grid) {
    if (type == CPG_T_F16) return launch<CPG_T_F16, CPG_T_F16>(a, HD, grid);
    if (type == CPG_T_BF16) return launch<CPG_T_BF16, CPG_T_BF16>(a, HD, grid);
    if (cache == CPG_T_F32) return launch<CPG_T_F32, CPG_T_F32>(a, HD, grid);
    if (cache == CPG_T_F16) return launch<CPG_T_F16, CPG_T_F32>(a, HD, grid);
    return launch<CPG_T_BF16, CPG_T_F32>(a, HD, grid);
}
