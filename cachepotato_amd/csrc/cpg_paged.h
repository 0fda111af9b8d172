/* cpg_paged.h — what the kernels of the paged key/value cache share: their arguments, the element
 * types, and each workgroup's walk over its share of the work (cpg_paged_sched.h). */
#ifndef CPG_PAGED_H
#define CPG_PAGED_H
#include "cpg_gemv.h"
#include "cpg_mfma.h"
#include "cpg_paged_sched.h"

#define PG_FEW_ROWS 16      /* query rows of a tile of k_paged_few: one MFMA tile */
#define PG_FEW_WGS 512      /* workgroups of k_paged_few at most: two per CU */

/* one call of cpg_paged_attn, as the kernels get it */
struct pg_args {
    const void *q;
    void *out;
    float *lse;
    const void *k, *v;
    pg_batch b;
    const int *pages;
    int64_t ldq, ldo, page_stride, slot_stride, head_stride;
    int H, G, n_pages, hpp; /* hpp: query heads per tile */
    float scale2;           /* scale * log2(e) */
    const void *zeros, *nans;
    float *pacc;            /* partial results: (2 per workgroup) x rows x HD, and (M, l) of each row */
    float2 *pml;
    int *ctr, *stat;
};

struct cpg_paged_ws {
    int H, KV, HD;
    void *block;
    float *pacc;
    float2 *pml;
    int *ctr, *stat;
    uint8_t *zeros, *nans;
    size_t rows;            /* partial rows there is room for */
};

int pg_launch_few(const pg_args &a, int type, int cache, int HD, int grid);

/* ---------------------------------------------------------------- element types */

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
template <int TYPE> struct pg_elem { typedef uint16_t t; };
template <> struct pg_elem<CPG_T_F32> { typedef float t; };

/* two values rounded to 16 bits, x in the low half */
template <int TYPE> __device__ static inline uint32_t pg_pack2(float x, float y) {
    if constexpr (TYPE == CPG_T_F16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{x, y}), half2_t));
    else
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{x, y}), bf16x2_t));
}
/* the values of a word's halves */
template <int TYPE> __device__ static inline float2 pg_unpack2(uint32_t w) {
    if constexpr (TYPE == CPG_T_F16) {
        const half2_t h = __builtin_bit_cast(half2_t, w);
        return make_float2((float)h.x, (float)h.y);
    } else {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
}
/* four consecutive values to p[0..3] */
template <int TYPE> __device__ static inline void pg_put4(void *p, size_t i, float4 v) {
    if constexpr (TYPE == CPG_T_F32)
        *(float4 *)((float *)p + i) = v;
    else
        *(uint2 *)((uint16_t *)p + i) = make_uint2(pg_pack2<TYPE>(v.x, v.y), pg_pack2<TYPE>(v.z, v.w));
}

/* ---------------------------------------------------------------- shares */

__device__ static inline int64_t pg_wave_scan(int64_t v) {           /* inclusive */
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t p = __shfl_up(v, o);
        if (lane >= o) v += p;
    }
    return v;
}

/* The share of this workgroup. Every thread of the 256 calls it. sc: 8 words of LDS; stat: the
   workspace's status word, set where the batch cannot be followed. */
__device__ static inline pg_share pg_find_share(const pg_batch &b, int64_t *sc, int *stat) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int per = b.KV * b.parts;
    auto units = [&](int s) {
        if (s >= b.S) return (int64_t)0;
        const pg_seq q = pg_get_seq(b.q_off, b.len, s, b.T, b.max_pages, b.plog);
        if (blockIdx.x == 0 && q.bad && (q.cut || q.n > 0)) *stat = 1;
        return q.n ? pg_units_before(q, b.tl, b.window, pg_tiles(q, b.tl)) * per : (int64_t)0;
    };
    pg_share r;
    r.s = 0;
    if (b.S == 1) {
        r.U = units(0);
        pg_deal(r, blockIdx.x, gridDim.x);
        r.rem = r.u0;
        return r;
    }
    /* one round of 256 sequences: the units before each of this thread's, and the round's sum */
    auto round = [&](int s0, int64_t &before, int64_t &mine) {
        mine = units(s0 + tid);
        const int64_t inc = pg_wave_scan(mine);
        __syncthreads();
        if (lane == 63) sc[wv] = inc;
        __syncthreads();
        int64_t sum = 0, ahead = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ahead += i < wv ? sc[i] : 0;
            sum += sc[i];
        }
        before = ahead + inc - mine;
        return sum;
    };
    int64_t before, mine;
    r.U = round(0, before, mine);
    for (int s0 = 256; s0 < b.S; s0 += 256) {
        int64_t b2, m2;
        r.U += round(s0, b2, m2);
    }
    pg_deal(r, blockIdx.x, gridDim.x);
    __syncthreads();
    int64_t base = 0;
    for (int s0 = 0; s0 < b.S && base <= r.u0; s0 += 256) {
        int64_t sum = 0;
        if (b.S > 256) sum = round(s0, before, mine);
        const int64_t at = base + before;
        if (mine > 0 && at <= r.u0 && r.u0 < at + mine) {
            sc[4] = s0 + tid;
            sc[5] = r.u0 - at;
        }
        base += sum;
        if (b.S <= 256) break;
    }
    __syncthreads();
    r.s = (int)sc[4];
    r.rem = sc[5];
    return r;
}

#endif
