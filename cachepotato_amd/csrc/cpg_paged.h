/* cpg_paged.h — what the kernels of the paged key/value cache share: their arguments, the element
 * types, and each workgroup's walk over its share of the work (cpg_paged_sched.h). */
#ifndef CPG_PAGED_H
#define CPG_PAGED_H
#include "cpg_gemv.h"
#include "cpg_mfma.h"
#include "cpg_paged_sched.h"

#define PG_FEW_ROWS 16      /* query rows of a tile of k_paged_few: one MFMA tile */
#define PG_FEW_WGS 256      /* workgroups of k_paged_few at most: one per CU. Its four wavefronts keep
                               64 KiB in flight, and an item has half the pieces of two per CU: 16
                               conversations 20.4 -> 18.6 us, one token over 32767 26.3 -> 21.9, 96
                               sequences 212 -> 200 */
#define PG_MANY_ROWS 128    /* query rows of a tile of k_paged_many: 32 to a wavefront */
#define PG_MANY_WGS 512     /* workgroups of k_paged_many at most: two per CU */

/* one call of cpg_paged_attn, as the kernels get it. Row offsets in the pool are taken in units of
   2^ush bytes, the largest power of two that divides both strides, so that they fit 32 bits. */
struct pg_args {
    const void *q;
    const uint8_t *k, *v;
    const int *pages;
    pg_batch b;
    int64_t ldq, head_bytes;
    int H, G, n_pages;
    int hpp, hinv;          /* query heads per tile; 2^16 / hpp rounded up: r hinv >> 16 = r / hpp for r < 128 */
    uint32_t page_units, slot_units;
    int ush;
    float scale2;           /* scale * log2(e) */
    const uint8_t *blank;   /* 1 KiB of zeros, then 1 KiB of NaNs of every type: rows that are no key's */
    /* ahead of here what the loop over the keys needs */
    void *out;
    float *lse;
    int64_t ldo;
    float *pacc;            /* partial results: (2 per workgroup) x rows x HD, and (M, l) of each row */
    float2 *pml;
    int *ctr, *stat;        /* ctr: PG_MANY_WGS x 3, all zero between calls */
};
/* The kernel's arguments read again where they are used: held in scalar registers over the loop,
   the ones that only the end needs would be spilled. */
__device__ static inline const pg_args *pg_late_args() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return (const pg_args *)p;
}

#define PG_NO_ROW 0xFFFFFFFFu   /* row offsets that are none: a key that no row sees, a bad page id */
#define PG_BAD_ROW 0xFFFFFFFEu

struct cpg_paged_ws {
    int H, KV, HD;
    void *block;
    float *pacc;
    float2 *pml;
    int *ctr, *stat;
    uint8_t *blank;
    size_t rows;            /* partial rows there is room for */
};

int pg_launch_few(const pg_args &a, int type, int cache, int HD, int grid);
int pg_launch_many(const pg_args &a, int type, int cache, int HD, int grid);

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

/* (x, y) as NP pieces of CT, a pair to a word */
template <int CT, int NP>
__device__ static inline void pg_pieces2(float x, float y, uint32_t (&w)[NP]) {
    if constexpr (NP == 1) {
        w[0] = pg_pack2<CT>(x, y);
    } else if constexpr (NP == 2) {
        const f16pair2 p = split_f16x2(x, y);
        w[0] = p.hi;
        w[1] = p.lo;
    } else {                                     /* leading bits, leading bits of the rest, the rest */
        const uint32_t xa = __float_as_uint(x), ya = __float_as_uint(y);
        const float xr = x - __uint_as_float(xa & 0xFFFF0000u), yr = y - __uint_as_float(ya & 0xFFFF0000u);
        const uint32_t xb = __float_as_uint(xr), yb = __float_as_uint(yr);
        const float xs = xr - __uint_as_float(xb & 0xFFFF0000u), ys = yr - __uint_as_float(yb & 0xFFFF0000u);
        w[0] = __builtin_amdgcn_perm(ya, xa, 0x07060302u);
        w[1] = __builtin_amdgcn_perm(yb, xb, 0x07060302u);
        w[2] = __builtin_amdgcn_perm(__float_as_uint(ys), __float_as_uint(xs), 0x07060302u);
    }
}

/* the top bit of a word (of both its halves, for 16-bit types) set where the exponent is all ones,
   an infinity's or a NaN's: one step more carries into it. Words, not truth values, which would
   fill the scalar registers. */
template <int CT> __device__ static inline uint32_t pg_wild(uint32_t w) {
    constexpr uint32_t E = CT == CPG_T_F32 ? 0x7F800000u : CT == CPG_T_F16 ? 0x7C007C00u : 0x7F807F80u;
    constexpr uint32_t ONE = CT == CPG_T_F32 ? 0x00800000u : CT == CPG_T_F16 ? 0x04000400u : 0x00800080u;
    return ((w & E) + ONE) & (CT == CPG_T_F32 ? 0x80000000u : 0x80008000u);
}
/* a word with its infinities and NaNs replaced by zero */
template <int CT> __device__ static inline uint32_t pg_tame(uint32_t w) {
    const uint32_t t = pg_wild<CT>(w);
    return w & ~(t | (t - (t >> (CT == CPG_T_F32 ? 31 : 15))));
}
/* An address computed as a number, for loads from global memory: as a generic pointer its loads
   would count as LDS operations too, and every LDS read would wait for all of them. */
template <typename T> __device__ static inline T pg_load(uint64_t p) {
    return *(const __attribute__((address_space(1))) T *)p;
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

/* the address of a row at offset r of the pool (of keys or of values) */
__device__ static inline uint64_t pg_row_ptr(const uint8_t *base, uint32_t r, int ush, const uint8_t *blank, bool key) {
    const uint64_t p = (uint64_t)base + ((uint64_t)r << ush);
    const uint64_t no = (uint64_t)blank + (key && r == PG_BAD_ROW ? 1024 : 0);
    return r >= PG_BAD_ROW ? no : p;
}

/* 16 bytes stored for another workgroup of this launch (st_agent's form, four words at once) */
__device__ static inline void pg_st_agent16(void *base, uint32_t off, float4 v) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(
        v4i_t{__float_as_int(v.x), __float_as_int(v.y), __float_as_int(v.z), __float_as_int(v.w)}, r, off, 0, 16);
}

/* eight consecutive values to p[i..], a store of 16 bytes for 16-bit types */
template <int TYPE> __device__ static inline void pg_put8(void *p, size_t i, const float (&x)[8]) {
    if constexpr (TYPE == CPG_T_F32) {
        pg_put4<TYPE>(p, i, make_float4(x[0], x[1], x[2], x[3]));
        pg_put4<TYPE>(p, i + 4, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        *(uint4 *)((uint16_t *)p + i) = make_uint4(pg_pack2<TYPE>(x[0], x[1]), pg_pack2<TYPE>(x[2], x[3]),
                                                   pg_pack2<TYPE>(x[4], x[5]), pg_pack2<TYPE>(x[6], x[7]));
    }
}

/* ---------------------------------------------------------------- shares */

/* Where a share begins: the sequence of its first unit and the units before it there. Each
   wavefront finds it by itself, without a barrier: lane l counts the units of sequences l c .. l c +
   c - 1 (c = S / 64, rounded up), a scan over the lanes gives all units and the lane whose sequences
   hold the first of the share, and those are gone through in the same way. stat: the workspace's
   status word, set where the batch cannot be followed. Rows that do not ascend within 0 .. T are no
   batch (two sequences could have a row, and the units would pass their bound): then there is no
   share, in no workgroup, since each looks at all of them. */
struct pg_start {
    int s;
    uint32_t rem;
};

__device__ static inline uint32_t pg_wave_scan(uint32_t v) {         /* inclusive */
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t p = __shfl_up(v, o);
        v += lane >= o ? p : 0;
    }
    return v;
}

__device__ static inline pg_share pg_find_share(const pg_batch &b, pg_start &st, int *stat) {
    const int lane = threadIdx.x & 63;
    bool cut = false;
    auto units = [&](int s) {
        const pg_seq q = pg_get_seq(b.q_off, b.len, s, b.T, b.max_pages, b.plog);
        if (blockIdx.x == 0 && q.bad && (q.cut || q.n > 0)) *stat = 1;
        cut |= q.cut;
        return pg_seq_units(b, q);
    };
    st.s = 0;
    if (b.S == 1) {
        const uint32_t U = units(0);
        const pg_share r = pg_deal(cut ? 0 : U, blockIdx.x, gridDim.x);
        st.rem = r.u0;
        return r;
    }
    int first = 0, n = b.S, c = (n + 63) >> 6;   /* sequences [first, first + n) are looked at */
    uint32_t mine = 0;
    for (int i = 0; i < c; i++) {
        const int s = lane * c + i;
        mine += s < n ? units(s) : 0;
    }
    uint32_t inc = pg_wave_scan(mine);
    const pg_share r = pg_deal(__any(cut) ? 0 : __builtin_amdgcn_readlane(inc, 63), blockIdx.x, gridDim.x);
    st.rem = r.u0;
    if (r.u0 == r.u1) return r;
    for (;;) {
        /* the first lane with the unit among its units or before them: lanes of no units are passed */
        const uint64_t m = __ballot(inc > st.rem);
        const int l = __ffsll((unsigned long long)m) - 1;
        st.rem -= __builtin_amdgcn_readlane(inc - mine, l);
        first += l * c;
        if (c == 1) break;
        n = min(c, first + c <= b.S ? c : b.S - first);
        c = (n + 63) >> 6;
        mine = 0;
        for (int i = 0; i < c; i++) {
            const int s = lane * c + i;
            mine += s < n ? units(first + s) : 0;
        }
        inc = pg_wave_scan(mine);
    }
    st.s = first;
    return r;
}

#endif
