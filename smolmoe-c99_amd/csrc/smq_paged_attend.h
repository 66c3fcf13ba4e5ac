/* Attention of a ragged batch of new tokens over a paged KV cache, on MFMA.
 *
 * The rows of a sequence and KV head are its new tokens times the query heads of that KV head, row = token * G + head.
 * A wave takes 16 rows (RT times 16 where it owns rows) as the columns of its products and 32 positions a step:
 *   S^T = K Q^T   two 16 x 16 tiles of positions x rows, K as the A operand straight from the page (its rows are
 *                 positions), position 8 u + i of the step in tile i / 4, row 4 u + i % 4;
 *   P   = 2^(S' - m + 7), S' the score in units of log2 e: by this order a lane holds the scores of 8 consecutive
 *                 positions 8 (lane / 16) .. + 7 for row lane % 16, which is the B operand of
 *   O^T += V^T P^T  as it stands, no exchange between lanes: V^T is the A operand straight from the page, whose
 *                 values lie with positions innermost.
 * So neither product passes through LDS. One pass over the positions: the maximum m of a row is moved (and O and the sum
 * rescaled) only where a score exceeds it by 8, which costs a vote instead of a reduction across lanes in most steps;
 * the weights then reach 2^15, in f16's range, and what f16 subnormals drop is below 2^-32 of the row's largest weight.
 *
 * f32 accuracy on f16 MFMA: q (scaled by a power of two per row) and P are each two f16, value and remainder (22 bits);
 * f16 keys and values and Q8 codes are f16 exactly. Q8 key scales multiply the f32 product of their 32-wide block; value
 * scales multiply P before its split, divided by 2^E, E the exponent of the largest scale of the block so far (O is held
 * in units of 2^E). An f32 cache takes the f32 MFMA, a sixteenth of the rate: its steps are bound by that in chunks, by
 * memory while decoding. */
#ifndef SMQ_PAGED_ATTEND_H
#define SMQ_PAGED_ATTEND_H

#include "smq_paged.h"

namespace smq {

constexpr int PA_WG = 256, PA_WAVES = 4;
constexpr uint32_t PA_STEP = 32;      /* positions */
constexpr uint32_t PA_MIN_STEPS = 8;  /* of a split, at least */
constexpr uint32_t PA_MAX_SPLITS = 64;

/* How a launch covers the rows: tiles of tile_rows rows of one sequence and KV head (`tiles`: as many as the batch can
 * need), each over splits workgroups. owns: a wave owns 16 * RT of the tile's rows over all positions; else the tile has
 * 16 rows and the four waves share the positions out. */
struct AttendPlan {
    bool owns;
    uint32_t tile_rows, tiles, splits, steps;
};
/* Partial results of one split tile: per tile and KV head the splits in use (a word), then per split, row: the maximum,
 * the sum, O. */
inline size_t attend_used_bytes(const PagedArgs &a, const AttendPlan &p) {
    return ((size_t)p.tiles * a.kv_heads * 4 + 15) & ~(size_t)15;
}
inline size_t attend_part_bytes(const PagedArgs &a, const AttendPlan &p) {
    return (size_t)p.tiles * a.kv_heads * p.tile_rows * (a.head_dim + 2) * 4;
}

template <uint32_t TYPE>
hipError_t launch_attend(const PagedArgs &a, const AttendPlan &p, const float *q, float *att, uint32_t *used, float *part,
                         hipStream_t s);

/* RT of the kernels whose waves own rows, by the head size's 32-wide steps: what fits two waves per SIMD. */
constexpr uint32_t attend_rt(uint32_t type, uint32_t ks) { return type == 0 ? (ks <= 2 ? 2 : 1) : ks <= 2 ? 4 : ks <= 4 ? 2 : 1; }
constexpr int attend_waves(uint32_t type, uint32_t ks) { return ks == 8 || (type == 0 && ks > 2) ? 1 : 2; }
constexpr uint32_t attend_ks(uint32_t hd) { return hd <= 32 ? 1 : hd <= 64 ? 2 : hd <= 96 ? 3 : hd <= 128 ? 4 : 8; }

#ifdef SMQ_ATTEND_KERNELS
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float wave_max_quads(float x) { /* over the lanes of one column */
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float wave_sum_quads(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

/* x[0..8) as two f16, value and remainder. The rounded pair is opaque to the compiler: it would round the value a second
 * time elsewhere, from a product that it has not rounded to f32, and the remainder would belong to another value. */
__device__ __forceinline__ void split8(const float *x, h8 &hi, h8 &lo) {
    union {
        h8 h;
        uint32_t u[4];
    } r, s;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        union {
            h2 h;
            uint32_t u;
        } p, q;
        p.h = __builtin_convertvector(f2{x[2 * j], x[2 * j + 1]}, h2);
        asm("" : "+v"(p.u));
        q.h = __builtin_convertvector(f2{__builtin_fmaf((float)p.h[0], -1.0f, x[2 * j]),
                                         __builtin_fmaf((float)p.h[1], -1.0f, x[2 * j + 1])}, h2);
        r.u[j] = p.u;
        s.u[j] = q.u;
    }
    hi = r.h;
    lo = s.h;
}

/* Eight int8 as f16, exactly: the byte plus 128 in the mantissa of 1024 + byte, less 1152. */
__device__ __forceinline__ h8 codes8(u2 w) {
    union {
        uint32_t u[4];
        h8 h;
    } r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t x = w[i] ^ 0x80808080u;
        r.u[2 * i] = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
        r.u[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    }
    return r.h - (_Float16)1152.0f;
}

template <uint32_t TYPE>
struct Elem;
template <>
struct Elem<0> {
    static constexpr uint32_t bytes = 4;
    struct Frag {
        f4 a, b;
    };
};
template <>
struct Elem<1> {
    static constexpr uint32_t bytes = 2;
    typedef h8 Frag;
};
template <>
struct Elem<2> {
    static constexpr uint32_t bytes = 1;
    typedef u2 Frag;
};
/* A lane's part of an A operand: 8 dims of a key or 8 positions of a value dim. */
template <uint32_t TYPE, typename P>
__device__ __forceinline__ typename Elem<TYPE>::Frag load_frag(P p) {
    if constexpr (TYPE == 0) return {*(const f4 *)p, *((const f4 *)p + 1)};
    else return *(const typename Elem<TYPE>::Frag *)p;
}

/* q's fragments: the f32 values or two f16. */
template <uint32_t TYPE>
struct QFrag {
    h8 hi, lo;
};
template <>
struct QFrag<0> {
    float x[8];
};

/* The steps of 32 positions that a tile's rows see: `sinks` of them from position 0, then `total - sinks` from step
 * `first` on. */
struct Steps {
    uint32_t sinks, first, total;
    __device__ __forceinline__ uint32_t at(uint32_t u) const { return u < sinks ? u : u - sinks + first; }
};
__device__ __forceinline__ Steps tile_steps(const PagedArgs &a, int64_t pmin, int64_t pmax) {
    Steps s = {0, 0, 0};
    pmax = min(pmax, (int64_t)a.limit - 1);
    if (pmax < 0) return s;
    const uint32_t low = a.window && pmin + 1 > (int64_t)a.window ? (uint32_t)(pmin + 1 - a.window) : 0;
    if (a.window) s.sinks = (min(a.sinks, (uint32_t)pmax + 1) + PA_STEP - 1) / PA_STEP;
    s.first = max(low / PA_STEP, s.sinks);
    const uint32_t end = (uint32_t)pmax / PA_STEP + 1;
    s.total = s.sinks + (end > s.first ? end - s.first : 0);
    return s;
}

/* Positions that some rows see: [0, sinks) and [low, high]. */
struct Span {
    int high;
    uint32_t low, sinks;
    __device__ __forceinline__ bool holds(uint32_t p) const { return ((int)p <= high && p >= low) || p < sinks; }
    __device__ __forceinline__ bool meets(uint32_t p, uint32_t n) const { /* [p, p + n) */
        return ((int)p <= high && p + n > low) || p < sinks;
    }
};
__device__ __forceinline__ Span span_of(const PagedArgs &a, int pmin, int pmax) {
    Span s;
    s.high = pmax;
    s.low = a.window && (uint32_t)(pmin + 1) > a.window ? (uint32_t)(pmin + 1) - a.window : 0;
    s.sinks = a.window ? min(a.sinks, (uint32_t)(pmax + 1)) : 0;
    return s;
}

/* Where the two halves of 16 positions of a step lie. */
struct Place {
    uint32_t page[2], slot[2];
    uint32_t ok; /* bit h: half h has a page */
};
/* A sequence's page ids, 64 of them in the lanes of a wave. */
struct Table {
    const int32_t *table;
    uint32_t base, ids;
    __device__ __forceinline__ void open(const PagedArgs &a, uint32_t seq) {
        table = a.table + (size_t)seq * a.table_stride;
        base = 0x7fffffff;
        ids = 0;
    }
    /* A page that is none and that `span` needs raises the flag; page 0 then stands in, its positions unseen. */
    __device__ __forceinline__ Place locate(const PagedArgs &a, uint32_t step, const Span &span) {
        const uint32_t p0 = step * PA_STEP, i0 = p0 >> a.shift, i1 = (p0 + 16) >> a.shift, P = 1u << a.shift;
        if (i0 < base || i1 >= base + 64) { /* uniform */
            base = i0;
            ids = (uint32_t)table[min(base + threadIdx.x % 64, a.table_stride - 1)];
        }
        Place pl;
        pl.ok = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            pl.page[h] = (uint32_t)__builtin_amdgcn_readlane(ids, (h ? i1 : i0) - base);
            pl.slot[h] = (p0 + 16 * h) & (P - 1);
            if (pl.page[h] < a.pages) {
                pl.ok |= 1u << h;
            } else {
                if (span.meets(p0 + 16 * h, 16)) *a.flag = 1;
                pl.page[h] = 0;
            }
        }
        return pl;
    }
};
/* Byte offsets of a half's first position: of its keys (head_dim elements a position), of its values (dim 0), of its
 * scales (block 0). */
__device__ __forceinline__ size_t key_at(const PagedArgs &a, uint32_t kh, uint32_t page, uint32_t slot, uint32_t bytes) {
    return ((((size_t)page * a.kv_heads + kh) << a.shift) + slot) * a.head_dim * bytes;
}
__device__ __forceinline__ size_t value_at(const PagedArgs &a, uint32_t kh, uint32_t page, uint32_t slot, uint32_t bytes) {
    return (((((size_t)page * a.kv_heads + kh) * a.head_dim) << a.shift) + slot) * bytes;
}
__device__ __forceinline__ size_t scale_at(const PagedArgs &a, uint32_t kh, uint32_t page, uint32_t slot) {
    return (((((size_t)page * a.kv_heads + kh) * a.nb) << a.shift) + slot) * 4;
}

/* A wave's rows: queries, positions, and the running maximum, sum and O. */
template <uint32_t TYPE, int KS, int RT>
struct Rows {
    static constexpr int DT = 2 * KS;
    typedef typename Elem<TYPE>::Frag Frag;

    const PagedArgs &a;
    uint32_t lane, col, quad;
    /* What this lane's column sees: positions of [from, from + reach] and below first. */
    uint32_t from[RT], reach[RT], first[RT];
    float factor[RT];   /* of a product: the score's scale, log2 e, the row's power of two */
    QFrag<TYPE> qf[RT][KS];
    int pmin;
    Span span;
    uint32_t low_last; /* where the last row's window begins */
    f4 o[RT][DT];
    float m[RT], l[RT];
    float inv_e[TYPE == 2 ? KS : 1]; /* 2^-E of each block of the values */

    /* `count` rows of the sequence from row0 on; columns past them see what the first one sees and are not stored. */
    __device__ __forceinline__ Rows(const PagedArgs &a_, const float *q, const Seq &sq, uint32_t kh, uint32_t row0, int count)
        : a(a_) {
        lane = threadIdx.x % 64;
        col = lane % 16;
        quad = lane / 16;
        const uint32_t G = a.heads / a.kv_heads, hd = a.head_dim;
        const float scale = 1.44269504088896340736f / sqrtf((float)hd);
        int lo = 0x7fffffff, hi = -1;
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const bool in = c * 16 + (int)col < count;
            const uint32_t r = row0 + (in ? c * 16 + col : 0), tok = r / G, g = r % G;
            const int64_t p = sq.first + tok;
            const bool place = p >= 0 && p < (int64_t)a.limit;
            if (in && !place) *a.flag = 1;
            const int pc = place ? (int)p : -1;
            from[c] = !place ? 0xffffffffu : a.window && p + 1 > (int64_t)a.window ? (uint32_t)(p + 1 - a.window) : 0;
            reach[c] = place ? (uint32_t)pc - from[c] : 0;
            first[c] = a.window ? min(a.sinks, (uint32_t)(pc + 1)) : 0;
            lo = min(lo, pc);
            hi = max(hi, pc);
            const float *x = q + ((size_t)(sq.begin + (int)tok) * a.heads + (size_t)kh * G + g) * hd;
            float t[KS][8], big = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint32_t d = s * 32 + quad * 8;
                const bool have = in && d < hd;
                const f4u *y = (const f4u *)(x + (have ? d : 0));
                const f4 y0 = y[0], y1 = y[1];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    t[s][j] = have ? (j < 4 ? y0[j & 3] : y1[j & 3]) : 0.0f;
                    big = fmaxf(big, fabsf(t[s][j]));
                }
            }
            if constexpr (TYPE == 0) {
                factor[c] = scale;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) qf[c][s].x[j] = t[s][j];
            } else {
                big = wave_max_quads(big);
                /* the row's largest below 1024; rows that are nearly 0 keep a factor that is a normal number */
                const int e = big > 0.0f && big <= FLT_MAX ? max(__builtin_amdgcn_frexp_expf(big) - 10, -90) : 0;
                factor[c] = __builtin_ldexpf(scale, e);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[s][j] = __builtin_ldexpf(t[s][j], -e);
                    split8(t[s], qf[c][s].hi, qf[c][s].lo);
                }
            }
            m[c] = -FLT_MAX;
            l[c] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[c][d] = f4{};
        }
#pragma unroll
        for (int off = 1; off < 16; off *= 2) {
            lo = min(lo, __shfl_xor(lo, off));
            hi = max(hi, __shfl_xor(hi, off));
        }
        pmin = __builtin_amdgcn_readfirstlane(lo);
        const int pmax = __builtin_amdgcn_readfirstlane(hi);
        span = span_of(a, pmin, pmax);
        low_last = span_of(a, pmax, pmax).low;
#pragma unroll
        for (int b = 0; b < (TYPE == 2 ? KS : 1); ++b) inv_e[b] = __builtin_ldexpf(1.0f, 100);
    }

    __device__ __forceinline__ bool sees(uint32_t pos, int c) const { return pos - from[c] <= reach[c] || pos < first[c]; }
    /* Whether every row sees all of the step at p0 (rows without a place: pmin -1, never). */
    __device__ __forceinline__ bool full(uint32_t p0, uint32_t ok) const {
        const uint32_t last = p0 + PA_STEP - 1;
        return (int)last <= pmin && ok == 3 && (p0 >= low_last || last < a.sinks);
    }
    __device__ __forceinline__ f4 mma(const h8 &x, const h8 &y, f4 c) const {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    }

    /* The step's products q . k, before `factor`. */
    template <typename Src>
    __device__ __forceinline__ void scores(const Src &src, float (&x)[RT][8]) const {
        if constexpr (TYPE == 2) {
            const f4 z = {};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const h8 k0 = codes8(src.k(0, i)), k1 = codes8(src.k(1, i));
                const f4 w0 = src.kscale(i, 0), w1 = src.kscale(i, 1);
#pragma unroll
                for (int c = 0; c < RT; ++c) {
                    const f4 s0 = mma(k0, qf[c][i].hi, mma(k0, qf[c][i].lo, z));
                    const f4 s1 = mma(k1, qf[c][i].hi, mma(k1, qf[c][i].lo, z));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[c][j] = i ? __builtin_fmaf(s0[j], w0[j], x[c][j]) : s0[j] * w0[j];
                        x[c][4 + j] = i ? __builtin_fmaf(s1[j], w1[j], x[c][4 + j]) : s1[j] * w1[j];
                    }
                }
            }
        } else {
            f4 s[RT][2] = {};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const Frag k = src.k(t, i);
#pragma unroll
                    for (int c = 0; c < RT; ++c) {
                        if constexpr (TYPE == 0) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                s[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(j < 4 ? k.a[j & 3] : k.b[j & 3],
                                                                               qf[c][i].x[j], s[c][t], 0, 0, 0);
                        } else {
                            s[c][t] = mma(k, qf[c][i].lo, s[c][t]);
                            s[c][t] = mma(k, qf[c][i].hi, s[c][t]);
                        }
                    }
                }
#pragma unroll
            for (int c = 0; c < RT; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] = s[c][j >> 2][j & 3];
        }
    }

    /* Products to weights 2^(S' - m + 7), and their sums. */
    __device__ __forceinline__ void weights(uint32_t p0, uint32_t ok, bool full, float (&x)[RT][8]) {
        if (!full) {
            /* positions of a page that is none: past every row */
            const uint32_t p = ok >> (quad >> 1) & 1 ? p0 + quad * 8 : 0xfffffff0u;
#pragma unroll
            for (int c = 0; c < RT; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] = sees(p + j, c) ? x[c][j] : -INFINITY;
        }
        bool up = false;
        float mx[RT];
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            mx[c] = x[c][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx[c] = fmaxf(mx[c], x[c][j]);
            mx[c] *= factor[c];
            up = up || mx[c] > m[c] + 8.0f;
        }
        if (__any(up)) {
#pragma unroll
            for (int c = 0; c < RT; ++c) {
                /* a whole number: 7 - m and the rescaling are exact */
                const float n = fmaxf(m[c], ceilf(wave_max_quads(mx[c]))), alpha = __builtin_amdgcn_exp2f(m[c] - n);
                m[c] = n;
                l[c] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[c][t] *= alpha;
            }
        }
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const float off = 7.0f - m[c];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c][j], factor[c], off));
                l[c] += x[c][j];
            }
        }
    }

    /* Whether x is no number that a product with 0 makes 0. */
    static __device__ __forceinline__ bool odd(float x) { return !(fabsf(x) <= FLT_MAX); }
    /* Element j of a fragment, put and got. */
    static __device__ __forceinline__ float get(const Frag &v, int j) {
        if constexpr (TYPE == 0) return j < 4 ? v.a[j & 3] : v.b[j & 3];
        else return (float)v[j];
    }
    static __device__ __forceinline__ void zero(Frag &v, int j) {
        if constexpr (TYPE == 0) (j < 4 ? v.a : v.b)[j & 3] = 0.0f;
        else v[j] = (_Float16)0.0f;
    }
    /* 0, or a NaN where one of the eight is not finite. */
    static __device__ __forceinline__ float test(const Frag &v) {
        float r = 0.0f;
        if constexpr (TYPE == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r = __builtin_fmaf(get(v, j), 0.0f, r);
        } else {
            const h8 z = v * (_Float16)0.0f;
            const h2 y = h2{z[0], z[1]} + h2{z[2], z[3]} + h2{z[4], z[5]} + h2{z[6], z[7]};
            r = (float)y[0] + (float)y[1];
        }
        return r;
    }
    /* The rows that see positions of `bits` (of the lane's eight) get a NaN for their sum. */
    __device__ __forceinline__ void spoil(uint32_t p0, uint32_t bits) {
#pragma unroll
        for (int off = 1; off < 16; off *= 2) bits |= __shfl_xor(bits, off); /* over the dims of the quad */
#pragma unroll
        for (int c = 0; c < RT; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((bits >> j & 1) && sees(p0 + quad * 8 + j, c)) l[c] = __builtin_nanf("");
    }

    /* O += V^T P^T. In a step that not every row sees whole, a value that is not finite would reach rows that do not see
     * it, as 0 times it: it counts as 0, and the sums of the rows that see it become NaN. Slots that no row sees hold
     * anything; a Q8 scale there must not set E either. */
    template <typename Src>
    __device__ __forceinline__ void product(uint32_t p0, uint32_t ok, bool full, const Src &src, const float (&x)[RT][8]) {
        uint32_t bits = 0;
        if constexpr (TYPE == 2) {
#pragma unroll
            for (int b = 0; b < KS; ++b) {
                f4 w0 = src.vscale(b, 0), w1 = src.vscale(b, 1);
                if (!full) {
                    const bool have = ok >> (quad >> 1) & 1;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float &w = j < 4 ? *((float *)&w0 + j) : *((float *)&w1 + j - 4);
                        w = have && span.holds(p0 + quad * 8 + j) ? w : 0.0f;
                        bits |= odd(w) ? 1u << j : 0;
                        w = odd(w) ? 0.0f : w;
                    }
                }
                float mx = fabsf(w0[0]);
#pragma unroll
                for (int j = 1; j < 8; ++j) mx = fmaxf(mx, fabsf(j < 4 ? w0[j & 3] : w1[j & 3]));
                if (__any(mx * inv_e[b] > 1.0f)) {
                    const int e = max(-100, __builtin_amdgcn_frexp_expf(wave_max_quads(mx)));
                    const float n = __builtin_ldexpf(1.0f, -e), r = n / inv_e[b]; /* a power of two <= 1 */
                    inv_e[b] = n;
#pragma unroll
                    for (int c = 0; c < RT; ++c) {
                        o[c][2 * b] *= r;
                        o[c][2 * b + 1] *= r;
                    }
                }
                w0 *= inv_e[b];
                w1 *= inv_e[b];
                const h8 v0 = codes8(src.v(2 * b)), v1 = codes8(src.v(2 * b + 1));
#pragma unroll
                for (int c = 0; c < RT; ++c) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        w[j] = x[c][j] * (j < 4 ? w0[j & 3] : w1[j & 3]);
                        asm("" : "+v"(w[j])); /* rounded to f32, for both halves of the split */
                    }
                    h8 hi, lo;
                    split8(w, hi, lo);
                    o[c][2 * b] = mma(v0, hi, mma(v0, lo, o[c][2 * b]));
                    o[c][2 * b + 1] = mma(v1, hi, mma(v1, lo, o[c][2 * b + 1]));
                }
            }
            if (!full && __any(bits)) spoil(p0, bits);
        } else {
            bool some = false;
            if (!full) {
                float r = 0.0f;
#pragma unroll
                for (int t = 0; t < DT; ++t) r += test(src.v(t));
                some = __any(!(r == 0.0f));
            }
            h8 hi[RT], lo[RT];
            if constexpr (TYPE == 1) {
#pragma unroll
                for (int c = 0; c < RT; ++c) split8(x[c], hi[c], lo[c]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                Frag v = src.v(t);
                if (some) { /* uniform, rare */
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (odd(get(v, j))) {
                            zero(v, j);
                            bits |= 1u << j;
                        }
                }
#pragma unroll
                for (int c = 0; c < RT; ++c) {
                    if constexpr (TYPE == 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            o[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(get(v, j), x[c][j], o[c][t], 0, 0, 0);
                    } else {
                        o[c][t] = mma(v, hi[c], mma(v, lo[c], o[c][t]));
                    }
                }
            }
            if (some) spoil(p0, ok >> (quad >> 1) & 1 ? bits : 0);
        }
    }

    /* O in units of 1 and the sum over the lanes of a column. */
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            l[c] = wave_sum_quads(l[c]);
            if constexpr (TYPE == 2) {
#pragma unroll
                for (int b = 0; b < KS; ++b) {
                    const float r = 1.0f / inv_e[b];
                    o[c][2 * b] *= r;
                    o[c][2 * b + 1] *= r;
                }
            }
        }
    }
};

/* A step's keys and values in registers, loaded straight from the pages. SMALL: pages of 16, so a step lies in two;
 * else in one, whose address is uniform. Where head_dim ends inside 32 dims of keys the lanes past it read the 16 before
 * again (q is 0 there); value dims past it are read at 0 and not stored. */
template <uint32_t TYPE, int KS, bool SMALL>
struct InRegisters {
    typedef typename Elem<TYPE>::Frag Frag;
    static constexpr uint32_t EB = Elem<TYPE>::bytes;
    static constexpr int DT = 2 * KS, NS = TYPE == 2 ? KS : 1;
    Frag kf[2][KS], vf[DT];
    f4 kw[NS][2], vw[NS][2];

    __device__ __forceinline__ Frag k(int t, int s) const { return kf[t][s]; }
    __device__ __forceinline__ Frag v(int t) const { return vf[t]; }
    __device__ __forceinline__ f4 kscale(int s, int h) const { return kw[s][h]; }
    __device__ __forceinline__ f4 vscale(int s, int h) const { return vw[s][h]; }

    __device__ __forceinline__ void load_k(const PagedArgs &a, uint32_t kh, const Place &pl) {
        const uint32_t lane = threadIdx.x % 64, u = lane % 16 >> 2, quad = lane / 16, hd = a.head_dim;
        const uint32_t row = (u & 1) * 8 + (lane & 3);
        const unsigned char *p = (const unsigned char *)a.keys;
        uint32_t r;
        if constexpr (SMALL) {
            const size_t p0 = key_at(a, kh, pl.page[0], pl.slot[0], EB), p1 = key_at(a, kh, pl.page[1], pl.slot[1], EB);
            p += u >> 1 ? p1 : p0;
            r = row * hd * EB;
        } else {
            p += key_at(a, kh, pl.page[0], pl.slot[0], EB);
            r = (row + (u >> 1) * 16) * hd * EB;
        }
        const uint32_t whole = r + quad * 8 * EB, part = r + (quad & 1) * 8 * EB;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const unsigned char *b = p + (((uint32_t)s * 32 < hd ? s * 32 : 0) + t * 4 * hd) * EB;
                kf[t][s] = load_frag<TYPE>(b + ((uint32_t)s * 32 + 32 <= hd ? whole : part));
            }
        if constexpr (TYPE == 2) load_scales(a, a.ks, kh, pl, kw);
    }
    __device__ __forceinline__ void load_v(const PagedArgs &a, uint32_t kh, const Place &pl) {
        const uint32_t lane = threadIdx.x % 64, quad = lane / 16;
        const unsigned char *p = (const unsigned char *)a.values;
        uint32_t r = (lane % 16 << a.shift) * EB;
        if constexpr (SMALL) {
            const size_t p0 = value_at(a, kh, pl.page[0], pl.slot[0], EB), p1 = value_at(a, kh, pl.page[1], pl.slot[1], EB);
            p += quad >> 1 ? p1 : p0;
            r += (quad & 1) * 8 * EB;
        } else {
            p += value_at(a, kh, pl.page[0], pl.slot[0], EB);
            r += quad * 8 * EB;
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) vf[t] = load_frag<TYPE>(p + (((t * 16u < a.head_dim ? t * 16 : 0) << a.shift) * EB) + r);
        if constexpr (TYPE == 2) load_scales(a, a.vs, kh, pl, vw);
    }
    __device__ __forceinline__ void load_scales(const PagedArgs &a, const float *sc, uint32_t kh, const Place &pl, f4 (&x)[NS][2]) {
        const uint32_t quad = threadIdx.x % 64 / 16;
        const unsigned char *p = (const unsigned char *)sc;
        uint32_t r = quad * 32;
        if constexpr (SMALL) {
            const size_t p0 = scale_at(a, kh, pl.page[0], pl.slot[0]), p1 = scale_at(a, kh, pl.page[1], pl.slot[1]);
            p += quad >> 1 ? p1 : p0;
            r = (quad & 1) * 32;
        } else {
            p += scale_at(a, kh, pl.page[0], pl.slot[0]);
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const f4 *y = (const f4 *)(p + (((uint32_t)s < a.nb ? s : 0) << a.shift) * 4 + r);
            x[s][0] = y[0];
            x[s][1] = y[1];
        }
    }
};

/* A step's keys and values in LDS, brought there by the whole workgroup without registers (global loads to LDS, 16
 * bytes a lane, the lanes' pieces one after another): pieces in the order in which the products read them, so that a
 * fragment's read is free of bank conflicts. f16 and f32: a piece is (half) a lane's fragment. Q8: a piece is 16 codes,
 * the fragments of two quads; one more KiB holds the scales of both, block by block. */
template <uint32_t TYPE, int KS>
struct InLds {
    typedef typename Elem<TYPE>::Frag Frag;
    static constexpr uint32_t EB = Elem<TYPE>::bytes;
    static constexpr int DT = 2 * KS;
    static constexpr uint32_t K_BYTES = 32 * 32 * KS * EB, V_BYTES = K_BYTES;
    static constexpr uint32_t W_BYTES = TYPE == 2 ? 128 * KS : 0; /* the scales of keys or of values */
    static constexpr uint32_t BYTES = K_BYTES + V_BYTES + 2 * W_BYTES;
    static constexpr uint32_t K_LOADS = K_BYTES / 1024, LOADS = 2 * K_LOADS + (2 * W_BYTES + 1023) / 1024; /* of a wave */
    const unsigned char *b; /* the buffer of the step */

    __device__ __forceinline__ Frag k(int t, int s) const {
        const uint32_t lane = threadIdx.x % 64;
        if constexpr (TYPE == 2) /* [dim / 16][t][m][16] */
            return *(const u2 *)(b + (s * 2 + lane / 32) * 512 + t * 256 + lane % 16 * 16 + (lane / 16 & 1) * 8);
        else if constexpr (TYPE == 1) return *(const h8 *)(b + (s * 2 + t) * 1024 + lane * 16);
        else return {*(const f4 *)(b + (s * 2 + t) * 2048 + lane * 16), *(const f4 *)(b + (s * 2 + t) * 2048 + 1024 + lane * 16)};
    }
    __device__ __forceinline__ Frag v(int t) const {
        const uint32_t lane = threadIdx.x % 64;
        const unsigned char *p = b + K_BYTES;
        if constexpr (TYPE == 2) /* [t][position / 16][dim % 16][16] */
            return *(const u2 *)(p + t * 512 + lane / 32 * 256 + lane % 16 * 16 + (lane / 16 & 1) * 8);
        else if constexpr (TYPE == 1) return *(const h8 *)(p + t * 1024 + lane * 16);
        else return {*(const f4 *)(p + t * 2048 + lane * 16), *(const f4 *)(p + t * 2048 + 1024 + lane * 16)};
    }
    __device__ __forceinline__ f4 kscale(int s, int h) const {
        return *(const f4 *)(b + K_BYTES + V_BYTES + s * 128 + (threadIdx.x % 64 / 16) * 32 + h * 16);
    }
    __device__ __forceinline__ f4 vscale(int s, int h) const {
        return *(const f4 *)(b + K_BYTES + V_BYTES + W_BYTES + s * 128 + (threadIdx.x % 64 / 16) * 32 + h * 16);
    }

    /* The lane's piece of load i of a step. */
    static __device__ __forceinline__ const unsigned char *source(const PagedArgs &a, uint32_t kh, const Place &pl, uint32_t i) {
        const uint32_t lane = threadIdx.x % 64, hd = a.head_dim;
        if (i < K_LOADS) {
            uint32_t t, m, d; /* tile, row, first dim */
            if constexpr (TYPE == 2) {
                t = lane / 16 & 1;
                m = lane % 16;
                d = (i * 2 + lane / 32) * 16;
            } else if constexpr (TYPE == 1) {
                t = i & 1;
                m = lane % 16;
                d = i / 2 * 32 + lane / 16 * 8;
            } else {
                t = i / 2 & 1;
                m = lane % 16;
                d = i / 4 * 32 + lane / 16 * 8 + (i & 1) * 4;
            }
            d = d < hd ? d : 0; /* q is 0 there */
            const uint32_t u = m >> 2, pos = u * 8 + t * 4 + (m & 3), h = pos >> 4;
            return (const unsigned char *)a.keys + key_at(a, kh, h ? pl.page[1] : pl.page[0], h ? pl.slot[1] : pl.slot[0], EB) +
                   ((pos & 15) * hd + d) * EB;
        }
        if (i < 2 * K_LOADS) {
            i -= K_LOADS;
            uint32_t d, pos;
            if constexpr (TYPE == 2) {
                d = (i * 2 + lane / 32) * 16 + lane % 16;
                pos = (lane / 16 & 1) * 16;
            } else if constexpr (TYPE == 1) {
                d = i * 16 + lane % 16;
                pos = lane / 16 * 8;
            } else {
                d = i / 2 * 16 + lane % 16;
                pos = lane / 16 * 8 + (i & 1) * 4;
            }
            d = d < hd ? d : 0; /* not stored */
            const uint32_t h = pos >> 4;
            return (const unsigned char *)a.values + value_at(a, kh, h ? pl.page[1] : pl.page[0], h ? pl.slot[1] : pl.slot[0], EB) +
                   ((d << a.shift) + (pos & 15)) * EB;
        }
        const uint32_t x = (i - 2 * K_LOADS) * 64 + lane, block = x / 8 % KS, pos = x % 8 * 4, h = pos >> 4;
        const float *sc = x / 8 < KS ? a.ks : a.vs; /* past both (heads of 32): the values' again, not read */
        return (const unsigned char *)sc + scale_at(a, kh, h ? pl.page[1] : pl.page[0], h ? pl.slot[1] : pl.slot[0]) +
               ((block < a.nb ? block : 0) << a.shift) * 4 + (pos & 15) * 4;
    }
    /* The wave's share of a step's loads into `to`. */
    static __device__ __forceinline__ void load(const PagedArgs &a, uint32_t kh, const Place &pl, uint32_t wave, unsigned char *to) {
#pragma unroll
        for (uint32_t j = 0; j < (LOADS + PA_WAVES - 1) / PA_WAVES; ++j) {
            const uint32_t i = j * PA_WAVES + wave;
            if (i < LOADS)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)source(a, kh, pl, i),
                                                 (__attribute__((address_space(3))) void *)(to + i * 1024), 16, 0, 0);
        }
    }
    static constexpr uint32_t BUFFER = LOADS * 1024;
    /* This wave's loads to LDS are done, then everyone's. */
    static __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
};

/* Where a tile's results go: its rows of att, or the split's partial results. */
struct Out {
    const PagedArgs &a;
    const Seq &sq;
    uint32_t kh, row0, n;  /* n: the tile's rows */
    float *att, *po, *pml; /* po null: att */
    __device__ __forceinline__ void put(uint32_t r, uint32_t d, f4 o, float m, float l) const {
        if (po) {
            *(f4 *)(po + (size_t)r * a.head_dim + d) = o;
            if (d == 0) {
                pml[2 * r] = m;
                pml[2 * r + 1] = l;
            }
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l; /* a row that sees nothing is 0 */
            *(f4u *)(att + row_at(a, sq, kh, row0 + r) + d) = o * inv;
        }
    }
};

/* 16 rows or fewer: the four waves share the steps [u0, u1) out, each with its steps' keys and values in registers, and
 * join their results in LDS. The keys of a wave's next step are requested as soon as this step's are used. */
template <uint32_t TYPE, int KS, bool SMALL>
__device__ __forceinline__ void tile_shared(const PagedArgs &a, const float *q, const Seq &sq, uint32_t seq, const Steps &st,
                                            uint32_t u0, uint32_t u1, uint32_t wave, const Out &out, unsigned char *lds) {
    constexpr int LD = 32 * KS + 4;
    float(*so)[16][LD] = (float(*)[16][LD])lds;
    float(*sml)[16][2] = (float(*)[16][2])(lds + PA_WAVES * 16 * LD * 4);
    Rows<TYPE, KS, 1> w(a, q, sq, out.kh, out.row0, (int)out.n);
    const uint32_t n = u1 - u0, e = u0 + n * (wave + 1) / PA_WAVES;
    u0 += n * wave / PA_WAVES;
    if (u0 < e) {
        Table table;
        table.open(a, seq);
        InRegisters<TYPE, KS, SMALL> src;
        uint32_t at = st.at(u0);
        Place pl = table.locate(a, at, w.span);
        src.load_k(a, out.kh, pl);
        for (uint32_t u = u0; u < e; ++u) {
            const uint32_t p0 = at * PA_STEP;
            at = st.at(min(u + 1, e - 1)); /* the last one's keys twice */
            const Place next = table.locate(a, at, w.span);
            const bool full = w.full(p0, pl.ok);
            float x[1][8];
            src.load_v(a, out.kh, pl);
            w.scores(src, x);
            src.load_k(a, out.kh, next);
            w.weights(p0, pl.ok, full, x);
            w.product(p0, pl.ok, full, src, x);
            pl = next;
        }
    }
    w.finish();
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) *(f4 *)&so[wave][w.col][t * 16 + w.quad * 4] = w.o[0][t];
    if (w.quad == 0) {
        sml[wave][w.col][0] = w.m[0];
        sml[wave][w.col][1] = w.l[0];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < out.n * (a.head_dim / 4); i += PA_WG) {
        const uint32_t r = i / (a.head_dim / 4), d = 4 * (i % (a.head_dim / 4));
        float m = sml[0][r][0], l = 0.0f;
#pragma unroll
        for (int x = 1; x < PA_WAVES; ++x) m = fmaxf(m, sml[x][r][0]);
        f4 o = {};
#pragma unroll
        for (int x = 0; x < PA_WAVES; ++x) {
            const float y = __builtin_amdgcn_exp2f(sml[x][r][0] - m);
            l += y * sml[x][r][1];
            o += y * *(const f4 *)&so[x][r][d];
        }
        out.put(r, d, o, m, l);
    }
}
constexpr uint32_t shared_lds(int ks) { return PA_WAVES * 16 * (32 * ks + 4) * 4 + PA_WAVES * 16 * 8; }

/* Each wave has 16 * RT rows of the tile over the steps [u0, u1), whose keys and values the workgroup brings to LDS, the
 * next step's while this one is computed. A wave without rows (or whose rows do not see a step) only loads. */
template <uint32_t TYPE, int KS, int RT>
__device__ __forceinline__ void tile_owned(const PagedArgs &a, const float *q, const Seq &sq, uint32_t seq, const Steps &st,
                                           uint32_t u0, uint32_t u1, uint32_t wave, const Out &out, unsigned char *lds) {
    typedef InLds<TYPE, KS> Src;
    const uint32_t first = wave * 16 * RT, G = a.heads / a.kv_heads;
    const bool mine = first < out.n;
    /* the last wave's rows again where there are none: never stored */
    Rows<TYPE, KS, RT> w(a, q, sq, out.kh, out.row0 + (mine ? first : 0), mine ? (int)min(16u * RT, out.n - first) : 1);
    /* what the tile sees: the pages that the workgroup needs */
    const int64_t tmin = sq.first + out.row0 / G, tmax = min(sq.first + (out.row0 + out.n - 1) / G, (int64_t)a.limit - 1);
    const Span span = span_of(a, (int)max((int64_t)-1, tmin), (int)max((int64_t)-1, tmax));
    if (u0 < u1) {
        Table table;
        table.open(a, seq);
        uint32_t at = st.at(u0);
        Place pl = table.locate(a, at, span);
        Src::load(a, out.kh, pl, wave, lds);
        Src::wait();
        for (uint32_t u = u0; u < u1; ++u) {
            const uint32_t p0 = at * PA_STEP;
            Place next = pl;
            if (u + 1 < u1) {
                at = st.at(u + 1);
                next = table.locate(a, at, span);
                Src::load(a, out.kh, next, wave, lds + ((u + 1 - u0) & 1) * Src::BUFFER);
            }
            __builtin_amdgcn_sched_barrier(0); /* the loads first: the compiler would sink them behind the products */
            if (mine && w.span.meets(p0, PA_STEP)) {
                const Src src = {lds + ((u - u0) & 1) * Src::BUFFER};
                const bool full = w.full(p0, pl.ok);
                float x[RT][8];
                w.scores(src, x);
                w.weights(p0, pl.ok, full, x);
                w.product(p0, pl.ok, full, src, x);
            }
            pl = next;
            Src::wait(); /* the next step is there, and this one's buffer free */
        }
    }
    if (!mine) return;
    w.finish();
#pragma unroll
    for (int c = 0; c < RT; ++c) {
        const uint32_t r = first + c * 16 + w.col;
        if (r >= out.n) continue;
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) {
            const uint32_t d = t * 16 + w.quad * 4;
            if (d < a.head_dim) out.put(r, d, w.o[c][t], w.m[c], w.l[c]);
        }
    }
}

/* Workgroups by split, KV head, tile: those of one KV head and split follow each other at a distance of all heads and
 * splits, so where these are a multiple of the eight XCDs the tiles of a sequence that read the same pages share an L2.
 * Tiles run from the last to the first: the last rows of a chunk see the most. */
template <uint32_t TYPE, int KS, int RT, bool OWNS, bool SMALL>
__global__ __launch_bounds__(PA_WG, attend_waves(TYPE, KS)) void k_paged_attend(PagedArgs a, const float *q, float *att,
                                                                                uint32_t tile_rows, uint32_t tiles, uint32_t splits,
                                                                                uint32_t *used, float *part) {
    constexpr uint32_t OWN_LDS = OWNS ? 2 * InLds<TYPE, KS>::BUFFER : 0;
    __shared__ __attribute__((aligned(16))) unsigned char lds[OWN_LDS > shared_lds(KS) ? OWN_LDS : shared_lds(KS)];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), split = blockIdx.x % splits;
    const uint32_t kh = blockIdx.x / splits % a.kv_heads, tile = tiles - 1 - blockIdx.x / splits / a.kv_heads;
    const uint32_t G = a.heads / a.kv_heads;
    const size_t slot = (size_t)tile * a.kv_heads + kh;
    uint32_t seq, row0;
    Seq sq;
    if (!find_tile(a, tile, tile_rows, seq, row0) || !sequence(a, seq, sq)) {
        if (used && split == 0 && threadIdx.x == 0) used[slot] = 0;
        return;
    }
    const uint32_t n = min(tile_rows, (uint32_t)sq.n * G - row0);
    const Steps st = tile_steps(a, sq.first + row0 / G, sq.first + (row0 + n - 1) / G);
    const uint32_t parts = max(1u, min(splits, st.total / PA_MIN_STEPS));
    if (used && split == 0 && threadIdx.x == 0) used[slot] = parts;
    if (split >= parts) return;
    const uint32_t u0 = (uint32_t)((uint64_t)st.total * split / parts), u1 = (uint32_t)((uint64_t)st.total * (split + 1) / parts);
    Out out = {a, sq, kh, row0, n, att, nullptr, nullptr};
    if (parts > 1) {
        const size_t r = (slot * splits + split) * tile_rows;
        out.po = part + r * a.head_dim;
        out.pml = part + (size_t)tiles * a.kv_heads * splits * tile_rows * a.head_dim + 2 * r;
    }
    if constexpr (OWNS) {
        if (n > 16) tile_owned<TYPE, KS, RT>(a, q, sq, seq, st, u0, u1, wave, out, lds);
        else tile_shared<TYPE, KS, SMALL>(a, q, sq, seq, st, u0, u1, wave, out, lds);
    } else {
        tile_shared<TYPE, KS, SMALL>(a, q, sq, seq, st, u0, u1, wave, out, lds);
    }
}

}  // namespace

template <uint32_t TYPE>
hipError_t launch_attend(const PagedArgs &a, const AttendPlan &p, const float *q, float *att, uint32_t *used, float *part,
                         hipStream_t s) {
    const dim3 grid(a.kv_heads * p.splits * p.tiles);
#define SMQ_ATTEND3(KS, RT, OWNS, SMALL)                                                                              \
    hipLaunchKernelGGL((k_paged_attend<TYPE, KS, RT, OWNS, SMALL>), grid, dim3(PA_WG), 0, s, a, q, att, p.tile_rows,  \
                       p.tiles, p.splits, used, part)
#define SMQ_ATTEND(KS)                                                            \
    do {                                                                          \
        constexpr int RT = attend_rt(TYPE, KS);                                   \
        if (p.owns && a.shift > 4) SMQ_ATTEND3(KS, RT, true, false);              \
        else if (p.owns) SMQ_ATTEND3(KS, RT, true, true);                         \
        else if (a.shift > 4) SMQ_ATTEND3(KS, 1, false, false);                   \
        else SMQ_ATTEND3(KS, 1, false, true);                                     \
    } while (0)
    switch (attend_ks(a.head_dim)) {
        case 1: SMQ_ATTEND(1); break;
        case 2: SMQ_ATTEND(2); break;
        case 3: SMQ_ATTEND(3); break;
        case 4: SMQ_ATTEND(4); break;
        default: SMQ_ATTEND(8); break;
    }
#undef SMQ_ATTEND
#undef SMQ_ATTEND3
    return hipGetLastError();
}
#endif
}  // namespace smq

#endif
