/* Attention of a ragged batch of new tokens over a paged KV cache, on MFMA.
 *
 * The rows of a sequence and KV head are its new tokens times the query heads of that KV head, row = token * G + head.
 * A wave takes 16 rows (RT times 16 where it owns rows) as the columns of its products and 32 positions a step:
 *   S^T = K Q^T   two 16 x 16 tiles of positions x rows, K as the A operand straight from the page (its rows are
 *                 positions), position 8 u + i of the step in tile i / 4, row 4 u + i % 4;
 *   P   = 2^(S' - m + 7), S' the score in units of log2 e (f32 caches: Rows::unit): by this order a lane holds the
 *                 scores of 8 consecutive positions 8 (lane / 16) .. + 7 for row lane % 16, which is the B operand of
 *   O^T += V^T P^T  as it stands, no exchange between lanes: V^T is the A operand straight from the page, whose
 *                 values lie with positions innermost.
 * So no score passes through LDS (keys and values do where waves own rows: InLds). One pass over the positions: the
 * maximum m of a row is moved (and O and the sum rescaled) only where a score exceeds it by 8, which costs a vote instead
 * of a reduction across lanes in most steps; the weights then reach 2^15, in f16's range, and what f16 subnormals round
 * off is at most 2^-25, 2^-31 of the row's largest weight, which is above 2^6.
 *
 * f32 accuracy on f16 MFMA: q (scaled by a power of two per row) and P are each two f16, value and remainder (22 bits);
 * f16 keys and values and Q8 codes are f16 exactly. Q8 key scales multiply the f32 product of their 32-wide block; value
 * scales multiply P before its split, divided by 2^E, E the exponent of the largest scale that the row has seen of the
 * block (O is held in units of 2^E): the 2^-25 is then of that scale. An f32 cache takes the f32 MFMA, a sixteenth of the
 * rate.
 *
 * What bounds it: chunks the matrix cores and the softmax's VALU beside them (64 chunks of 128 tokens at 4096, 32 heads on 8
 * of 128: f16 543 TFLOP/s of products without their remainders, twice that on the matrix cores; Q8 353, whose scales are
 * VALU work; f32 123); decoding the bytes of the cache (16 f16 sequences at up to 16384, 815 MB: 152 us, 5.4 TB/s) once
 * pieces are long, else the latency of a piece: batch, page ids, keys, products and the join one after another (32 Q8
 * sequences at up to 4090: 27 us for 58 MB; one at 131: 8 us). */
#ifndef SMQ_PAGED_ATTEND_H
#define SMQ_PAGED_ATTEND_H

#include "smq_paged.h"

namespace smq {

constexpr int PA_WAVES = 4; /* of a workgroup */
constexpr uint32_t PA_STEP = 32;      /* positions */
constexpr uint32_t PA_MIN_STEPS = 8;  /* of a workgroup, at least, where steps are dealt out */
constexpr uint32_t PA_LONG = 32;      /* of a piece, at least, where `stream` is exceeded */
constexpr uint32_t PA_FIXED = 16;     /* steps that a tile costs beside its own */

/* How a launch covers the rows: tiles of tile_rows rows of one sequence and KV head (`tiles`: as many as the batch can
 * need). owns: a wave owns 16 * RT of the tile's rows over all positions; else the tile has 16 rows and the waves share
 * the positions out.
 *
 * stream > 0: tiles are cut into pieces, each with a workgroup of its own, so that about `stream` of them per KV head (up
 * to `most`: see by_piece) cost the same; k_paged_join joins a tile's. Lengths are known on the device only: each workgroup
 * finds its piece there. A tile counts (c0 + c1 j, at most cw) units of 2^unit / 64 steps, j its number in the sequence:
 * its steps nearly, with sums that need no loop, and PA_FIXED for what it costs beside its steps (the batch looked at,
 * queries, the first keys, the join). A sequence's units laid end to end are cut into equal parts; a tile has a piece for
 * each part that it meets, and these are made equal. There are at most `pieces` of them. stream 0 (no workspace, or nothing
 * to gain): a workgroup per tile. */
typedef int i4 __attribute__((ext_vector_type(4)));
struct AttendPlan {
    bool owns;
    uint32_t tile_rows, row_shift, tiles, stream, most, pieces;
    uint32_t unit, fixed, c1, cw, tile_tokens; /* units; tokens of a tile, at most */
};
/* The workspace: per tile and KV head four words (its pieces, its rows << 16; the sequence's first token; the first row;
 * the first piece's number), then per piece and KV head tile_rows rows: O, and behind all of them the maxima and sums. */
inline size_t attend_used_bytes(const PagedArgs &a, const AttendPlan &p) { return (size_t)p.tiles * a.kv_heads * 16; }
inline size_t attend_piece_bytes(const PagedArgs &a, uint32_t tile_rows) { /* of all KV heads */
    return (size_t)a.kv_heads * tile_rows * (a.head_dim + 2) * 4;
}

template <uint32_t TYPE>
hipError_t launch_attend(const PagedArgs &a, const AttendPlan &p, const float *q, float *att, i4 *used, float *part,
                         hipStream_t s);

/* RT, at most, of the kernels whose waves own rows, by the head size's 32-wide steps, and waves per SIMD. Two column tiles
 * and two waves: each fragment read from LDS serves twice, one wave's softmax runs beside the other's products, and the
 * registers hold (f32 heads of 128: 15 spilled). Useful rate over 64 sequences of 128 tokens at 4096, 32 heads on 8 (RT 1 / 2
 * / 3 or 4), before a column had its own E: f16 heads of 64 403 / 445 / 409 TFLOP/s, of 128 488 / 586 / 215; Q8 252 / 298 /
 * 301, 301 / 363 / 195; f32 123 / 129 / 115, 99 / 127 / 114. Three waves of RT 2: the same or spills. Heads above 128 have one
 * step count (8) and one column tile of one wave a SIMD, whose O and queries fill the registers: 192 dims cost what 256 do (4
 * chunks of 500 at 3000, 32 heads on 8: f16 0.42 and 0.41 ms, Q8 0.74 and 0.75). */
constexpr uint32_t attend_rt(uint32_t ks) { return ks <= 4 ? 2 : 1; }
constexpr int attend_waves(uint32_t ks) { return ks == 8 ? 1 : 2; }
constexpr uint32_t attend_ks(uint32_t hd) { return hd <= 32 ? 1 : hd <= 64 ? 2 : hd <= 96 ? 3 : hd <= 128 ? 4 : 8; }

#ifdef SMQ_ATTEND_KERNELS
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float wave_max_quads(float x) { /* over the lanes of one column */
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float wave_sum_quads(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

/* x[0..8) as two f16, value and remainder (one v_fma_mix each: the remainder is exact). The rounded pair is opaque to
 * the compiler: it would round the value a second time elsewhere, from a product that it has not rounded to f32, and the
 * remainder would belong to another value. */
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
        float r0, r1;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(p.u), "v"(x[2 * j]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(p.u), "v"(x[2 * j + 1]));
        q.h = __builtin_convertvector(f2{r0, r1}, h2);
        r.u[j] = p.u;
        s.u[j] = q.u;
    }
    hi = r.h;
    lo = s.h;
}
/* The largest of three, in one instruction: the compiler's fmaxf makes every input canonical first. A NaN loses. */
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ float max8(const float *x) {
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
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
__device__ __forceinline__ Steps tile_steps(const PagedArgs &a, int pmin, int pmax) {
    Steps s = {0, 0, 0};
    pmax = min(pmax, (int)a.limit - 1);
    if (pmax < 0) return s;
    const uint32_t low = a.window && pmin >= 0 && (uint32_t)pmin + 1 > a.window ? (uint32_t)pmin + 1 - a.window : 0;
    if (a.window) s.sinks = (min(a.sinks, (uint32_t)pmax + 1) + PA_STEP - 1) / PA_STEP;
    s.first = max(low / PA_STEP, s.sinks);
    const uint32_t end = (uint32_t)pmax / PA_STEP + 1;
    s.total = s.sinks + (end > s.first ? end - s.first : 0);
    return s;
}

/* A tile: sequence, its number in it, its number in the batch; its pieces, the number of the first one, which one is
 * meant. */
struct Tile {
    uint32_t seq, j, t, pieces, slot, piece;
    Seq sq;
};
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t x) { /* x plus the lane's neighbour by CTRL, in the rows of the mask */
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t scan_wave(uint32_t x) { /* inclusive, over the 64 lanes */
    x = dpp_add<0x111, 0xf>(x); /* row_shr 1, 2, 4, 8: in rows of 16 */
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x); /* row_bcast 15 into rows 1 and 3 */
    return dpp_add<0x143, 0xc>(x); /* row_bcast 31 into rows 2 and 3 */
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int w) { return (uint32_t)__builtin_amdgcn_readlane(x, w); }

/* The batch's tiles; a wave looks at 64 sequences at a time, one per lane, their lengths requested with their begins. */
struct Tiles {
    const PagedArgs &a;
    const AttendPlan &p;
    int b0, b1, len;
    uint32_t n, c0, c1, cw; /* the lane's sequence: its tiles and their units */
    uint32_t mine, upto, tiles_upto; /* its units, and those and the tiles of the sequences up to it, of the 64 */
    uint32_t at;                     /* the first of the 64 */

    __device__ __forceinline__ Tiles(const PagedArgs &a_, const AttendPlan &p_) : a(a_), p(p_) { look(0); }
    __device__ __forceinline__ void look(uint32_t s0) {
        const uint32_t s = s0 + threadIdx.x % 64;
        at = s0;
        b0 = b1 = len = 0;
        if (s < a.seqs) {
            b0 = a.begin[s];
            b1 = a.begin[s + 1];
            len = a.length[s];
        }
        const bool fine = b0 >= 0 && b1 > b0 && (uint32_t)b1 <= a.tokens; /* else no tile; check_begin raises the flag */
        const uint32_t tokens = fine ? (uint32_t)(b1 - b0) : 0;
        n = (tokens * (a.heads / a.kv_heads) + p.tile_rows - 1) >> p.row_shift;
        const uint32_t pos = len > (int)tokens ? min((uint32_t)len - tokens, a.limit) : 0;
        cw = p.cw;
        c1 = p.c1;
        c0 = min((2 * (pos + min(p.tile_tokens, tokens)) + p.fixed >> p.unit) + 1, cw);
        mine = sum(n, c0, c1, cw);
        upto = scan_wave(mine);
        tiles_upto = scan_wave(n);
    }
    /* Units of the first j tiles of a sequence. */
    static __device__ __forceinline__ uint32_t sum(uint32_t j, uint32_t c0, uint32_t c1, uint32_t cw) {
        const uint32_t k = c1 ? min(j, (cw - c0 + c1 - 1) / c1) : j; /* those below cw */
        return k * c0 + (uint32_t)((uint64_t)k * (k - (k ? 1 : 0)) / 2 * c1) + (j - k) * cw;
    }
    /* More tiles than a batch can have: its sequences overlap (begin does not ascend). None then, the units would not fit. */
    __device__ __forceinline__ void total(uint32_t &units, uint32_t &tiles) {
        units = tiles = 0;
        for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
            if (s0 != at) look(s0);
            units += lane_of(upto, 63);
            tiles += lane_of(tiles_upto, 63);
            if (tiles > p.tiles) {
                units = tiles = 0;
                return;
            }
        }
    }
    __device__ __forceinline__ void take(Tile &t, int w, uint32_t tiles_before) {
        t.seq = at + (uint32_t)w;
        t.t = tiles_before;
        t.sq.begin = (int)lane_of((uint32_t)b0, w);
        t.sq.n = (int)lane_of((uint32_t)b1, w) - t.sq.begin;
        t.sq.first = first_position((int)lane_of((uint32_t)len, w), t.sq.n);
    }
    /* The tile of number x. False behind the last. */
    __device__ __forceinline__ bool by_number(uint32_t x, Tile &t) {
        uint32_t before = 0;
        for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
            if (s0 != at) look(s0);
            const uint64_t past = __ballot(before + tiles_upto > x);
            if (past) {
                const int w = __ffsll((unsigned long long)past) - 1;
                const uint32_t first = before + lane_of(tiles_upto, w) - lane_of(n, w);
                take(t, w, x);
                t.j = x - first;
                t.pieces = 1;
                t.piece = 0;
                return true;
            }
            before += lane_of(tiles_upto, 63);
        }
        return false;
    }
    /* Pieces of the tiles that `units` of a sequence cover, `tiles` of them, where a piece has at most 1 / inv units. Grows
     * with both; a rounding of the product moves a cut by a unit. */
    static __device__ __forceinline__ uint32_t pieces(uint32_t units, uint32_t tiles, float inv) {
        return (uint32_t)((float)units * inv) + tiles;
    }
    /* The tile that piece x is of, of `units` / `count` in all. False behind the last.
     *
     * aim: pieces at most. `stream` of them, two or three times as many where they stay long (decoding: uneven lengths
     * even out; 24 f16 sequences at up to 4000, 8 KV heads of 128: 98 -> 70 us), or every tile's own beside these, where
     * tiles fill half of the workgroups and equal shares would cut only some of them (4 chunks of 300 Q8 tokens at 2600, 8
     * KV heads of 128: 263 -> 194 us).
     *
     * Pieces of u units give units / u + tiles pieces at most: with u = units / (aim - tiles), the start of the search,
     * there are `aim` or fewer; half of aim at least is kept for cuts. Every sequence's last part is rounded up, so a
     * smaller u often has no more than aim either, down to units / aim: six halvings find it, where one look at the
     * batch holds all sequences (16 f16 sequences at up to 16384: 215 -> 154 us). */
    __device__ __forceinline__ bool by_piece(uint32_t x, uint32_t units, uint32_t count, Tile &t) {
        const float all = (float)units, least = (float)(PA_MIN_STEPS * 64 >> p.unit) + 1.0f;
        uint32_t aim = p.stream;
        if (p.owns) aim += 2 * count > aim ? count : 0;
        else aim *= max(units / ((PA_LONG * 64 >> p.unit) + 1) / aim, 1u);
        aim = min(aim, p.most);
        const uint32_t cuts = max(aim > count ? aim - count : 0, (aim + 1) / 2);
        float hi = 1.0f / fmaxf(all / (float)cuts * 1.0001f, least); /* hi, lo: pieces per unit */
        if (a.seqs <= 64) {
            float lo = hi;
            hi = 1.0f / fmaxf(all / (float)aim, least);
            for (int k = 0; k < 6; ++k) {
                const float mid = 0.5f * (lo + hi);
                const bool fits = lane_of(scan_wave(pieces(mine, n, mid)), 63) <= aim;
                lo = fits ? mid : lo;
                hi = fits ? hi : mid;
            }
            hi = lo;
        }
        uint32_t before = 0, tiles = 0;
        for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
            if (s0 != at) look(s0);
            const uint32_t own = pieces(mine, n, hi), to = scan_wave(own);
            const uint64_t past = __ballot(before + to > x);
            if (past) {
                const int w = __ffsll((unsigned long long)past) - 1;
                before += lane_of(to, w) - lane_of(own, w);
                tiles += lane_of(tiles_upto, w) - lane_of(n, w);
                const uint32_t N = lane_of(n, w), d0 = lane_of(c0, w), d1 = lane_of(c1, w), dw = lane_of(cw, w);
                uint32_t j = 0, span = N; /* the last j of [j, j + span) whose first piece is x or before it */
                while (span > 1) {
                    const uint32_t step = (span + 63) / 64, k = j + threadIdx.x % 64 * step;
                    const uint64_t fit = __ballot(k < j + span && before + pieces(sum(k, d0, d1, dw), k, hi) <= x);
                    const uint32_t f = 63 - (uint32_t)__builtin_clzll(fit); /* lane 0 fits */
                    span = min(step, span - f * step);
                    j += f * step;
                }
                take(t, w, tiles + j);
                t.j = j;
                t.slot = before + pieces(sum(j, d0, d1, dw), j, hi);
                t.pieces = before + pieces(sum(j + 1, d0, d1, dw), j + 1, hi) - t.slot;
                t.piece = x - t.slot;
                return true;
            }
            before += lane_of(to, 63);
            tiles += lane_of(tiles_upto, 63);
        }
        return false;
    }
};

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

/* A sequence's pages for one KV head. SMALL: pages of 16 positions, so that a step of 32 lies in two; else in one. The
 * page ids are read 64 at a time, one per lane. */
template <uint32_t TYPE, bool SMALL>
struct Pages {
    static constexpr uint32_t EB = Elem<TYPE>::bytes;
    static constexpr int N = SMALL ? 2 : 1;
    /* Where a step lies, for each of its N parts: its first position's key and dim 0 of its value, and the scales of
     * block 0. Uniform. */
    struct Place {
        const unsigned char *k[N], *v[N], *kw[N], *vw[N];
        uint32_t ok; /* bit h: the half of 16 positions has a page */
    };
    const PagedArgs &a;
    const int32_t *table;
    const unsigned char *k0, *v0, *kw0, *vw0; /* page 0 */
    size_t stride, wstride;                   /* bytes of a page */
    uint32_t base, ids;

    __device__ __forceinline__ Pages(const PagedArgs &a_, uint32_t seq, uint32_t kh) : a(a_) {
        table = a.table + (size_t)seq * a.table_stride;
        base = 0x7fffffff;
        ids = 0;
        const size_t head = ((size_t)a.head_dim << a.shift) * EB, whead = ((size_t)a.nb << a.shift) * 4;
        stride = head * a.kv_heads;
        wstride = whead * a.kv_heads;
        k0 = (const unsigned char *)a.keys + head * kh;
        v0 = (const unsigned char *)a.values + head * kh;
        if constexpr (TYPE == 2) {
            kw0 = (const unsigned char *)a.ks + whead * kh;
            vw0 = (const unsigned char *)a.vs + whead * kh;
        }
    }
    /* A page that is none and that `span` needs raises the flag; page 0 then stands in, its positions unseen. */
    __device__ __forceinline__ Place locate(uint32_t step, const Span &span) {
        const uint32_t p0 = step * PA_STEP, i0 = p0 >> a.shift;
        if (i0 < base || i0 + N > base + 64) { /* uniform */
            base = i0;
            ids = (uint32_t)table[min(base + threadIdx.x % 64, a.table_stride - 1)];
        }
        Place pl;
        pl.ok = 3;
        const uint32_t slot = SMALL ? 0 : p0 & ((1u << a.shift) - 1);
#pragma unroll
        for (int h = 0; h < N; ++h) {
            uint32_t page = (uint32_t)__builtin_amdgcn_readlane(ids, i0 + h - base);
            if (page >= a.pages) {
                if (span.meets(p0 + 16 * h, SMALL ? 16 : 32)) *a.flag = 1;
                page = 0;
                pl.ok = SMALL ? pl.ok & ~(1u << h) : 0;
            }
            pl.k[h] = k0 + stride * page + slot * a.head_dim * EB;
            pl.v[h] = v0 + stride * page + slot * EB;
            if constexpr (TYPE == 2) {
                pl.kw[h] = kw0 + wstride * page + slot * 4;
                pl.vw[h] = vw0 + wstride * page + slot * 4;
            }
        }
        return pl;
    }
};

/* A wave's rows: queries, positions, and the running maximum, sum and O. */
template <uint32_t TYPE, int KS, int RT>
struct Rows {
    static constexpr int DT = 2 * KS;
    typedef typename Elem<TYPE>::Frag Frag;

    const PagedArgs &a;
    uint32_t lane, col, quad;
    /* What this lane's column sees: positions of [from, from + reach] and below first. */
    uint32_t from[RT], reach[RT], first[RT];
    int row[RT]; /* of q and att; -1: none */
    float factor[RT];   /* of a product: the score's scale, log2 e, the row's power of two */
    QFrag<TYPE> qf[RT][KS];
    int pmin;
    Span span;
    uint32_t low_last; /* where the last row's window begins */
    /* Weights are 2^(S' - m + LIFT) * unit, and m moves where a score exceeds it by more than SLACK. An f32 cache needs no
     * f16 range: there a row's weights, one for each position up to the wave's last, sum to less than 1, so that O stays
     * below the values (with weights of 2^15 those of 5e36 made it infinite). The same in every piece: one join takes them.
     * A factor, not part of LIFT: an exponent rounds relative to its size (one sequence at 131: 4.0e-7 off, 4.3e-7). */
    static constexpr float SLACK = TYPE == 0 ? 0.0f : 8.0f, LIFT = TYPE == 0 ? 0.0f : 7.0f;
    float unit;
    f4 o[RT][DT];
    float m[RT], l[RT]; /* l: of this lane's positions, until finish() */
    float inv_e[RT][TYPE == 2 ? KS : 1]; /* 2^-E of each block of the values, of this lane's columns */
    bool alike = true;                   /* every lane's columns have the same E each */

    /* `count` rows of the sequence from row0 on; columns past them see what the first one sees and are not stored. First
     * what they see, then (queries) their values, so that loads of keys can run beside those. */
    __device__ __forceinline__ Rows(const PagedArgs &a_, const Seq &sq, uint32_t kh, uint32_t row0, int count) : a(a_) {
        lane = threadIdx.x % 64;
        col = lane % 16;
        quad = lane / 16;
        const uint32_t G = a.heads / a.kv_heads, tok0 = row0 / G, rest = row0 - tok0 * G;
        const float inv = 1.0f / (float)G;
        int lo = 0x7fffffff, hi = -1;
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const bool in = c * 16 + (int)col < count;
            const uint32_t r = rest + (in ? c * 16 + col : 0);
            const uint32_t up = (uint32_t)(((float)r + 0.5f) * inv); /* r / G: r is below 2^17, where this is exact */
            const uint32_t tok = tok0 + up, g = r - up * G;
            const uint32_t p = (uint32_t)(sq.first + (int)tok);
            const bool place = p < a.limit;
            if (in && !place) *a.flag = 1;
            const int pc = place ? (int)p : -1;
            from[c] = !place ? 0xffffffffu : a.window && p + 1 > a.window ? p + 1 - a.window : 0;
            reach[c] = place ? p - from[c] : 0;
            first[c] = a.window ? min(a.sinks, (uint32_t)(pc + 1)) : 0;
            lo = min(lo, pc);
            hi = max(hi, pc);
            row[c] = in ? (int)(((uint32_t)sq.begin + tok) * a.heads + kh * G + g) : -1; /* below 2^22 */
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
        unit = TYPE == 0 ? __builtin_ldexpf(1.0f, pmax > 0 ? __builtin_clz((uint32_t)pmax) - 33 : -1) : 1.0f;
#pragma unroll
        for (int c = 0; c < RT; ++c)
#pragma unroll
            for (int b = 0; b < (TYPE == 2 ? KS : 1); ++b) inv_e[c][b] = __builtin_ldexpf(1.0f, 112);
    }
    __device__ __forceinline__ void queries(const float *q) {
        const uint32_t hd = a.head_dim;
        const float scale = 1.44269504088896340736f / sqrtf((float)hd);
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const bool in = row[c] >= 0;
            const float *x = q + (size_t)(in ? row[c] : 0) * hd;
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
                    if constexpr (TYPE == 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int c = 0; c < RT; ++c)
                                s[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(get(k, j), qf[c][i].x[j], s[c][t], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int c = 0; c < RT; ++c) s[c][t] = mma(k, qf[c][i].lo, s[c][t]);
#pragma unroll
                        for (int c = 0; c < RT; ++c) s[c][t] = mma(k, qf[c][i].hi, s[c][t]);
                    }
                }
#pragma unroll
            for (int c = 0; c < RT; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] = s[c][j >> 2][j & 3];
        }
    }

    /* Products to weights, and their sums. */
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
            mx[c] = max8(x[c]) * factor[c];
            up = up || mx[c] > m[c] + SLACK;
        }
        if (__any(up)) {
#pragma unroll
            for (int c = 0; c < RT; ++c) {
                /* a whole number: LIFT - m and the rescaling are exact */
                const float n = fmaxf(m[c], ceilf(wave_max_quads(mx[c]))), alpha = __builtin_amdgcn_exp2f(m[c] - n);
                m[c] = n;
                l[c] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[c][t] *= alpha;
            }
        }
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const float off = LIFT - m[c];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c][j], factor[c], off));
                if constexpr (TYPE == 0) x[c][j] *= unit;
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
     * it, as 0 times it: it counts as 0, and the sums of the rows that see it become NaN.
     *
     * Q8 scales belong to the weights: a row takes those that it sees, and E comes of them alone, so that no other position
     * coarsens its weights (with one E for the wave, one of 1e6 times the size that only later rows saw left 1e-4). A
     * column is a row, so E is a lane's own. Where all rows see the step and a lane's columns have the same E, the scales are
     * divided by 2^E once for both (64 chunks of 128 tokens at 4096, 8 KV heads of 128: 1.23 ms; always apart 1.28). */
    template <typename Src>
    __device__ __forceinline__ void product(uint32_t p0, uint32_t ok, bool full, const Src &src, const float (&x)[RT][8]) {
        const bool have = ok >> (quad >> 1) & 1;
        if constexpr (TYPE == 2) {
            f4 w[KS][2];
#pragma unroll
            for (int b = 0; b < KS; ++b) {
                w[b][0] = src.vscale(b, 0);
                w[b][1] = src.vscale(b, 1);
            }
            auto largest = [](const float(&y)[8]) {
                float z[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = fabsf(y[j]);
                return max8(z);
            };
            /* of the scales what column c sees: elsewhere its weight is 0 */
            auto seen = [&](int c, const float(&y)[8], float(&z)[8]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = x[c][j] > 0.0f ? y[j] : 0.0f;
            };
            typedef float(&F8)[8];
            const bool same = RT == 1 || (full && alike); /* one set of scales in units of 2^E serves all columns */
            if (RT == 1 && !full) {
#pragma unroll
                for (int b = 0; b < KS; ++b) seen(0, (F8)w[b], (F8)w[b]);
            }
            float mx[RT][KS];
            if (same) {
#pragma unroll
                for (int b = 0; b < KS; ++b) {
                    mx[0][b] = largest((F8)w[b]);
#pragma unroll
                    for (int c = 1; c < RT; ++c) mx[c][b] = mx[0][b];
                }
            } else {
#pragma unroll
                for (int c = 0; c < RT; ++c)
#pragma unroll
                    for (int b = 0; b < KS; ++b) {
                        float z[8];
                        seen(c, (F8)w[b], z);
                        mx[c][b] = largest(z);
                    }
            }
            bool up = false;
#pragma unroll
            for (int c = 0; c < RT; ++c)
#pragma unroll
                for (int b = 0; b < KS; ++b) up = up || mx[c][b] * inv_e[c][b] > 1.0f;
            if (__any(up)) {
                bool other = false;
#pragma unroll
                for (int c = 0; c < RT; ++c)
#pragma unroll
                    for (int b = 0; b < KS; ++b) {
                        const float top = wave_max_quads(mx[c][b]), old = inv_e[c][b];
                        const int e = max(-112, __builtin_amdgcn_frexp_expf(top));
                        /* zeros: E stays, whichever block asked */
                        inv_e[c][b] = top > 0.0f ? fminf(__builtin_ldexpf(1.0f, -e), old) : old;
                        const float r = __builtin_ldexpf(1.0f, __builtin_amdgcn_frexp_expf(inv_e[c][b]) -
                                                                   __builtin_amdgcn_frexp_expf(old)); /* <= 1 */
                        o[c][2 * b] *= r;
                        o[c][2 * b + 1] *= r;
                        other = other || inv_e[c][b] != inv_e[0][b];
                    }
                alike = RT == 1 || !__any(other);
            }
#pragma unroll
            for (int b = 0; b < KS; ++b) {
                const h8 v0 = codes8(src.v(2 * b)), v1 = codes8(src.v(2 * b + 1));
                float u[8]; /* the scales in units of 2^E */
#pragma unroll
                for (int c = 0; c < RT; ++c) {
                    if (c == 0 || !same) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) u[j] = w[b][j >> 2][j & 3] * inv_e[c][b];
                        if (!same) seen(c, u, u);
                    }
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        y[j] = x[c][j] * u[j];
                        asm("" : "+v"(y[j])); /* rounded to f32, for both halves of the split */
                    }
                    h8 hi, lo;
                    split8(y, hi, lo);
                    o[c][2 * b] = mma(v0, lo, o[c][2 * b]);
                    o[c][2 * b + 1] = mma(v1, lo, o[c][2 * b + 1]);
                    o[c][2 * b] = mma(v0, hi, o[c][2 * b]);
                    o[c][2 * b + 1] = mma(v1, hi, o[c][2 * b + 1]);
                }
            }
        } else {
            Frag v[DT];
#pragma unroll
            for (int t = 0; t < DT; ++t) v[t] = src.v(t);
            if (!full) {
                float r = 0.0f;
#pragma unroll
                for (int t = 0; t < DT; ++t) r += test(v[t]);
                if (__any(!(r == 0.0f))) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (odd(get(v[t], j))) {
                                zero(v[t], j);
                                bits |= 1u << j;
                            }
                    spoil(p0, have ? bits : 0);
                }
            }
            h8 hi[RT], lo[RT];
            if constexpr (TYPE == 1) {
#pragma unroll
                for (int c = 0; c < RT; ++c) split8(x[c], hi[c], lo[c]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if constexpr (TYPE == 0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int c = 0; c < RT; ++c)
                            o[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(get(v[t], j), x[c][j], o[c][t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < RT; ++c) o[c][t] = mma(v[t], lo[c], o[c][t]);
#pragma unroll
                    for (int c = 0; c < RT; ++c) o[c][t] = mma(v[t], hi[c], o[c][t]);
                }
            }
        }
    }

    /* O in units of 1 and the sum over the lanes of a column; both times the power of two that brings the sum into
     * [1/2, 1), with m for it, so that O is no larger than the values (f16 ones cannot leave f32's range). */
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            l[c] = wave_sum_quads(l[c]);
            if constexpr (TYPE != 1) {
                const int k = __builtin_amdgcn_frexp_expf(l[c]); /* 0 where the sum is 0 */
                l[c] = __builtin_ldexpf(l[c], -k);
                m[c] += (float)k;
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int e = TYPE == 2 ? 1 - __builtin_amdgcn_frexp_expf(inv_e[c][TYPE == 2 ? t / 2 : 0]) : 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[c][t][j] = __builtin_ldexpf(o[c][t][j], e - k);
                }
            }
        }
    }
};

/* A step's keys and values in registers, loaded straight from the pages. Where head_dim ends inside 32 dims of keys the
 * lanes past it read the 16 before again (q is 0 there); value dims past it are read at 0 and not stored. */
template <uint32_t TYPE, int KS, bool SMALL>
struct InRegisters {
    typedef typename Elem<TYPE>::Frag Frag;
    typedef typename Pages<TYPE, SMALL>::Place Place;
    static constexpr uint32_t EB = Elem<TYPE>::bytes;
    static constexpr int DT = 2 * KS, NS = TYPE == 2 ? KS : 1;
    Frag kf[2][KS], vf[DT];
    f4 kw[NS][2], vw[NS][2];
    uint32_t hd, shift, nb, kwhole, kpart, voff, woff; /* the lane's offsets */
    bool second;                                       /* SMALL: of the second page; keys and values alike */
    bool ksecond;

    __device__ __forceinline__ InRegisters(const PagedArgs &a) : hd(a.head_dim), shift(a.shift), nb(a.nb) {
        const uint32_t lane = threadIdx.x % 64, u = lane % 16 >> 2, quad = lane / 16;
        ksecond = SMALL && u >> 1;
        second = SMALL && quad >> 1;
        const uint32_t r = ((SMALL ? u & 1 : u) * 8 + (lane & 3)) * hd * EB, q = SMALL ? quad & 1 : quad;
        kwhole = r + quad * 8 * EB;
        kpart = r + (quad & 1) * 8 * EB;
        voff = ((lane % 16 << shift) + q * 8) * EB;
        woff = q * 32;
    }
    __device__ __forceinline__ Frag k(int t, int s) const { return kf[t][s]; }
    __device__ __forceinline__ Frag v(int t) const { return vf[t]; }
    __device__ __forceinline__ f4 kscale(int s, int h) const { return kw[s][h]; }
    __device__ __forceinline__ f4 vscale(int s, int h) const { return vw[s][h]; }

    static __device__ __forceinline__ const unsigned char *pick(const unsigned char *const (&p)[Pages<TYPE, SMALL>::N], bool second) {
        if constexpr (SMALL) return second ? p[1] : p[0];
        else return p[0];
    }
    __device__ __forceinline__ void load_k(const Place &pl) {
        const unsigned char *p = pick(pl.k, ksecond);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const unsigned char *b = p + (((uint32_t)s * 32 < hd ? s * 32 : 0) + t * 4 * hd) * EB;
                kf[t][s] = load_frag<TYPE>(b + ((uint32_t)s * 32 + 32 <= hd ? kwhole : kpart));
            }
        if constexpr (TYPE == 2) load_scales(pick(pl.kw, second), kw);
    }
    __device__ __forceinline__ void load_v(const Place &pl) {
        const unsigned char *p = pick(pl.v, second);
#pragma unroll
        for (int t = 0; t < DT; ++t) vf[t] = load_frag<TYPE>(p + (((t * 16u < hd ? t * 16 : 0) << shift) * EB) + voff);
        if constexpr (TYPE == 2) load_scales(pick(pl.vw, second), vw);
    }
    __device__ __forceinline__ void load_scales(const unsigned char *p, f4 (&x)[NS][2]) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const f4 *y = (const f4 *)(p + (((uint32_t)s < nb ? s : 0) << shift) * 4 + woff);
            x[s][0] = y[0];
            x[s][1] = y[1];
        }
    }
};

/* A step's keys and values in LDS, brought there by the whole workgroup without registers (global loads to LDS, 16
 * bytes a lane, the lanes' pieces one after another): pieces in the order in which the products read them, so that a
 * fragment's read is free of bank conflicts. f16 and f32: a piece is (half) a lane's fragment. Q8: a piece is 16 codes,
 * the fragments of two quads; behind them the scales of both, block by block. */
template <uint32_t TYPE, int KS, bool SMALL>
struct InLds {
    typedef typename Elem<TYPE>::Frag Frag;
    typedef typename Pages<TYPE, SMALL>::Place Place;
    static constexpr uint32_t EB = Elem<TYPE>::bytes;
    static constexpr int DT = 2 * KS;
    static constexpr uint32_t K_BYTES = 32 * 32 * KS * EB;
    static constexpr uint32_t W_BYTES = TYPE == 2 ? 128 * KS : 0; /* the scales of keys or of values */
    static constexpr uint32_t K_LOADS = K_BYTES / 1024, W_LOADS = (2 * W_BYTES + 1023) / 1024; /* of a wave */
    static constexpr uint32_t BUFFER = 2 * K_BYTES + W_LOADS * 1024, EACH = (K_LOADS + PA_WAVES - 1) / PA_WAVES;
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
        return *(const f4 *)(b + 2 * K_BYTES + s * 128 + (threadIdx.x % 64 / 16) * 32 + h * 16);
    }
    __device__ __forceinline__ f4 vscale(int s, int h) const {
        return *(const f4 *)(b + 2 * K_BYTES + W_BYTES + s * 128 + (threadIdx.x % 64 / 16) * 32 + h * 16);
    }

    /* A wave's part of a step's loads: every fourth piece of keys and of values, one wave the scales. The lane's
     * offsets from the step's place, and which of two pages they are from. */
    struct Loader {
        uint32_t wave, koff[EACH], voff[EACH], woff[W_LOADS ? W_LOADS : 1];
        bool ksecond, vsecond, wsecond, wvalues[W_LOADS ? W_LOADS : 1];

        __device__ __forceinline__ Loader(const PagedArgs &a, uint32_t wave_) : wave(wave_) {
            const uint32_t lane = threadIdx.x % 64, hd = a.head_dim, m = lane % 16, quad = lane / 16;
            ksecond = SMALL && m >> 3;
            vsecond = SMALL && (TYPE == 2 ? quad & 1 : quad >> 1);
            wsecond = SMALL && lane % 8 / 4;
#pragma unroll
            for (uint32_t j = 0; j < EACH; ++j) {
                const uint32_t i = j * PA_WAVES + wave;
                uint32_t t, d; /* keys: tile and first dim */
                if constexpr (TYPE == 2) {
                    t = quad & 1;
                    d = (i * 2 + lane / 32) * 16;
                } else if constexpr (TYPE == 1) {
                    t = i & 1;
                    d = i / 2 * 32 + quad * 8;
                } else {
                    t = i / 2 & 1;
                    d = i / 4 * 32 + quad * 8 + (i & 1) * 4;
                }
                d = d < hd ? d : 0; /* q is 0 there */
                uint32_t pos = (m >> 2) * 8 + t * 4 + (m & 3);
                koff[j] = ((SMALL ? pos & 15 : pos) * hd + d) * EB;
                if constexpr (TYPE == 2) { /* values: dim and first position */
                    d = (i * 2 + lane / 32) * 16 + m;
                    pos = (quad & 1) * 16;
                } else if constexpr (TYPE == 1) {
                    d = i * 16 + m;
                    pos = quad * 8;
                } else {
                    d = i / 2 * 16 + m;
                    pos = quad * 8 + (i & 1) * 4;
                }
                d = d < hd ? d : 0; /* not stored */
                voff[j] = ((d << a.shift) + (SMALL ? pos & 15 : pos)) * EB;
            }
#pragma unroll
            for (uint32_t j = 0; j < W_LOADS; ++j) {
                const uint32_t x = j * 64 + lane, block = x / 8 % KS, pos = x % 8 * 4;
                wvalues[j] = x / 8 >= KS; /* past both (heads of 32): the values' again, not read */
                woff[j] = (((block < a.nb ? block : 0) << a.shift) + (SMALL ? pos & 15 : pos)) * 4;
            }
        }
        static __device__ __forceinline__ void move(const unsigned char *from, unsigned char *to) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                             (__attribute__((address_space(3))) void *)to, 16, 0, 0);
        }
        __device__ __forceinline__ void load(const Place &pl, unsigned char *to) const {
            typedef InRegisters<TYPE, KS, SMALL> Pick;
            const unsigned char *k = Pick::pick(pl.k, ksecond), *v = Pick::pick(pl.v, vsecond);
#pragma unroll
            for (uint32_t j = 0; j < EACH; ++j) {
                const uint32_t i = j * PA_WAVES + wave;
                if (K_LOADS % PA_WAVES == 0 || i < K_LOADS) {
                    move(k + koff[j], to + i * 1024);
                    move(v + voff[j], to + K_BYTES + i * 1024);
                }
            }
            if constexpr (TYPE == 2) {
                if (wave == PA_WAVES - 1) {
                    const unsigned char *kw = Pick::pick(pl.kw, wsecond), *vw = Pick::pick(pl.vw, wsecond);
#pragma unroll
                    for (uint32_t j = 0; j < W_LOADS; ++j)
                        move((wvalues[j] ? vw : kw) + woff[j], to + 2 * K_BYTES + j * 1024);
                }
            }
        }
    };
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
            *(f4u *)(att + row_at(a, sq.begin, kh, row0 + r) + d) = o * inv;
        }
    }
};

/* 16 rows or fewer: the waves take the steps [u0, u1) in turn, each with its steps' keys and values in registers, and
 * join their results in LDS. In turn, not in runs: a step's values are 64 bytes (f16) of each dim's row in the page, and
 * the cache lines' other halves are the next steps'; with runs half of every line was fetched twice. The keys of a wave's next step are requested as soon as this step's are used. */
template <uint32_t TYPE, int KS, bool SMALL>
__device__ __forceinline__ void tile_shared(const PagedArgs &a, const float *q, const Seq &sq, uint32_t seq, const Steps &st,
                                            uint32_t u0, uint32_t u1, uint32_t wave, const Out &out, unsigned char *lds) {
    constexpr int LD = 32 * KS + 4;
    float(*so)[16][LD] = (float(*)[16][LD])lds;
    float(*sml)[16][2] = (float(*)[16][2])(lds + PA_WAVES * 16 * LD * 4);
    Rows<TYPE, KS, 1> w(a, sq, out.kh, out.row0, (int)out.n);
    u0 += wave;
    if (u0 >= u1) {
        w.queries(q);
    } else {
        Pages<TYPE, SMALL> pages(a, seq, out.kh);
        InRegisters<TYPE, KS, SMALL> src(a);
        uint32_t at = st.at(u0);
        auto pl = pages.locate(at, w.span);
        src.load_k(pl);
        w.queries(q);
        for (uint32_t u = u0; u < u1; u += PA_WAVES) {
            const uint32_t p0 = at * PA_STEP;
            at = st.at(u + PA_WAVES < u1 ? u + PA_WAVES : u); /* the last one's keys twice */
            src.load_v(pl);
            const auto next = pages.locate(at, w.span);
            const bool full = w.full(p0, pl.ok);
            float x[1][8];
            w.scores(src, x);
            src.load_k(next);
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
    for (uint32_t i = threadIdx.x; i < out.n * (a.head_dim / 4); i += 64 * PA_WAVES) {
        const uint32_t r = i / (a.head_dim / 4), d = 4 * (i % (a.head_dim / 4));
        float m = sml[0][r][0], l = 0.0f;
#pragma unroll
        for (int x = 1; x < PA_WAVES; ++x) m = fmaxf(m, sml[x][r][0]);
        m += 2.0f; /* a quarter of each of the four: O stays below the values, however large */
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
template <uint32_t TYPE, int KS, int RT, bool SMALL>
__device__ __forceinline__ void tile_owned(const PagedArgs &a, const float *q, const Seq &sq, uint32_t seq, const Steps &st,
                                           uint32_t u0, uint32_t u1, uint32_t wave, const Out &out, unsigned char *lds) {
    typedef InLds<TYPE, KS, SMALL> Src;
    const uint32_t first = wave * 16 * RT, G = a.heads / a.kv_heads;
    const bool mine = first < out.n;
    /* the last wave's rows again where there are none: never stored */
    Rows<TYPE, KS, RT> w(a, sq, out.kh, out.row0 + (mine ? first : 0), mine ? (int)min(16u * RT, out.n - first) : 1);
    /* what the tile sees: the pages that the workgroup needs */
    const int tmin = sq.first + (int)(out.row0 / G), tmax = min(sq.first + (int)((out.row0 + out.n - 1) / G), (int)a.limit - 1);
    const Span span = span_of(a, max(-1, tmin), max(-1, tmax));
    if (u0 >= u1) {
        w.queries(q);
    } else {
        Pages<TYPE, SMALL> pages(a, seq, out.kh);
        const typename Src::Loader loader(a, wave);
        uint32_t at = st.at(u0);
        auto pl = pages.locate(at, span);
        loader.load(pl, lds);
        w.queries(q);
        Src::wait();
        for (uint32_t u = u0; u < u1; ++u) {
            const uint32_t p0 = at * PA_STEP, ok = pl.ok;
            if (u + 1 < u1) {
                at = st.at(u + 1);
                pl = pages.locate(at, span);
                loader.load(pl, lds + ((u + 1 - u0) & 1) * Src::BUFFER);
            }
            __builtin_amdgcn_sched_barrier(0); /* the loads first: the compiler would sink them behind the products */
            if (mine && w.span.meets(p0, PA_STEP)) {
                const Src src = {lds + ((u - u0) & 1) * Src::BUFFER};
                const bool full = w.full(p0, ok);
                float x[RT][8];
                w.scores(src, x);
                w.weights(p0, ok, full, x);
                w.product(p0, ok, full, src, x);
            }
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

/* A tile's piece. */
template <uint32_t TYPE, int KS, int RT, bool OWNS, bool SMALL>
__device__ __forceinline__ void tile_part(const PagedArgs &a, const AttendPlan &p, const float *q, float *att, i4 *used,
                                          float *part, uint32_t kh, const Tile &t, unsigned char *lds) {
    const uint32_t G = a.heads / a.kv_heads, row0 = t.j * p.tile_rows, n = min(p.tile_rows, (uint32_t)t.sq.n * G - row0);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Steps st = tile_steps(a, t.sq.first + (int)(row0 / G), t.sq.first + (int)((row0 + n - 1) / G));
    Out out = {a, t.sq, kh, row0, n, att, nullptr, nullptr};
    uint32_t u0 = 0, u1 = st.total;
    if (p.stream && t.piece == 0 && threadIdx.x == 0)
        used[(size_t)t.t * a.kv_heads + kh] = i4{(int)(t.pieces | n << 16), t.sq.begin, (int)row0, (int)t.slot};
    if (t.pieces > 1) {
        const size_t r = ((size_t)(t.slot + t.piece) * a.kv_heads + kh) * p.tile_rows;
        out.po = part + r * a.head_dim;
        out.pml = part + (size_t)p.pieces * a.kv_heads * p.tile_rows * a.head_dim + 2 * r;
        u0 = st.total * t.piece / t.pieces; /* 2^15 steps at most, pieces below 2^16 */
        u1 = st.total * (t.piece + 1) / t.pieces;
    }
    if constexpr (OWNS) {
        if (n > 16) {
            tile_owned<TYPE, KS, RT, SMALL>(a, q, t.sq, t.seq, st, u0, u1, wave, out, lds);
            return;
        }
    }
    tile_shared<TYPE, KS, SMALL>(a, q, t.sq, t.seq, st, u0, u1, wave, out, lds);
}

/* Workgroups of one KV head follow each other at a distance of all heads, so where these are a multiple of the eight XCDs
 * the tiles of a sequence that read the same pages share an L2. From the last tile to the first: the last rows of a chunk
 * see the most. A piece has a workgroup of its own: a loop over several costs the products their registers (heads of 128:
 * 40 spilled), and one that takes a second piece, however short, pays a tile's fixed cost twice. */
template <uint32_t TYPE, int KS, int RT, bool OWNS, bool SMALL>
__global__ __launch_bounds__(64 * PA_WAVES, attend_waves(KS)) void k_paged_attend(PagedArgs a, const float *q, float *att,
                                                                                  AttendPlan p, i4 *used, float *part) {
    constexpr uint32_t OWN_LDS = OWNS ? 2 * InLds<TYPE, KS, SMALL>::BUFFER : 0;
    __shared__ __attribute__((aligned(16))) unsigned char lds[OWN_LDS > shared_lds(KS) ? OWN_LDS : shared_lds(KS)];
    const uint32_t kh = blockIdx.x % a.kv_heads, i = blockIdx.x / a.kv_heads;
    if (blockIdx.x == 0) check_begin(a, threadIdx.x, 64 * PA_WAVES);
    Tile t;
    {
        Tiles tiles(a, p);
        if (!p.stream) {
            if (!tiles.by_number(p.tiles - 1 - i, t)) return;
        } else {
            uint32_t units, count;
            tiles.total(units, count);
            if (i == 0) /* tiles that the batch does not need */
                for (uint32_t x = count + threadIdx.x; x < p.tiles; x += 64 * PA_WAVES) used[(size_t)x * a.kv_heads + kh] = i4{};
            if (!count || !tiles.by_piece(p.pieces - 1 - i, units, count, t)) return;
        }
    }
    tile_part<TYPE, KS, RT, OWNS, SMALL>(a, p, q, att, used, part, kh, t, lds);
}

}  // namespace

template <uint32_t TYPE>
hipError_t launch_attend(const PagedArgs &a, const AttendPlan &p, const float *q, float *att, i4 *used, float *part,
                         hipStream_t s) {
    const dim3 grid(a.kv_heads * (p.stream ? p.pieces : p.tiles));
#define SMQ_ATTEND3(KS, RT, OWNS, SMALL)                                                                               \
    hipLaunchKernelGGL((k_paged_attend<TYPE, KS, RT, OWNS, SMALL>), grid, dim3(64 * PA_WAVES), 0, s, a, q, att, p, used, \
                       part)
#define SMQ_ATTEND(KS)                                                            \
    do {                                                                          \
        constexpr int RT = attend_rt(KS);                                         \
        const bool most = p.tile_rows == 64 * RT; /* else 64 */                   \
        if (p.owns && most && a.shift > 4) SMQ_ATTEND3(KS, RT, true, false);      \
        else if (p.owns && most) SMQ_ATTEND3(KS, RT, true, true);                 \
        else if (p.owns && a.shift > 4) SMQ_ATTEND3(KS, 1, true, false);          \
        else if (p.owns) SMQ_ATTEND3(KS, 1, true, true);                          \
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
