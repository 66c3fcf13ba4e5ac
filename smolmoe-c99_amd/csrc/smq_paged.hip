/* Paged KV cache on gfx950: RoPE and the store of new tokens (f32, f16, Q8), rows read back, and the attention of a
 * ragged batch of new tokens over the pages (include/smq.h has the layout of a page). */
#include "smq_paged_attend.h"

namespace smq {
namespace {

constexpr uint32_t ST_WG = 256;
constexpr uint32_t ST_POS = 32; /* positions of a block */

/* Blocks of ST_POS positions (from a multiple of it on) that the new tokens of the sequences touch: block x's sequence and
 * positions [p0, p1), all of them places. Uniform over a wave; false behind the last. */
struct Block {
    uint32_t seq, p0, p1;
    int row; /* of position 0: begin - first */
};
__device__ __forceinline__ bool find_block(const PagedArgs &a, uint32_t x, Block &b) {
    const uint32_t lane = threadIdx.x % 64;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
        const uint32_t s = s0 + lane;
        int b0 = 0, n = 0, first = 0;
        if (s < a.seqs) {
            b0 = a.begin[s];
            n = a.begin[s + 1] - b0;
            if (b0 < 0 || n < 0 || (uint32_t)n > a.tokens - (uint32_t)min((uint32_t)b0, a.tokens)) n = 0; /* check_begin */
            first = first_position(a.length[s], n);
        }
        const int from = max(first, 0), to = min(first + n, (int)a.limit);
        if (n && (from != first || to != first + n)) *a.flag = 1; /* rows without a place */
        const uint32_t blocks = to > from ? (uint32_t)(to - 1) / ST_POS - (uint32_t)from / ST_POS + 1 : 0;
        uint32_t upto = blocks;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const uint32_t y = __shfl_up(upto, off);
            upto += (int)lane >= off ? y : 0;
        }
        const uint64_t past = __ballot(before + upto > x);
        if (past) {
            const int w = __ffsll((unsigned long long)past) - 1;
            const uint32_t k = x - before - (uint32_t)(__builtin_amdgcn_readlane(upto, w) - __builtin_amdgcn_readlane(blocks, w));
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane(from, w), hi = (uint32_t)__builtin_amdgcn_readlane(to, w);
            const uint32_t at = (lo / ST_POS + k) * ST_POS;
            b.seq = s0 + (uint32_t)w;
            b.p0 = max(at, lo);
            b.p1 = min(at + ST_POS, hi);
            b.row = __builtin_amdgcn_readlane(b0, w) - __builtin_amdgcn_readlane(first, w);
            return true;
        }
        before += (uint32_t)__builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}
/* As many blocks as a batch can need: n tokens touch (n - 1) / 32 + 2 at most, and n. */
uint32_t most_blocks(const PagedArgs &a) {
    const uint64_t most = a.tokens / ST_POS + 2 * (uint64_t)a.seqs;
    return most < a.tokens ? (uint32_t)most : a.tokens;
}
/* The block's page ids of 16 positions each, one per lane of 0 .. 1 (blocks of one page have the same one twice); -1, with
 * the flag, where a page that the block needs is none. */
__device__ __forceinline__ void block_pages(const PagedArgs &a, const Block &b, int (&page)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t p = b.p0 / ST_POS * ST_POS + 16 * h;
        page[h] = p < b.p1 && p + 16 > b.p0 ? page_of(a, b.seq, max(p, b.p0)) : -1;
    }
}
/* Element of position 0, dim 0 of a page's head; slot of a position. */
__device__ __forceinline__ size_t head_at(const PagedArgs &a, int page, uint32_t h) {
    return (((size_t)page * a.kv_heads + h) * a.head_dim) << a.shift;
}
__device__ __forceinline__ size_t scales_at(const PagedArgs &a, int page, uint32_t h) {
    return (((size_t)page * a.kv_heads + h) * a.nb) << a.shift;
}

/* Dims d .. d + 3 of a head row, rotated (smq_rope_kv's products and order). */
__device__ __forceinline__ f4 rotated(f4 x, uint32_t d, uint32_t pairs, const float *c, const float *s) {
#pragma unroll
    for (uint32_t e = 0; e < 4; e += 2) {
        const uint32_t i = (d + e) / 2;
        if (i >= pairs) continue;
        const float p = x[e], q = x[e + 1];
        const float pc = p * c[i], qs = q * s[i], ps = p * s[i], qc = q * c[i];
        x[e] = pc - qs;
        x[e + 1] = ps + qc;
    }
    return x;
}

template <uint32_t TYPE>
struct Four; /* four elements as the cache holds them */
template <>
struct Four<0> {
    typedef f4 T;
};
template <>
struct Four<1> {
    typedef uint32_t T __attribute__((ext_vector_type(2)));
};
template <>
struct Four<2> {
    typedef uint32_t T;
};

/* Four values to elements; Q8: eight lanes hold a 32-wide block (values past head_dim are 0), whose scale comes back.
 * bad: a value that is not finite there (the block's, for Q8). */
template <uint32_t TYPE>
__device__ __forceinline__ typename Four<TYPE>::T encode(f4 x, float &scale, bool &bad) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bad = bad || !(fabsf(x[e]) <= FLT_MAX);
        m = fmaxf(m, fabsf(x[e]));
    }
    if constexpr (TYPE == 0) {
        return x;
    } else if constexpr (TYPE == 1) {
        union {
            h4 h;
            typename Four<1>::T u;
        } r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r.h[e] = (_Float16)x[e];
            bad = bad || !(fabsf((float)r.h[e]) <= FLT_MAX);
        }
        return r.u;
    } else {
        int any = bad;
#pragma unroll
        for (int off = 1; off < 8; off *= 2) {
            m = fmaxf(m, __shfl_xor(m, off));
            any |= __shfl_xor(any, off);
        }
        bad = any;
        scale = any ? __builtin_nanf("") : m / 127.0f;
        const float inv = !any && scale >= FLT_MIN ? 1.0f / scale : 0.0f;
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p = __builtin_rintf(any ? 0.0f : x[e] * inv);
            r |= ((uint32_t)(int)fminf(fmaxf(p, -127.0f), 127.0f) & 255u) << (8 * e);
        }
        return r;
    }
}

/* First two workgroups per block and KV head, one its keys, one its values: up to ST_POS positions, four dims a thread,
 * the loads of four passes at once; values are turned through LDS so that a dim's positions are written together (one or
 * two positions: straight, element by element). Then a workgroup per row of q (all heads): they hold nothing up, the
 * blocks' chains of loads come first.
 *
 * Bound by the launch and three round trips (batch, page ids, rows) for a decode step: 4.7 us for 48 tokens of 2 KV heads of
 * 64; by bytes for chunks: 4 prompts of up to 700 tokens, 12 heads on 2 of 128, f16, 10.4 us (keys and values in one
 * workgroup, one pass after another: 5 us longer). */
constexpr uint32_t ST_PASSES = 4;
template <uint32_t TYPE>
__global__ __launch_bounds__(ST_WG) void k_paged_store(PagedArgs a, const float *q, float *q_out, const float *k,
                                                       const float *v, const float *cs, const float *sn, uint32_t kv_groups) {
    typedef typename Four<TYPE>::T T;
    constexpr uint32_t EB = sizeof(T) / 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char turn[]; /* [head_dim][ST_POS * EB + 4] */
    const uint32_t tid = threadIdx.x, hd = a.head_dim;
    if (blockIdx.x == 0) check_begin(a, tid, ST_WG);
    if (blockIdx.x >= kv_groups) {
        uint32_t s, pos;
        const uint32_t r = blockIdx.x - kv_groups;
        if (!place_of(a, r, s, pos)) return;
        const float *c = cs + (size_t)pos * a.pairs, *sr = sn + (size_t)pos * a.pairs;
        const size_t row = (size_t)r * a.heads * hd;
#pragma unroll 2
        for (uint32_t i = tid; i < a.heads * hd / 4; i += ST_WG)
            *(f4u *)(q_out + row + 4 * i) = rotated(*(const f4u *)(q + row + 4 * i), 4 * i % hd, a.pairs, c, sr);
        return;
    }
    const uint32_t kind = blockIdx.x & 1, x = blockIdx.x >> 1, h = x % a.kv_heads; /* kind 0: keys, 1: values */
    Block b;
    if (!find_block(a, x / a.kv_heads, b)) return;
    int page[2];
    block_pages(a, b, page);
    const uint32_t P = 1u << a.shift, lanes = a.nb * 8, n = b.p1 - b.p0; /* lanes of a row: whole 32-wide blocks */
    const bool few = n <= 2;
    const float *from = kind ? v : k;
    for (uint32_t i0 = tid; i0 < (n * lanes + ST_WG - 1) / ST_WG * ST_WG; i0 += ST_PASSES * ST_WG) { /* whole waves: encode shuffles */
        f4 y[ST_PASSES];
#pragma unroll
        for (uint32_t u = 0; u < ST_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG, j = i / lanes, d = 4 * (i - j * lanes);
            y[u] = f4{};
            if (j < n && d < hd) y[u] = *(const f4u *)(from + ((size_t)(b.row + (int)(b.p0 + j)) * a.kv_heads + h) * hd + d);
        }
#pragma unroll
        for (uint32_t u = 0; u < ST_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG, j = i / lanes, d = 4 * (i - j * lanes), pos = b.p0 + j, slot = pos & (P - 1);
            const int pg = pos & 16 ? page[1] : page[0];
            const bool in = j < n && d < hd;
            if (!kind && in) y[u] = rotated(y[u], d, a.pairs, cs + (size_t)pos * a.pairs, sn + (size_t)pos * a.pairs);
            float scale;
            bool bad = false;
            const T t = encode<TYPE>(y[u], scale, bad);
            if (!in || pg < 0) continue;
            if (bad) *a.flag = 1;
            if (TYPE == 2 && d % 32 == 0) (kind ? a.vs : a.ks)[scales_at(a, pg, h) + ((size_t)(d / 32) << a.shift) + slot] = scale;
            if (!kind) {
                *(T *)((unsigned char *)a.keys + (head_at(a, pg, h) + (size_t)slot * hd + d) * EB) = t;
            } else {
                unsigned char *to = few ? (unsigned char *)a.values + (head_at(a, pg, h) + ((size_t)d << a.shift) + slot) * EB
                                        : turn + d * (ST_POS * EB + 4) + (pos % ST_POS) * EB;
                const size_t step = few ? (size_t)EB << a.shift : ST_POS * EB + 4;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    if constexpr (TYPE == 0) *(float *)(to + e * step) = t[e];
                    else if constexpr (TYPE == 1) *(uint16_t *)(to + e * step) = (uint16_t)(t[e / 2] >> (16 * (e & 1)));
                    else *(to + e * step) = (unsigned char)(t >> (8 * e));
                }
            }
        }
    }
    if (few || !kind) return;
    __syncthreads();
    for (uint32_t i = tid; i < hd * (ST_POS / 4); i += ST_WG) { /* four positions of a dim */
        const uint32_t d = i / (ST_POS / 4), j = 4 * (i % (ST_POS / 4)), pos = b.p0 / ST_POS * ST_POS + j;
        const int pg = j & 16 ? page[1] : page[0];
        if (pg < 0 || pos >= b.p1 || pos + 4 <= b.p0) continue;
        const unsigned char *t = turn + d * (ST_POS * EB + 4) + j * EB;
        unsigned char *to = (unsigned char *)a.values + (head_at(a, pg, h) + ((size_t)d << a.shift) + (pos & (P - 1))) * EB;
        if (pos >= b.p0 && pos + 4 <= b.p1) {
            union {
                uint32_t u[EB];
                T t;
            } y;
#pragma unroll
            for (uint32_t w = 0; w < EB; ++w) y.u[w] = ((const uint32_t *)t)[w];
            *(T *)to = y.t;
        } else {
            for (uint32_t e = 0; e < 4; ++e)
                if (pos + e >= b.p0 && pos + e < b.p1) {
                    if constexpr (TYPE == 0) ((uint32_t *)to)[e] = ((const uint32_t *)t)[e];
                    else if constexpr (TYPE == 1) ((uint16_t *)to)[e] = ((const uint16_t *)t)[e];
                    else to[e] = t[e];
                }
        }
    }
}

template <uint32_t TYPE>
__device__ __forceinline__ f4 decode(typename Four<TYPE>::T t) {
    f4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (TYPE == 0) {
            r[e] = t[e];
        } else if constexpr (TYPE == 1) {
            union {
                uint16_t u;
                _Float16 h;
            } y = {(uint16_t)(t[e / 2] >> (16 * (e & 1)))};
            r[e] = (float)y.h;
        } else {
            r[e] = (float)(int8_t)(t >> (8 * e));
        }
    }
    return r;
}

/* A workgroup per block and KV head: keys four dims a thread, values four positions of a dim a thread, turned through LDS.
 * A block has as many of the ones as of the others; both are requested together, RD_PASSES of them at once (heads of 128
 * have four: all at once took 182 us below, one after another 145). The results are stored past the caches, which they
 * would fill: the pages stay there.
 *
 * Bound by bytes: 8 Q8 sequences at up to 8100, 8 KV heads of 128, 553 MB, 140 us, 3.9 TB/s, where a large copy reaches 4.9;
 * a fifth of it is read and the rest written. A wave per position: 370 us. */
constexpr uint32_t RD_PASSES = 2;
template <uint32_t TYPE>
__global__ __launch_bounds__(ST_WG) void k_paged_read(PagedArgs a, float *keys, float *values) {
    typedef typename Four<TYPE>::T T;
    constexpr uint32_t EB = sizeof(T) / 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    float *turn = (float *)lds; /* [ST_POS][head_dim + 4] */
    const uint32_t tid = threadIdx.x, hd = a.head_dim, h = blockIdx.x % a.kv_heads, P = 1u << a.shift, q = hd / 4;
    if (blockIdx.x == 0) check_begin(a, tid, ST_WG);
    Block b;
    if (!find_block(a, blockIdx.x / a.kv_heads, b)) return;
    int page[2];
    block_pages(a, b, page);
    const uint32_t base = b.p0 / ST_POS * ST_POS, first = base & (P - 1);
    const float inv = 1.0f / (float)q;
    auto row_of = [&](uint32_t i) { return (uint32_t)(((float)i + 0.5f) * inv); }; /* i / q: i is below 2^12, where this is exact */
    auto holds = [&](uint32_t j) { return base + j >= b.p0 && base + j < b.p1 && page[j >> 4] >= 0; };
    /* the block's two halves, from position 0 of the page on; in one page the second begins where the first ends */
    const unsigned char *kp[2], *vp[2];
    const float *kw[2], *vw[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int pg = max(page[x], 0);
        const uint32_t slot = (first + 16 * x & (P - 1)) - 16 * x; /* of the half's position j, less j */
        kp[x] = (const unsigned char *)a.keys + (head_at(a, pg, h) + (ptrdiff_t)(int)slot * hd) * EB;
        vp[x] = (const unsigned char *)a.values + (head_at(a, pg, h) + (ptrdiff_t)(int)slot) * EB;
        kw[x] = a.ks + scales_at(a, pg, h) + (ptrdiff_t)(int)slot;
        vw[x] = a.vs + scales_at(a, pg, h) + (ptrdiff_t)(int)slot;
    }
    const ptrdiff_t row0 = ((ptrdiff_t)(b.row + (int)base) * a.kv_heads + h) * hd;
    const uint32_t step = a.kv_heads * hd; /* of the rows */
    for (uint32_t i0 = tid; i0 < hd * (ST_POS / 4); i0 += RD_PASSES * ST_WG) {
        T tv[RD_PASSES], tk[RD_PASSES];
        f4 wv[RD_PASSES];
        float wk[RD_PASSES];
#pragma unroll
        for (uint32_t u = 0; u < RD_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG;
            if (i >= hd * (ST_POS / 4)) continue;
            const uint32_t dv = i / (ST_POS / 4), jv = 4 * (i % (ST_POS / 4)), jk = row_of(i), dk = 4 * (i - jk * q);
            if (page[jv >> 4] >= 0) {
                tv[u] = *(const T *)(vp[jv >> 4] + ((dv << a.shift) + jv) * EB);
                if constexpr (TYPE == 2) wv[u] = *(const f4 *)(vw[jv >> 4] + (dv / 32 << a.shift) + jv);
            }
            if (holds(jk)) {
                tk[u] = *(const T *)(kp[jk >> 4] + (jk * hd + dk) * EB);
                if constexpr (TYPE == 2) wk[u] = kw[jk >> 4][(dk / 32 << a.shift) + jk];
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < RD_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG;
            if (i >= hd * (ST_POS / 4)) continue;
            const uint32_t dv = i / (ST_POS / 4), jv = 4 * (i % (ST_POS / 4)), jk = row_of(i), dk = 4 * (i - jk * q);
            if (page[jv >> 4] >= 0) {
                f4 y = decode<TYPE>(tv[u]);
                if constexpr (TYPE == 2) y *= wv[u];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) turn[(jv + e) * (hd + 4) + dv] = y[e];
            }
            if (holds(jk)) {
                f4 y = decode<TYPE>(tk[u]);
                if constexpr (TYPE == 2) y *= wk[u];
                __builtin_nontemporal_store(y, (f4u *)(keys + row0 + (ptrdiff_t)(jk * step + dk)));
            }
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i < hd * (ST_POS / 4); i += ST_WG) {
        const uint32_t j = row_of(i), d = 4 * (i - j * q);
        if (holds(j))
            __builtin_nontemporal_store(*(const f4 *)&turn[j * (hd + 4) + d], (f4u *)(values + row0 + (ptrdiff_t)(j * step + d)));
    }
}

/* Joins what several workgroups have of a tile and KV head: the weights of their maxima, in their order. head_dim / 4 lanes
 * per row. A lane requests its part of O and the maxima and sums of eight workgroups at once: after the tile's four words
 * one round trip to memory joins up to eight. 4 to 6 us, a launch and two round trips. */
constexpr uint32_t JOIN_WG = 256, JOIN_AT_ONCE = 8;
__global__ __launch_bounds__(JOIN_WG) void k_paged_join(PagedArgs a, float *att, AttendPlan p, const i4 *used,
                                                        const float *part) {
    const uint32_t hd = a.head_dim, lanes = hd / 4, per = JOIN_WG / lanes;
    const uint32_t groups = (p.tile_rows + per - 1) / per, tile = blockIdx.x / groups, kh = tile % a.kv_heads;
    const uint32_t r = blockIdx.x % groups * per + threadIdx.x / lanes, d = 4 * (threadIdx.x % lanes);
    const i4 u = used[tile];
    const uint32_t parts = (uint32_t)u[0] & 0xffff, n = (uint32_t)u[0] >> 16, slot = (uint32_t)u[3];
    if (parts < 2 || r >= n || threadIdx.x / lanes >= per) return;
    const f2 *pml = (const f2 *)(part + (size_t)p.pieces * a.kv_heads * p.tile_rows * hd);
    float m = -FLT_MAX, l = 0.0f;
    const float share = (float)(32 - __builtin_clz(parts)); /* of 2^-share each: their sum stays below the values */
    f4 o = {};
    for (uint32_t i0 = 0; i0 < parts; i0 += JOIN_AT_ONCE) {
        f2 ml[JOIN_AT_ONCE];
        f4 x[JOIN_AT_ONCE];
        float top = m;
#pragma unroll
        for (uint32_t i = 0; i < JOIN_AT_ONCE; ++i) {
            const size_t y = ((size_t)(slot + min(i0 + i, parts - 1)) * a.kv_heads + kh) * p.tile_rows + r;
            ml[i] = pml[y];
            x[i] = *(const f4 *)(part + y * hd + d);
        }
#pragma unroll
        for (uint32_t i = 0; i < JOIN_AT_ONCE; ++i) top = fmaxf(top, ml[i][0]);
        const float old = __builtin_amdgcn_exp2f(m - top);
        l *= old;
        o *= old;
        m = top;
#pragma unroll
        for (uint32_t i = 0; i < JOIN_AT_ONCE; ++i) {
            const float e = i0 + i < parts ? __builtin_amdgcn_exp2f(ml[i][0] - m - share) : 0.0f;
            l += e * ml[i][1];
            o += e * x[i];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *(f4u *)(att + row_at(a, u[1], kh, (uint32_t)u[2] + r) + d) = o * inv;
}

/* The pieces that tiles of so many rows are cut into: two a CU for products and for decoding heads of up to 64 (8 KiB of f16
 * a step and wave), one a CU for wider ones (one f16 sequence at 16384, 8 KV heads of 128: 22 us, two a CU 25); by_piece has
 * what becomes of these numbers.
 *
 * Cutting costs partial results and a second launch, which joins them. No cuts
 * - where the longest tile exceeds an equal share by about 24 steps or less (64 sequences at 700, 2 KV heads of 64: 11.8 us
 *   whole, 15.4 cut; 8 with a window of 1024, 4 KV heads of 64: 22 whole, 13 cut);
 * - where tiles that waves own, which keep two workgroups a CU busy, are 512 or more (2048 tokens of 8 KV heads of 128, 512
 *   tiles, from an empty cache: 100 us whole, 115 cut). Between one and two a CU some CUs have twice the others' work: cut
 *   unless the tiles' mean is short (2 x 800 tokens at 4000, 8 KV heads of 128: 260 us whole, 210 cut). */
AttendPlan plan_tiles(const PagedArgs &a, size_t ws_bytes, uint32_t tile_rows) {
    AttendPlan p;
    const uint32_t G = a.heads / a.kv_heads;
    const uint64_t rows = (uint64_t)a.tokens * G, seqs = a.seqs < a.tokens ? a.seqs : a.tokens;
    p.owns = tile_rows > 16;
    p.tile_rows = tile_rows;
    p.row_shift = p.tile_rows == 128 ? 7 : p.tile_rows == 64 ? 6 : 4;
    p.tiles = (uint32_t)((rows + seqs * (p.tile_rows - 1)) >> p.row_shift);
    const uint32_t groups = p.owns || a.head_dim <= 64 ? 512 : 256;
    p.stream = (groups + a.kv_heads - 1) / a.kv_heads;
    p.tile_tokens = p.tile_rows / G + 1;
    p.fixed = 64 * (PA_FIXED + 1);
    uint64_t most = a.limit + PA_STEP; /* positions of a tile's steps */
    if (a.window) {
        const uint64_t w = (uint64_t)a.window + a.sinks + p.tile_tokens + 2 * PA_STEP;
        most = w < most ? w : most;
    }
    most = 2 * most + p.fixed;
    p.unit = 0; /* all units and the last workgroup's end below 2^31 */
    while (((uint64_t)(p.tiles + 512) * ((most >> p.unit) + 1)) >= 1u << 30) ++p.unit;
    p.cw = (uint32_t)(most >> p.unit) + 1;
    p.c1 = 2 * p.tile_rows / G >> p.unit;
    /* tiles of an even batch, the steps of the longest and of the mean */
    const uint64_t tiles = seqs * ((rows / (seqs ? seqs : 1) + p.tile_rows - 1) >> p.row_shift) * a.kv_heads;
    const uint64_t steps = (most - p.fixed) / 2 / PA_STEP;
    if (p.owns && tiles > 256) {
        const uint64_t average = steps - (a.window ? 0 : min(rows / G / seqs / 64, steps / 2));
        if (tiles >= 512 || average * (512 - tiles) / 256 <= 24) p.stream = 0;
    } else if (tiles >= groups || steps * (groups - tiles) / groups <= 24) {
        p.stream = 0;
    }
    const size_t used = attend_used_bytes(a, p), each = attend_piece_bytes(a, p.tile_rows);
    const uint64_t room = ws_bytes > used ? (ws_bytes - used) / each : 0;
    auto pieces = [&](uint64_t aim) { return max(aim, (aim + 1) / 2 + p.tiles); }; /* at most: see by_piece */
    const uint64_t longest = p.owns ? 2 * p.tiles > p.stream ? p.stream + p.tiles : 0
                                    : p.tiles * most / (PA_LONG * 64); /* no fewer than by_piece has, growing with `most` */
    p.most = (uint32_t)max((uint64_t)p.stream, min(longest, (uint64_t)3 * p.stream));
    if (room < pieces(p.most)) p.most = p.stream;
    if (room < pieces(p.stream)) p.most = p.stream = room > p.tiles ? (uint32_t)min(room, 2 * (room - p.tiles)) : 0;
    p.pieces = p.stream ? (uint32_t)pieces(p.most) : 0;
    return p;
}

/* Up to 32 rows a sequence and KV head on average (decoding) the tiles have 16 rows; above, a workgroup's waves own theirs,
 * 16 or 32 each. 32 where tiles are cut or many: a fragment read serves twice. Few whole tiles take as long as the longest
 * one's chain of steps, and a step of half the rows is shorter (2048 tokens from an empty cache, f16, 8 KV heads of 64: 71
 * us, 58; 1024 of 128: 51, 40; but 2048 of 128: 100, 104). */
AttendPlan attend_plan(const PagedArgs &a, size_t ws_bytes) {
    const uint32_t ks = attend_ks(a.head_dim);
    const uint64_t rows = (uint64_t)a.tokens * (a.heads / a.kv_heads), seqs = a.seqs < a.tokens ? a.seqs : a.tokens;
    if (rows <= 32 * seqs) return plan_tiles(a, ws_bytes, 16);
    const AttendPlan p = plan_tiles(a, ws_bytes, 64 * attend_rt(ks));
    return p.stream || p.tile_rows == 64 || rows / 128 * a.kv_heads * ks >= 2048 ? p : plan_tiles(a, 0, 64);
}

}  // namespace

#define SMQ_PAGED(KERNEL, GRID, BLOCK, LDS, ...)                                                          \
    do {                                                                                             \
        if (a.type == 0) hipLaunchKernelGGL((KERNEL<0>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);         \
        else if (a.type == 1) hipLaunchKernelGGL((KERNEL<1>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);    \
        else hipLaunchKernelGGL((KERNEL<2>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);                     \
    } while (0)

hipError_t launch_paged_rope_kv(const PagedArgs &a, const float *q, float *q_out, const float *k, const float *v,
                                const float *cs, const float *sn, hipStream_t s) {
    const uint32_t kv_groups = 2 * most_blocks(a) * a.kv_heads;
    SMQ_PAGED(k_paged_store, dim3((q ? a.tokens : 0) + kv_groups), dim3(ST_WG),
              a.head_dim * (ST_POS * (4u >> a.type) + 4), q, q_out, k, v, cs, sn, kv_groups);
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedArgs &a, float *keys, float *values, hipStream_t s) {
    SMQ_PAGED(k_paged_read, dim3(most_blocks(a) * a.kv_heads), dim3(ST_WG), ST_POS * (a.head_dim + 4) * 4, keys, values);
    return hipGetLastError();
}

size_t paged_attention_workspace(const PagedArgs &given) {
    PagedArgs a = given;
    a.sinks = a.limit; /* the call brings them: a plan of more positions needs no fewer bytes, up to all of the context's */
    const AttendPlan p = attend_plan(a, ~(size_t)0);
    return p.stream ? attend_used_bytes(a, p) + p.pieces * attend_piece_bytes(a, p.tile_rows) : 0;
}

hipError_t launch_paged_attention(const PagedArgs &a, const float *q, float *att, void *ws, size_t ws_bytes,
                                  hipStream_t s) {
    const AttendPlan p = attend_plan(a, ws_bytes);
    i4 *used = p.stream ? (i4 *)ws : nullptr;
    float *part = p.stream ? (float *)((char *)ws + attend_used_bytes(a, p)) : nullptr;
    hipError_t e = a.type == 0 ? launch_attend<0>(a, p, q, att, used, part, s)
                 : a.type == 1 ? launch_attend<1>(a, p, q, att, used, part, s)
                               : launch_attend<2>(a, p, q, att, used, part, s);
    if (e != hipSuccess || !p.stream) return e;
    const uint32_t per = JOIN_WG / (a.head_dim / 4), groups = (p.tile_rows + per - 1) / per;
    hipLaunchKernelGGL(k_paged_join, dim3(a.kv_heads * p.tiles * groups), dim3(JOIN_WG), 0, s, a, att, p, used, part);
    return hipGetLastError();
}

}  // namespace smq
