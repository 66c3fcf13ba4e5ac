/* Paged KV cache on gfx950: RoPE and the store of new tokens (f32, f16, Q8), rows read back, and the attention of a
 * ragged batch of new tokens over the pages (include/smq.h has the layout of a page). */
#include <cmath>

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

/* Two dims rotated by a cosine and a sine (smq_rope_kv's products and order). */
__device__ __forceinline__ void turn_pair(float &p, float &q, float c, float s) {
    const float pc = p * c, qs = q * s, ps = p * s, qc = q * c;
    p = pc - qs;
    q = ps + qc;
}
/* Dims d .. d + 3 of a head row, rotated. */
__device__ __forceinline__ f4 rotated(f4 x, uint32_t d, uint32_t pairs, const float *c, const float *s) {
#pragma unroll
    for (uint32_t e = 0; e < 4; e += 2) {
        const uint32_t i = (d + e) / 2;
        if (i >= pairs) continue;
        float p = x[e], q = x[e + 1];
        turn_pair(p, q, c[i], s[i]);
        x[e] = p;
        x[e + 1] = q;
    }
    return x;
}

/* The lanes of a head's RMSNorm, four dims each: a power of two, so that they lie in one wave. */
__device__ __forceinline__ uint32_t norm_lanes(const PagedArgs &a) {
    return a.head_dim <= 32 ? 8 : a.head_dim <= 64 ? 16 : a.head_dim <= 128 ? 32 : 64;
}
template <int CTRL>
__device__ __forceinline__ double lane_add(double x) { /* x and the lane's that CTRL names */
    const int lo = __builtin_amdgcn_mov_dpp(__double2loint(x), CTRL, 0xf, 0xf, false),
              hi = __builtin_amdgcn_mov_dpp(__double2hiint(x), CTRL, 0xf, 0xf, false);
    return x + __hiloint2double(hi, lo);
}
template <int CTRL>
__device__ __forceinline__ float lane_of_four(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, false));
}
/* Four heads' dims d .. d + 3 (0 past the head), each head in `lanes` lanes, normed by g, their part of the norm. The sum of
 * squares, whose products are exact, the root and the quotient in 64 bits: no order of the sum shows in the f32 quotient, and the
 * bits are the same whichever lanes hold the head; the two products round to f32 as the formula has them. Roots and quotients,
 * about 40 instructions on 64 bits, one for the four heads: a lane of four does that of one. */
__device__ __forceinline__ void normed(f4 (&x)[4], f4 g, const PagedArgs &a, uint32_t lanes, float eps) {
    double sum[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        sum[u] = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[u] = __builtin_fma((double)x[u][e], (double)x[u][e], sum[u]);
        sum[u] = lane_add<0xB1>(sum[u]); /* the other of two, the other two of four, four of eight (mirrored, they are alike) */
        sum[u] = lane_add<0x4E>(sum[u]);
        sum[u] = lane_add<0x141>(sum[u]);
        if (lanes > 8) sum[u] = lane_add<0x140>(sum[u]);
        if (lanes > 16) sum[u] += __shfl_xor(sum[u], 16);
        if (lanes > 32) sum[u] += __shfl_xor(sum[u], 32);
    }
    const uint32_t k = threadIdx.x & 3;
    const double mean = (k & 2 ? k & 1 ? sum[3] : sum[2] : k & 1 ? sum[1] : sum[0]) / (double)a.head_dim;
    const float own = (float)(1.0 / sqrt(mean + (double)eps));
    const float inv[4] = {lane_of_four<0x00>(own), lane_of_four<0x55>(own), lane_of_four<0xAA>(own), lane_of_four<0xFF>(own)};
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = x[u][e] * inv[u];
            x[u][e] = y * g[e];
        }
}
/* The rotary position of a token whose sequence's new tokens begin at position first; false, with the flag, where the tables have none. */
__device__ __forceinline__ bool own_turn(const PagedArgs &a, int first, int depth, uint32_t &at) {
    const int64_t p = (int64_t)first + depth;
    if (p < 0 || p >= (int64_t)a.context) {
        *a.flag = 1;
        return false;
    }
    at = (uint32_t)p;
    return true;
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
 * workgroup, one pass after another: 5 us longer).
 *
 * NORM: rows with strides, heads normed before their rotation, rotary positions of the tokens' own. 5400 f16 tokens of 32 heads
 * on 8 of 128 49 us, 4.5 TB/s, a fifth of the issue the norms' 64-bit sums, roots and quotients (a root for each head: 53; heads
 * one after another: 77); 32 x 8 Q8 drafts of 14 heads on 2 of 64 6.1. */
constexpr uint32_t ST_PASSES = 4, ST_HEADS = 4;
template <uint32_t TYPE, bool NORM>
__global__ __launch_bounds__(ST_WG) void k_paged_store(PagedArgs a, RowArgs w, const float *cs, const float *sn,
                                                       uint32_t kv_groups) {
    typedef typename Four<TYPE>::T T;
    constexpr uint32_t EB = sizeof(T) / 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char turn[]; /* [head_dim][ST_POS * EB + 4] */
    const uint32_t tid = threadIdx.x, hd = a.head_dim;
    if (blockIdx.x == 0) check_begin(a, tid, ST_WG);
    if (blockIdx.x >= kv_groups) {
        uint32_t s, pos;
        const uint32_t r = blockIdx.x - kv_groups;
        if (!place_of(a, r, s, pos)) return;
        if constexpr (NORM) {
            uint32_t turn_at = pos;
            if (w.depth && !own_turn(a, (int)pos - (int)(r - (uint32_t)a.begin[s]), w.depth[r], turn_at)) return;
            /* a thread has the same dims of several heads: their norm, cosines and sines once, the heads requested together */
            const uint32_t lanes = norm_lanes(a), d = 4 * (tid % lanes), per = ST_WG / lanes;
            const size_t at = (size_t)turn_at * a.pairs;
            f4 g = {};
            f2 c = {}, sr = {};
            if (w.q_norm && d < hd) g = *(const f4u *)(w.q_norm + d);
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e)
                if (d / 2 + e < a.pairs) {
                    c[e] = cs[at + d / 2 + e];
                    sr[e] = sn[at + d / 2 + e];
                }
            const float *from = w.q + r * w.q_stride + d;
            float *to = w.q_out + r * w.q_out_stride + d;
            for (uint32_t h0 = tid / lanes; h0 < a.heads + tid / lanes; h0 += ST_HEADS * per) { /* uniform: the norm's sums shuffle */
                f4 x[ST_HEADS];
#pragma unroll
                for (uint32_t u = 0; u < ST_HEADS; ++u) {
                    x[u] = f4{};
                    if (h0 + u * per < a.heads && d < hd) x[u] = *(const f4u *)(from + (h0 + u * per) * hd);
                }
                if (w.q_norm) normed(x, g, a, lanes, w.eps);
#pragma unroll
                for (uint32_t u = 0; u < ST_HEADS; ++u) {
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        float y = x[u][2 * e], z = x[u][2 * e + 1];
                        if (d / 2 + e < a.pairs) turn_pair(y, z, c[e], sr[e]);
                        x[u][2 * e] = y;
                        x[u][2 * e + 1] = z;
                    }
                    if (h0 + u * per < a.heads && d < hd) *(f4u *)(to + (h0 + u * per) * hd) = x[u];
                }
            }
            return;
        }
        const float *c = cs + (size_t)pos * a.pairs, *sr = sn + (size_t)pos * a.pairs;
        const size_t row = (size_t)r * a.heads * hd;
#pragma unroll 2
        for (uint32_t i = tid; i < a.heads * hd / 4; i += ST_WG)
            *(f4u *)(w.q_out + row + 4 * i) = rotated(*(const f4u *)(w.q + row + 4 * i), 4 * i % hd, a.pairs, c, sr);
        return;
    }
    const uint32_t kind = blockIdx.x & 1, x = blockIdx.x >> 1, h = x % a.kv_heads; /* kind 0: keys, 1: values */
    Block b;
    if (!find_block(a, x / a.kv_heads, b)) return;
    int page[2];
    block_pages(a, b, page);
    /* lanes of a row: whole 32-wide blocks */
    const uint32_t P = 1u << a.shift, lanes = NORM ? norm_lanes(a) : a.nb * 8, n = b.p1 - b.p0;
    const bool few = n <= 2;
    const float *from = kind ? w.v : w.k;
    const size_t stride = NORM ? kind ? w.v_stride : w.k_stride : (size_t)a.kv_heads * hd;
    const int first = NORM && w.depth ? a.begin[b.seq] - b.row : 0;
    f4 g = {}; /* a thread's dims are the same in every pass */
    if (NORM && !kind && w.k_norm && 4 * (tid % lanes) < hd) g = *(const f4u *)(w.k_norm + 4 * (tid % lanes));
    for (uint32_t i0 = tid; i0 < (n * lanes + ST_WG - 1) / ST_WG * ST_WG; i0 += ST_PASSES * ST_WG) { /* whole waves: encode shuffles */
        f4 y[ST_PASSES];
#pragma unroll
        for (uint32_t u = 0; u < ST_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG, j = i / lanes, d = 4 * (i - j * lanes);
            y[u] = f4{};
            if (j < n && d < hd) y[u] = *(const f4u *)(from + (size_t)(b.row + (int)(b.p0 + j)) * stride + h * hd + d);
        }
        if constexpr (NORM) {
            if (!kind && w.k_norm) normed(y, g, a, lanes, w.eps);
        }
#pragma unroll
        for (uint32_t u = 0; u < ST_PASSES; ++u) {
            const uint32_t i = i0 + u * ST_WG, j = i / lanes, d = 4 * (i - j * lanes), pos = b.p0 + j, slot = pos & (P - 1);
            const int pg = pos & 16 ? page[1] : page[0];
            bool in = j < n && d < hd;
            uint32_t at = pos;
            if constexpr (NORM) {
                if (!kind) {
                    if (in && w.depth && !own_turn(a, first, w.depth[b.row + (int)pos], at)) {
                        in = false;
                        y[u] = f4{};
                    }
                }
            }
            if (!kind && in) y[u] = rotated(y[u], d, a.pairs, cs + (size_t)at * a.pairs, sn + (size_t)at * a.pairs);
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
 * what becomes of these numbers. Three a CU for products of trees whose registers leave room (tiles of 64
 * rows, 32 heads on 8, 8 drafts of 63 at 8000: heads of 64 f16 104 -> 71 us, Q8 178 -> 105, f32 391 -> 225, of 128 f16 176 ->
 * 115, Q8 304 -> 168; 24 of 8 at 3001, heads of 128: 60 -> 52, 80 -> 58).
 *
 * Cutting costs partial results and a second launch, which joins them. No cuts
 * - where the longest tile exceeds an equal share by about 24 steps or less (64 sequences at 700, 2 KV heads of 64: 11.8 us
 *   whole, 15.4 cut; 8 with a window of 1024, 4 KV heads of 64: 22 whole, 13 cut), 10 where waves own a tree's rows (24
 *   drafts of 40 Q8 tokens at 700, 2 KV heads of 128: 46 whole, 40 cut; at 300 27 and 32);
 * - where tiles that waves own, which keep two workgroups a CU busy, are 512 or more (2048 tokens of 8 KV heads of 128, 512
 *   tiles, from an empty cache: 100 us whole, 115 cut). Between one and two a CU some CUs have twice the others' work: cut
 *   unless the tiles' mean is short (2 x 800 tokens at 4000, 8 KV heads of 128: 260 us whole, 210 cut). A tree's tiles with
 *   three a CU are cut up to 768 of them, f16 ones, which stay ahead whole for longer, from 72 steps beside an equal share on
 *   (96 dims, 525 tiles of 29 steps 35 us whole, 53 cut; 528 of 220 steps 220 and 166). Heads above 96: f16
 *   ones gain nothing where two a CU are full (64 drafts of 8 at 4096, 32 heads on 8 of 128, 512 tiles: 181 whole, 197 cut; at
 *   16384 680 and 684; but 35 of 15 at 7803, 8 heads of 128, 280 tiles, 292 and 166). Q8 ones do, from 36 steps on (64 of 8 at
 *   4096 223 whole, 180 cut; at 16384 852 and 641; 24 of 40 at 3001 198 and 157; but 290 of 62 at 1538, 2 heads of 112, 116
 *   and 123), from 116 where tiles have few rows, whose steps leave the CU to others (170 of 27 at 5665, 4 heads of 128, 310
 *   whole, 339 cut; but 64 of 7 at 4987, 8 heads, 219 and 186). */
AttendPlan plan_tiles(const PagedArgs &a, size_t ws_bytes, uint32_t tile_rows, bool tree) {
    AttendPlan p;
    const uint32_t G = a.heads / a.kv_heads;
    const uint64_t rows = (uint64_t)a.tokens * G, seqs = a.seqs < a.tokens ? a.seqs : a.tokens;
    p.owns = tile_rows > 16;
    p.tile_rows = tile_rows;
    p.row_shift = p.tile_rows == 128 ? 7 : p.tile_rows == 64 ? 6 : 4;
    p.tiles = (uint32_t)((rows + seqs * (p.tile_rows - 1)) >> p.row_shift);
    const uint32_t ks = attend_ks(a.head_dim);
    const bool three = tree && p.owns && ks <= 4 && tree_waves(a.type, ks, tile_rows / 64) == 3;
    const uint32_t groups = three ? 768 : p.owns || a.head_dim <= 64 ? 512 : 256;
    p.stream = (groups + a.kv_heads - 1) / a.kv_heads;
    p.tile_tokens = tree ? a.tokens : p.tile_rows / G + 1; /* a tree's tile goes over all new tokens of its sequence */
    p.fixed = 64 * (PA_FIXED + 1);
    uint64_t most = a.limit + PA_STEP; /* positions of a tile's steps */
    if (a.window) {
        const uint64_t w = (uint64_t)a.window + a.sinks + p.tile_tokens + 2 * PA_STEP;
        most = w < most ? w : most;
    }
    most = 2 * most + p.fixed;
    p.unit = 0; /* all units and the last workgroup's end below 2^31 */
    while (((uint64_t)(p.tiles + max(groups, 512u)) * ((most >> p.unit) + 1)) >= 1u << 30) ++p.unit;
    p.cw = (uint32_t)(most >> p.unit) + 1;
    p.c1 = tree ? 0 : 2 * p.tile_rows / G >> p.unit;
    /* tiles of an even batch, the steps of the longest and of the mean */
    const uint64_t tiles = seqs * ((rows / (seqs ? seqs : 1) + p.tile_rows - 1) >> p.row_shift) * a.kv_heads;
    const uint64_t steps = (most - p.fixed) / 2 / PA_STEP;
    if (p.owns && tiles > 256) {
        const uint64_t average = steps - (a.window || tree ? 0 : min(rows / G / seqs / 64, steps / 2));
        /* the longest tile exceeds an equal share of so many workgroups by more than `least` steps */
        auto over = [&](uint32_t full, uint32_t least) { return tiles < full && average * (full - tiles) / 256 > least; };
        const bool few = rows * a.kv_heads <= 32 * tiles; /* half of a tile's waves, or more, have no rows */
        const bool cut = !three       ? over(512, 24)
                         : ks < 4     ? over(768, a.type == 1 ? 72 : 24)
                         : a.type == 1 ? over(512, 24) && over(768, 72)
                                       : over(512, 24) || over(768, few ? 116 : 36);
        if (!cut) p.stream = 0;
    } else if (tiles >= groups || steps * (groups - tiles) / groups <= (tree && p.owns ? 10u : 24u)) {
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

/* A tile's rows for trees, whose tiles all go over the whole context: 16, whose waves share the positions out, 64 or 128, by an
 * estimate of the time (us; the table, q8 and f16 heads of 128 on 2 and 8, 24 drafts of 40, 8 of 16 and 64 of 8). A step of a
 * tile of 16, 64, 128 rows takes 1 / r of the card once tiles fill it; before, tiles of 16 wait for a quarter of their steps
 * one after another (or a piece's, and the join), the others for a piece's steps, the batch and the join.
 *
 *                        16 rows   64   128                            16 rows   64   128
 *   q8  24 x 40 at 300        30   25    25      f16  8 x 16 at  700        19   25    28
 *               at 700        50   36    40                  at 2000        37   31    32
 *               at 3001      126   67    73      f16 64 x  8 at 2000       138   98    98
 *   f16 24 x 40 at 700        47   32    33      f16  8 x 63 at 16384      812  285   239
 *               at 1500       75   37    39      q8   8 x 16 at 1500        18   21    23 (14 heads on 2 of 64)
 *   f32 24 x 40 at 3001      247  157   156      q8  24 x  8 at 3001        98   58    91
 *                                                f32  8 x 16 at 2000        66   52    78 */
uint32_t tree_rows(const PagedArgs &a) {
    const double ks = attend_ks(a.head_dim), rows = (double)a.tokens * (a.heads / a.kv_heads);
    const double seqs = a.seqs < a.tokens ? a.seqs : a.tokens, each = rows / seqs;
    double reach = a.limit;
    if (a.window) reach = min(reach, (double)a.window + a.sinks + a.tokens);
    const double steps = reach / PA_STEP + 1;
    /* Of one 32-wide step, by type, heads of up to 64 first: tiles of 16 rows (and where heads are of 128), of 64, of 128. A
     * tile brings a step (and converts Q8 codes) once, whatever its rows, and then each wave has its part: the tiles' rates
     * and those of their waves' 16 and 32 rows. Fitted to 351 batches and tried on 194 others (profiles/tree_tile_rows.csv): the
     * choice costs 1.8 and 3.1 % of the best tile's time on average, at most 59 % (24 f32 drafts of 16 at 1000) and, for heads
     * above 128 at short contexts, 93 %. */
    static const double rate[2][3][6] = {
        {{1060, 1060, 870, 4050, 1050, 1080}, {2740, 2740, 3140, 12100, 5600, 3850}, {2800, 2800, 1910, 9100, 820, 6280}},
        {{1050, 1070, 710, 5800, 320, 4400}, {2480, 1890, 2190, 52000, 2290, 7560}, {2640, 1880, 3890, 5200, 1800, 2750}}};
    const double *r = rate[ks > 2][a.type], unit = seqs * a.kv_heads * steps * ks;
    const double chain = steps / 4 * (1.0 + 0.19 * ks), fill = unit * ceil(each / 16) / r[ks == 4];
    const double t16 = min(7 + max(chain, fill), 13 + fill);
    const double t64 = 15 + max(unit * (ceil(each / 64) / r[2] + ceil(each / 16) / r[3]), 3.0 * ks);
    const double t128 = 17 + max(unit * (ceil(each / 128) / r[4] + ceil(each / 32) / r[5]), 5.0 * ks);
    const bool wide = attend_rt(attend_ks(a.head_dim)) == 2 && t128 < t64;
    return t16 <= min(t64, t128) ? 16 : wide ? 128 : 64;
}

/* Up to 32 rows a sequence and KV head on average (decoding) the tiles have 16 rows; above, a workgroup's waves own theirs,
 * 16 or 32 each. 32 where tiles are cut or many: a fragment read serves twice. Few whole tiles take as long as the longest
 * one's chain of steps, and a step of half the rows is shorter (2048 tokens from an empty cache, f16, 8 KV heads of 64: 71
 * us, 58; 1024 of 128: 51, 40; but 2048 of 128: 100, 104). */
AttendPlan attend_plan(const PagedArgs &a, size_t ws_bytes, bool tree) {
    const uint32_t ks = attend_ks(a.head_dim);
    const uint64_t rows = (uint64_t)a.tokens * (a.heads / a.kv_heads), seqs = a.seqs < a.tokens ? a.seqs : a.tokens;
    const uint32_t tile = tree ? tree_rows(a) : rows <= 32 * seqs ? 16 : 64 * attend_rt(ks);
    const AttendPlan p = plan_tiles(a, ws_bytes, tile, tree);
    return p.stream || tile <= 64 || rows / 128 * a.kv_heads * ks >= 2048 ? p : plan_tiles(a, 0, 64, tree);
}

}  // namespace

#define SMQ_PAGED(KERNEL, GRID, BLOCK, LDS, ...)                                                          \
    do {                                                                                             \
        if (a.type == 0) hipLaunchKernelGGL((KERNEL<0>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);         \
        else if (a.type == 1) hipLaunchKernelGGL((KERNEL<1>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);    \
        else hipLaunchKernelGGL((KERNEL<2>), GRID, BLOCK, LDS, s, a, __VA_ARGS__);                     \
    } while (0)

template <bool NORM>
hipError_t launch_store(const PagedArgs &a, const RowArgs &r, const float *cs, const float *sn, hipStream_t s) {
    const uint32_t kv_groups = 2 * most_blocks(a) * a.kv_heads, lds = a.head_dim * (ST_POS * (4u >> a.type) + 4);
    const dim3 grid((r.q ? a.tokens : 0) + kv_groups);
    if (a.type == 0) hipLaunchKernelGGL((k_paged_store<0, NORM>), grid, dim3(ST_WG), lds, s, a, r, cs, sn, kv_groups);
    else if (a.type == 1) hipLaunchKernelGGL((k_paged_store<1, NORM>), grid, dim3(ST_WG), lds, s, a, r, cs, sn, kv_groups);
    else hipLaunchKernelGGL((k_paged_store<2, NORM>), grid, dim3(ST_WG), lds, s, a, r, cs, sn, kv_groups);
    return hipGetLastError();
}

hipError_t launch_paged_rope_kv(const PagedArgs &a, const float *q, float *q_out, const float *k, const float *v,
                                const float *cs, const float *sn, hipStream_t s) {
    RowArgs r = {};
    r.q = q;
    r.q_out = q_out;
    r.k = k;
    r.v = v;
    return launch_store<false>(a, r, cs, sn, s);
}

hipError_t launch_paged_norm_rope_kv(const PagedArgs &a, const RowArgs &r, const float *cs, const float *sn, hipStream_t s) {
    return launch_store<true>(a, r, cs, sn, s);
}

hipError_t launch_paged_read(const PagedArgs &a, float *keys, float *values, hipStream_t s) {
    SMQ_PAGED(k_paged_read, dim3(most_blocks(a) * a.kv_heads), dim3(ST_WG), ST_POS * (a.head_dim + 4) * 4, keys, values);
    return hipGetLastError();
}

size_t paged_attention_workspace(const PagedArgs &given, bool tree) {
    PagedArgs a = given;
    a.sinks = a.limit; /* the call brings them: a plan of more positions needs no fewer bytes, up to all of the context's */
    auto bytes = [&](const AttendPlan &p) {
        return p.stream ? attend_used_bytes(a, p) + p.pieces * attend_piece_bytes(a, p.tile_rows) : 0;
    };
    if (!tree) return bytes(attend_plan(a, ~(size_t)0, false));
    size_t most = 0; /* the call brings the cache's type too: any of the tiles, with any type's workgroups a CU */
    for (a.type = 0; a.type <= 2; ++a.type)
        for (uint32_t rows = 16; rows <= 64 * attend_rt(attend_ks(a.head_dim)); rows *= rows == 16 ? 4 : 2)
            most = max(most, bytes(plan_tiles(a, ~(size_t)0, rows, true)));
    return most;
}

hipError_t launch_paged_attention(const PagedArgs &a, const TreeArgs *tree, const float *q, float *att, void *ws,
                                  size_t ws_bytes, hipStream_t s) {
    const AttendPlan p = attend_plan(a, ws_bytes, tree != nullptr);
    i4 *used = p.stream ? (i4 *)ws : nullptr;
    float *part = p.stream ? (float *)((char *)ws + attend_used_bytes(a, p)) : nullptr;
    const TreeArgs t = tree ? *tree : TreeArgs{};
    hipError_t e;
    if (tree)
        e = a.type == 0 ? launch_attend<0, true>(a, t, p, q, att, used, part, s)
          : a.type == 1 ? launch_attend<1, true>(a, t, p, q, att, used, part, s)
                        : launch_attend<2, true>(a, t, p, q, att, used, part, s);
    else
        e = a.type == 0 ? launch_attend<0, false>(a, t, p, q, att, used, part, s)
          : a.type == 1 ? launch_attend<1, false>(a, t, p, q, att, used, part, s)
                        : launch_attend<2, false>(a, t, p, q, att, used, part, s);
    if (e != hipSuccess || !p.stream) return e;
    const uint32_t per = JOIN_WG / (a.head_dim / 4), groups = (p.tile_rows + per - 1) / per;
    hipLaunchKernelGGL(k_paged_join, dim3(a.kv_heads * p.tiles * groups), dim3(JOIN_WG), 0, s, a, att, p, used, part);
    return hipGetLastError();
}

}  // namespace smq
