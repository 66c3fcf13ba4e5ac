/* Paged KV cache on gfx950: RoPE and the store of new tokens (f32, f16, Q8), rows read back, and the attention of a
 * ragged batch of new tokens over the pages (include/smq.h has the layout of a page). */
#include <hip/hip_fp16.h>

#include "smq_paged_attend.h"

namespace smq {
namespace {

/* Coordinate d of a rotated head row x (smq_rope_kv's products and order). */
__device__ __forceinline__ float rotated(const float *x, uint32_t d, uint32_t pairs, const float *c, const float *s) {
    if (d >= 2 * pairs) return x[d];
    const uint32_t i = d / 2;
    const float p = x[2 * i], q = x[2 * i + 1];
    const float pc = p * c[i], qs = q * s[i], ps = p * s[i], qc = q * c[i];
    return d & 1 ? ps + qc : pc - qs;
}

constexpr int ST_WG = 256;

/* One workgroup per row; 32 lanes per block of 32 dims of a head, so that a Q8 block's maximum is a shuffle. */
template <uint32_t TYPE>
__global__ __launch_bounds__(ST_WG) void k_paged_store(PagedArgs a, const float *q, float *q_out, const float *k,
                                                       const float *v, const float *cs, const float *sn) {
    const uint32_t r = blockIdx.x, tid = threadIdx.x, lane = tid % 32;
    uint32_t s, pos;
    if (r == 0) check_begin(a, tid, ST_WG);
    if (!place_of(a, r, s, pos)) return;
    const float *c = cs + (size_t)pos * a.pairs, *sr = sn + (size_t)pos * a.pairs;
    if (q) {
        const size_t row = (size_t)r * a.heads * a.head_dim;
        for (uint32_t i = tid; i < a.heads * a.head_dim / 2; i += ST_WG) {
            const uint32_t h = i / (a.head_dim / 2), d = 2 * (i % (a.head_dim / 2));
            const float *x = q + row + (size_t)h * a.head_dim;
            const float y0 = rotated(x, d, a.pairs, c, sr), y1 = rotated(x, d + 1, a.pairs, c, sr);
            q_out[row + (size_t)h * a.head_dim + d] = y0; /* both read before either is written: q_out may be q */
            q_out[row + (size_t)h * a.head_dim + d + 1] = y1;
        }
    }
    const int page = page_of(a, s, pos);
    if (page < 0) return;
    const uint32_t P = 1u << a.shift, slot = pos & (P - 1);
    const size_t krow = (size_t)r * a.kv_heads * a.head_dim;
    for (uint32_t i = tid / 32; i < a.kv_heads * a.nb * 2; i += ST_WG / 32) {
        const bool isv = i >= a.kv_heads * a.nb;
        const uint32_t j = isv ? i - a.kv_heads * a.nb : i, h = j / a.nb, b = j % a.nb, d = b * 32 + lane;
        const bool in = d < a.head_dim;
        const float *x = (isv ? v : k) + krow + (size_t)h * a.head_dim;
        const float y = !in ? 0.0f : isv ? x[d] : rotated(x, d, a.pairs, c, sr);
        const size_t ph = (size_t)page * a.kv_heads + h;
        const size_t at = isv ? (ph * a.head_dim + d) * P + slot : (ph * P + slot) * a.head_dim + d;
        void *pool = isv ? a.values : a.keys;
        bool bad = !(fabsf(y) <= FLT_MAX);
        if constexpr (TYPE == 0) {
            if (in) ((float *)pool)[at] = y;
        } else if constexpr (TYPE == 1) {
            const __half hv = __float2half_rn(y);
            bad = bad || !(fabsf(__half2float(hv)) <= FLT_MAX);
            if (in) ((__half *)pool)[at] = hv;
        } else {
            float m = fabsf(y);
            int any = bad;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) {
                m = fmaxf(m, __shfl_xor(m, off, 32));
                any |= __shfl_xor(any, off, 32);
            }
            const float scale = m / 127.0f;
            const float inv = scale >= FLT_MIN ? 1.0f / scale : 0.0f;
            float p = __builtin_rintf(y * inv);
            p = p > 127.0f ? 127.0f : p < -127.0f ? -127.0f : p;
            if (in) ((int8_t *)pool)[at] = any ? 0 : (int8_t)(int)p;
            if (lane == 0) (isv ? a.vs : a.ks)[(ph * a.nb + b) * P + slot] = any ? __builtin_nanf("") : scale;
            bad = any;
        }
        if (bad) *a.flag = 1;
    }
}

template <uint32_t TYPE>
__device__ __forceinline__ float element(const void *pool, size_t at, const float *scales, size_t sat) {
    if constexpr (TYPE == 0) return ((const float *)pool)[at];
    if constexpr (TYPE == 1) return __half2float(((const __half *)pool)[at]);
    return (float)((const int8_t *)pool)[at] * scales[sat];
}

template <uint32_t TYPE>
__global__ __launch_bounds__(ST_WG) void k_paged_read(PagedArgs a, float *keys, float *values) {
    const uint32_t r = blockIdx.x;
    uint32_t s, pos;
    if (r == 0) check_begin(a, threadIdx.x, ST_WG);
    if (!place_of(a, r, s, pos)) return;
    const int page = page_of(a, s, pos);
    if (page < 0) return;
    const uint32_t P = 1u << a.shift, slot = pos & (P - 1), kd = a.kv_heads * a.head_dim;
    for (uint32_t i = threadIdx.x; i < kd; i += ST_WG) {
        const uint32_t h = i / a.head_dim, d = i % a.head_dim;
        const size_t ph = (size_t)page * a.kv_heads + h, sc = (ph * a.nb + d / 32) * P + slot;
        keys[(size_t)r * kd + i] = element<TYPE>(a.keys, (ph * P + slot) * a.head_dim + d, a.ks, sc);
        values[(size_t)r * kd + i] = element<TYPE>(a.values, (ph * a.head_dim + d) * P + slot, a.vs, sc);
    }
}

/* Joins what several workgroups have of a tile and KV head: the weights of their maxima, in their order. head_dim / 4 lanes
 * per row. A lane requests its part of O and the maxima and sums of eight workgroups at once: after the tile's four words
 * one round trip to memory joins up to eight. */
constexpr uint32_t JOIN_WG = 256, JOIN_AT_ONCE = 8;
__global__ __launch_bounds__(JOIN_WG) void k_paged_join(PagedArgs a, float *att, AttendPlan p, const i4 *used,
                                                        const float *part) {
    const uint32_t hd = a.head_dim, lanes = hd / 4, per = JOIN_WG / lanes;
    const uint32_t groups = (p.tile_rows + per - 1) / per, tile = blockIdx.x / groups, kh = tile % a.kv_heads;
    const uint32_t r = blockIdx.x % groups * per + threadIdx.x / lanes, d = 4 * (threadIdx.x % lanes);
    const i4 u = used[tile];
    const uint32_t parts = (uint32_t)u[0] & 0xffff, n = (uint32_t)u[0] >> 16, slot = (uint32_t)u[3];
    if (parts < 2 || r >= n || threadIdx.x / lanes >= per) return;
    const f2 *pml = (const f2 *)(part + (size_t)2 * p.stream * a.kv_heads * p.tile_rows * hd);
    float m = -FLT_MAX, l = 0.0f;
    f4 o = {};
    for (uint32_t i0 = 0; i0 < parts; i0 += JOIN_AT_ONCE) {
        f2 ml[JOIN_AT_ONCE];
        f4 x[JOIN_AT_ONCE];
        float top = m;
#pragma unroll
        for (uint32_t i = 0; i < JOIN_AT_ONCE; ++i) {
            const uint32_t k = min(i0 + i, parts - 1); /* the first one's slot, then slots 0 of the next workgroups */
            const size_t y = ((size_t)(k ? (slot & ~1u) + 2 * k : slot) * a.kv_heads + kh) * p.tile_rows + r;
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
            const float e = i0 + i < parts ? __builtin_amdgcn_exp2f(ml[i][0] - m) : 0.0f;
            l += e * ml[i][1];
            o += e * x[i];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *(f4u *)(att + row_at(a, u[1], kh, (uint32_t)u[2] + r) + d) = o * inv;
}

/* Up to 32 rows a sequence and KV head on average (decoding) the tiles have 16 rows; above, a workgroup's waves own
 * theirs.
 *
 * Workgroups that share the steps out: two a CU for products and for decoding heads of up to 64 (8 KiB of f16 a step and
 * wave: 64 sequences at 5000, 8 KV heads, 134 us with one a CU, 94 with two), one a CU for wider ones (16 x 12000, 8 KV
 * heads of 128: 145, 150; 32 x 3000 Q8, 2 KV heads: 31, 35).
 *
 * Sharing them out costs a second launch, which joins: not where there are tiles for every CU four times over, and not
 * where a tile's steps at the longest length exceed an equal share by less than that (about 24 steps: 64 sequences at 700,
 * 2 KV heads of 64: 11.8 us with a workgroup per tile, 15.4 shared out). */
AttendPlan attend_plan(const PagedArgs &a, size_t ws_bytes) {
    AttendPlan p;
    const uint32_t G = a.heads / a.kv_heads;
    const uint64_t rows = (uint64_t)a.tokens * G, seqs = a.seqs < a.tokens ? a.seqs : a.tokens;
    p.owns = rows > 32 * seqs;
    p.tile_rows = p.owns ? 64 * attend_rt(attend_ks(a.head_dim)) : 16;
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
    /* tiles of an even batch, and by how many steps the longest could exceed an equal share */
    const uint64_t tiles = seqs * ((rows / (seqs ? seqs : 1) + p.tile_rows - 1) >> p.row_shift) * a.kv_heads;
    const uint64_t steps = (most - p.fixed) / 2 / PA_STEP;
    if (tiles >= 1024 || (tiles < groups ? steps * (groups - tiles) / groups : 0) <= 24) p.stream = 0;
    const size_t used = attend_used_bytes(a, p), each = attend_part_bytes(a, p.tile_rows);
    const uint64_t room = ws_bytes > used ? (ws_bytes - used) / each : 0;
    if (room < p.stream) p.stream = room > p.tiles ? (uint32_t)room : 0;
    return p;
}

}  // namespace

#define SMQ_PAGED(KERNEL, GRID, BLOCK, ...)                                                          \
    do {                                                                                             \
        if (a.type == 0) hipLaunchKernelGGL((KERNEL<0>), GRID, BLOCK, 0, s, a, __VA_ARGS__);         \
        else if (a.type == 1) hipLaunchKernelGGL((KERNEL<1>), GRID, BLOCK, 0, s, a, __VA_ARGS__);    \
        else hipLaunchKernelGGL((KERNEL<2>), GRID, BLOCK, 0, s, a, __VA_ARGS__);                     \
    } while (0)

hipError_t launch_paged_rope_kv(const PagedArgs &a, const float *q, float *q_out, const float *k, const float *v,
                                const float *cs, const float *sn, hipStream_t s) {
    SMQ_PAGED(k_paged_store, dim3(a.tokens), dim3(ST_WG), q, q_out, k, v, cs, sn);
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedArgs &a, float *keys, float *values, hipStream_t s) {
    SMQ_PAGED(k_paged_read, dim3(a.tokens), dim3(ST_WG), keys, values);
    return hipGetLastError();
}


size_t paged_attention_workspace(const PagedArgs &a) {
    const AttendPlan p = attend_plan(a, ~(size_t)0);
    return p.stream ? attend_used_bytes(a, p) + p.stream * attend_part_bytes(a, p.tile_rows) : 0;
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
