/* Trees of drafted tokens on gfx950: which new tokens each one sees, and their attention over a paged cache
 * (include/smq.h has the rules). */
#include "smq_paged.h"

namespace smq {
namespace {

/* A workgroup per sequence, its parents in LDS; a thread per word of a row walks the row's ancestors, which descend, until
 * they are below the word. Depths by the thread of word 0, which walks them all. */
constexpr uint32_t DM_WG = 256, DM_MOST = 32 * MAX_MASK_WORDS;
__global__ __launch_bounds__(DM_WG) void k_draft_masks(PagedArgs a, const int32_t *parent, int32_t *depth, uint32_t *mask,
                                                       uint32_t words) {
    __shared__ int16_t up[DM_MOST];
    const uint32_t tid = threadIdx.x;
    const int b0 = a.begin[blockIdx.x], b1 = a.begin[blockIdx.x + 1];
    if (b0 < 0 || b1 < b0 || (uint32_t)b1 > a.tokens || (uint32_t)(b1 - b0) > 32 * words) {
        if (tid == 0) *a.flag = 1;
        return;
    }
    const uint32_t n = (uint32_t)(b1 - b0);
    for (uint32_t i = tid; i < n; i += DM_WG) {
        const int p = parent[b0 + i];
        if (p >= (int)i) *a.flag = 1;
        up[i] = (int16_t)(p >= (int)i ? -1 : max(p, -1));
    }
    __syncthreads();
    for (uint32_t x = tid; x < n * words; x += DM_WG) {
        const uint32_t i = x / words, w = x - i * words;
        uint32_t bits = 0;
        int steps = -1;
        for (int t = (int)i; t >= (int)(32 * w); t = up[t], ++steps)
            if ((uint32_t)t / 32 == w) bits |= 1u << (t % 32);
        mask[(size_t)(b0 + (int)i) * words + w] = bits;
        if (w == 0) depth[b0 + (int)i] = steps;
    }
}

/* A wave per row and head: 64 positions at a time, a lane the score of one, then a lane four dims of O. */
template <uint32_t TYPE>
__device__ __forceinline__ float element(const void *p, size_t i) {
    if constexpr (TYPE == 0) return ((const float *)p)[i];
    else if constexpr (TYPE == 1) return (float)((const _Float16 *)p)[i];
    else return (float)((const int8_t *)p)[i];
}
template <uint32_t TYPE>
__global__ __launch_bounds__(64) void k_tree(PagedArgs a, TreeArgs t, const float *q, float *att) {
    const uint32_t r = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kh = h / (a.heads / a.kv_heads), lane = threadIdx.x;
    if (blockIdx.x == 0) check_begin(a, lane, 64);
    uint32_t s, pos;
    float *out = att + ((size_t)r * a.heads + h) * a.head_dim;
    if (!place_of(a, r, s, pos)) { /* no place, or padding */
        if ((int)r >= a.begin[0] && (int)r < a.begin[a.seqs])
            for (uint32_t i = lane; i < a.head_dim; i += 64) out[i] = 0.0f;
        return;
    }
    Seq sq;
    sequence(a, s, sq);
    const uint32_t first = (uint32_t)max(sq.first, 0);
    const int d = t.depth ? t.depth[r] : 0;
    const bool fine = sq.first >= 0 && (uint32_t)sq.n <= 32 * t.words && d >= 0 && (uint32_t)d < a.context - min(first, a.context);
    if (!fine) *a.flag = 1;
    const uint32_t p = first + (uint32_t)d, low = a.window && p + 1 > a.window ? p + 1 - a.window : 0;
    float m = -INFINITY, l = 0.0f, o[4] = {};
    const float *x = q + ((size_t)r * a.heads + h) * a.head_dim;
    const uint32_t end = fine ? min(first + (uint32_t)sq.n, a.limit) : 0, P = 1u << a.shift;
    for (uint32_t j0 = 0; j0 < end; j0 += 64) {
        const uint32_t j = j0 + lane;
        bool seen = j < end && (j < first ? j >= low || j < a.sinks : (t.mask[(size_t)r * t.words + (j - first) / 32] >> ((j - first) % 32) & 1));
        const int page = seen ? page_of(a, s, j) : -1;
        seen = seen && page >= 0;
        float sc = -INFINITY;
        if (seen) {
            const size_t at = (((size_t)page * a.kv_heads + kh) << a.shift | (j & (P - 1))) * a.head_dim;
            const float *w = a.ks + ((((size_t)page * a.kv_heads + kh) * a.nb) << a.shift) + (j & (P - 1));
            sc = 0.0f;
            for (uint32_t i = 0; i < a.head_dim; ++i)
                sc += x[i] * (TYPE == 2 ? element<TYPE>(a.keys, at + i) * w[(size_t)(i / 32) << a.shift] : element<TYPE>(a.keys, at + i));
            sc /= sqrtf((float)a.head_dim);
        }
        float top = sc;
        for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
        top = fmaxf(top, m);
        if (top == -INFINITY) continue;
        const float e = seen ? expf(sc - top) : 0.0f, old = expf(m - top);
        m = top;
        l *= old;
        for (int k = 0; k < 4; ++k) o[k] *= old;
        for (uint32_t i = 0; i < 64; ++i) {
            const float ei = __shfl(e, (int)i);
            const int pg = __shfl(page, (int)i);
            l += ei;
            if (ei == 0.0f) continue;
            const uint32_t slot = j0 + i & (P - 1);
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t dim = lane + 64 * k;
                if (dim >= a.head_dim) break;
                float v = element<TYPE>(a.values, (((((size_t)pg * a.kv_heads + kh) * a.head_dim + dim)) << a.shift) + slot);
                if (TYPE == 2) v *= a.vs[((((size_t)pg * a.kv_heads + kh) * a.nb + dim / 32) << a.shift) + slot];
                o[k] += ei * v;
            }
        }
    }
    for (uint32_t k = 0; k < 4; ++k)
        if (lane + 64 * k < a.head_dim) out[lane + 64 * k] = l == 0.0f ? 0.0f : o[k] / l;
}

}  // namespace

hipError_t launch_draft_masks(const PagedArgs &a, const int32_t *parent, int32_t *depth, uint32_t *mask, uint32_t words,
                              hipStream_t s) {
    hipLaunchKernelGGL(k_draft_masks, dim3(a.seqs), dim3(DM_WG), 0, s, a, parent, depth, mask, words);
    return hipGetLastError();
}

size_t paged_tree_workspace(const PagedArgs &) { return 0; }

hipError_t launch_paged_tree(const PagedArgs &a, const TreeArgs &t, const float *q, float *att, void *, size_t,
                             hipStream_t s) {
    const dim3 grid(a.tokens * a.heads);
    if (a.type == 0) hipLaunchKernelGGL((k_tree<0>), grid, dim3(64), 0, s, a, t, q, att);
    else if (a.type == 1) hipLaunchKernelGGL((k_tree<1>), grid, dim3(64), 0, s, a, t, q, att);
    else hipLaunchKernelGGL((k_tree<2>), grid, dim3(64), 0, s, a, t, q, att);
    return hipGetLastError();
}

}  // namespace smq
