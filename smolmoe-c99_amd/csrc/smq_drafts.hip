/* Trees of drafted tokens on gfx950: which new tokens each one sees (include/smq.h has the rules; their attention is in
 * smq_paged_attend.h). */
#include "smq_paged.h"

namespace smq {
namespace {

/* A workgroup per sequence, its parents in LDS; a thread per word of a row walks the row's ancestors, which descend, until
 * they are below the word. Depths by the thread of word 0, which walks them all. Trees of drafts are bound by the launch, two
 * trips to memory and the deepest token's walk: 24 trees of 40 3.7 us, one of 13 1.9. Chains are bound by the walks of all
 * words on one CU, which grow with tokens * words * depth: of 40 4.7 us, 100 10, 400 240, 1000 3.5 ms, 4096 221 ms. */
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

}  // namespace

hipError_t launch_draft_masks(const PagedArgs &a, const int32_t *parent, int32_t *depth, uint32_t *mask, uint32_t words,
                              hipStream_t s) {
    hipLaunchKernelGGL(k_draft_masks, dim3(a.seqs), dim3(DM_WG), 0, s, a, parent, depth, mask, words);
    return hipGetLastError();
}

}  // namespace smq
