/* Rows of logits before the choice of a token on gfx950: penalties over a history, biases, grammar masks, and the
 * greedy choice (include/smq.h has the formulas). */
#include "smq_device.h"

namespace smq {
namespace {

constexpr uint32_t LG_WG = 256;
constexpr uint32_t NONE = 0xffffffffu;

/* The best of some ids: the first id that may be taken and whether its logit is a NaN, then the lowest id of the largest
 * logit among those that are no NaN. */
struct Part {
    float best;
    uint32_t id, first, first_nan;
};
__device__ __forceinline__ void join(Part &a, const Part &b) {
    if (b.id != NONE && (a.id == NONE || b.best > a.best || (b.best == a.best && b.id < a.id))) {
        a.best = b.best;
        a.id = b.id;
    }
    if (b.first < a.first) {
        a.first = b.first;
        a.first_nan = b.first_nan;
    }
}
__device__ __forceinline__ Part join_wave(Part p) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        Part o;
        o.best = __shfl_xor(p.best, off);
        o.id = __shfl_xor(p.id, off);
        o.first = __shfl_xor(p.first, off);
        o.first_nan = __shfl_xor(p.first_nan, off);
        join(p, o);
    }
    return p;
}

/* [begin[r], begin[r + 1]) cut to the list's count entries. */
__device__ __forceinline__ void list_range(const int32_t *begin, uint32_t r, uint32_t count, uint32_t &b, uint32_t &e) {
    const int x = begin[r], y = begin[r + 1];
    b = x < 0 ? 0 : min((uint32_t)x, count);
    e = y < 0 ? 0 : min((uint32_t)y, count);
}

/* One workgroup per span of SPAN ids of a row, one pass over the logits. The whole history of the row is read and
 * counted in LDS where it falls into the span (integers: no order), biases 256 entries at a time: the first entry of an
 * id adds up the later ones in the order of the list, so that the same id twice gives the same bits on every run. */
template <uint32_t SPAN>
__global__ __launch_bounds__(LG_WG) void k_logits(LogitArgs a, Part *parts) {
    __shared__ uint32_t count[SPAN];
    __shared__ float add[SPAN];
    __shared__ uint32_t ids[LG_WG];
    __shared__ float vals[LG_WG];
    __shared__ Part best[LG_WG / 64];
    const uint32_t tid = threadIdx.x, r = blockIdx.y, v0 = blockIdx.x * SPAN;
    constexpr uint32_t EPT = SPAN / LG_WG;
    const float *row = a.logits + (size_t)r * a.stride;
    float l[EPT];
#pragma unroll
    for (uint32_t u = 0; u < EPT; ++u) {
        const uint32_t v = v0 + u * LG_WG + tid;
        l[u] = v < a.vocab ? row[v] : 0.0f;
        count[u * LG_WG + tid] = 0;
        add[u * LG_WG + tid] = 0.0f;
    }
    uint32_t mb = 0;
    bool masked = a.allowed != nullptr, none = false;
    if (masked) {
        const int mr = a.mask_row ? a.mask_row[r] : (int)r;
        masked = mr >= 0;
        none = masked && (uint32_t)mr >= a.allowed_rows;
        mb = (uint32_t)mr;
        if (none && tid == 0) *a.flag = 1;
    }
    __syncthreads();
    uint32_t hb = 0, he = 0, bb = 0, be = 0;
    if (a.history) {
        list_range(a.history_begin, r, a.history_count, hb, he);
        for (uint32_t i = hb + tid; i < he; i += LG_WG) {
            const uint32_t v = a.history[i] - v0;
            if (v < SPAN) atomicAdd(&count[v], 1u);
        }
    }
    if (a.bias_ids) {
        list_range(a.bias_begin, r, a.bias_count, bb, be);
        for (uint32_t i0 = bb; i0 < be; i0 += LG_WG) {
            const uint32_t n = min(LG_WG, be - i0), id = tid < n ? a.bias_ids[i0 + tid] - v0 : NONE;
            const float x = tid < n ? a.bias[i0 + tid] : 0.0f;
            __syncthreads();
            ids[tid] = id;
            vals[tid] = x;
            __syncthreads();
            if (id < SPAN) {
                bool first = true;
                for (uint32_t j = 0; j < tid; ++j) first = first && ids[j] != id;
                if (first) {
                    float sum = add[id] + x;
                    for (uint32_t j = tid + 1; j < n; ++j)
                        if (ids[j] == id) sum += vals[j];
                    add[id] = sum;
                }
            }
        }
    }
    __syncthreads();
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (he > hb) {
        rep = a.penalty[3 * (size_t)r];
        pres = a.penalty[3 * (size_t)r + 1];
        freq = a.penalty[3 * (size_t)r + 2];
    }
    const uint32_t words = (a.vocab + 31) / 32;
    Part p = {0.0f, NONE, NONE, 0};
#pragma unroll
    for (uint32_t u = 0; u < EPT; ++u) {
        const uint32_t i = u * LG_WG + tid, v = v0 + i;
        if (v >= a.vocab) continue;
        float x = l[u];
        const uint32_t c = count[i];
        if (c) {
            x = x > 0.0f ? x / rep : x * rep;
            const float t = (float)c * freq;
            x = x - (t + pres);
        }
        if (be > bb) x = x + add[i];
        const bool may = !masked || (!none && (a.allowed[(size_t)mb * words + v / 32] >> (v % 32) & 1u));
        if (!may) x = -INFINITY;
        if (a.out) a.out[(size_t)r * a.out_stride + v] = x;
        if (may) {
            const bool nan = x != x;
            const Part o = {x, nan ? NONE : v, v, nan};
            join(p, o);
        }
    }
    if (!parts) return;
    p = join_wave(p);
    if (tid % 64 == 0) best[tid / 64] = p;
    __syncthreads();
    if (tid == 0) {
        for (uint32_t w = 1; w < LG_WG / 64; ++w) join(p, best[w]);
        parts[(size_t)r * gridDim.x + blockIdx.x] = p;
    }
}

__global__ __launch_bounds__(64) void k_logits_pick(const Part *parts, uint32_t n, uint32_t *token) {
    Part p = {0.0f, NONE, NONE, 0};
    for (uint32_t i = threadIdx.x; i < n; i += 64) join(p, parts[(size_t)blockIdx.x * n + i]);
    p = join_wave(p);
    if (threadIdx.x == 0) token[blockIdx.x] = p.first_nan ? p.first : p.id;
}

constexpr uint32_t SPAN = 1024;
uint32_t spans(uint32_t vocab) { return (vocab + SPAN - 1) / SPAN; }

}  // namespace

size_t logits_workspace(uint32_t rows, uint32_t vocab) { return (size_t)rows * spans(vocab) * sizeof(Part); }

hipError_t launch_logits(const LogitArgs &a, uint32_t *token, void *ws, hipStream_t s) {
    const uint32_t n = spans(a.vocab);
    hipLaunchKernelGGL((k_logits<SPAN>), dim3(n, a.rows), dim3(LG_WG), 0, s, a, token ? (Part *)ws : nullptr);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !token) return e;
    hipLaunchKernelGGL(k_logits_pick, dim3(a.rows), dim3(64), 0, s, (const Part *)ws, n, token);
    return hipGetLastError();
}

}  // namespace smq
