/* A step of a beam search on gfx950: of each group of beams the best continuations over the vocabulary, and the histories
 * that go on from them (include/smq.h has the rules). */
#include "smq_device.h"

namespace smq {
namespace {

constexpr uint32_t BM_WG = 256, NONE = 0xffffffffu;

/* Keys of one row: the larger logit, then the lower id, is the larger key. 0: no candidate. */
__device__ __forceinline__ uint64_t key_of(float l, uint32_t id) {
    const uint32_t b = __float_as_uint(l == 0.0f ? 0.0f : l); /* one zero */
    return (uint64_t)(b >> 31 ? ~b : b | 1u << 31) << 32 | (NONE - id);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b >> 31 ? b & ~(1u << 31) : ~b);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return NONE - (uint32_t)key; }

template <typename T, typename F>
__device__ __forceinline__ T reduce(T x, T *lds, F f) { /* over the workgroup */
    for (int off = 1; off < 64; off *= 2) x = f(x, __shfl_xor(x, off));
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    x = lds[0];
    for (uint32_t w = 1; w < BM_WG / 64; ++w) x = f(x, lds[w]);
    return x;
}

/* A workgroup per row: its maximum, its sum, its best ids one after another. */
__global__ __launch_bounds__(BM_WG) void k_beam_rows(BeamArgs a, double *value, uint32_t *id) {
    __shared__ double sums[BM_WG / 64];
    __shared__ float tops[BM_WG / 64];
    __shared__ unsigned long long keys[BM_WG / 64];
    __shared__ int bads[BM_WG / 64];
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const float *row = a.logits + (size_t)r * a.stride;
    const float score = a.score[r];
    value += (size_t)r * a.select;
    id += (size_t)r * a.select;
    const bool done = a.done && a.done[r];
    float top = -INFINITY;
    int bad = !(score < INFINITY);
    if (!done)
        for (uint32_t i = tid; i < a.vocab; i += BM_WG) {
            bad |= !(row[i] < INFINITY);
            top = fmaxf(top, row[i]);
        }
    bad = reduce(bad, bads, [](int x, int y) { return x | y; });
    top = reduce(top, tops, [](float x, float y) { return fmaxf(x, y); });
    if (bad && tid == 0) *a.flag = 1;
    const bool none = bad || score == -INFINITY || (!done && top == -INFINITY);
    if (none || done) {
        for (uint32_t k = tid; k < a.select; k += BM_WG) {
            value[k] = !none && k == 0 ? (double)score : -INFINITY;
            id[k] = a.pad;
        }
        return;
    }
    double sum = 0.0;
    for (uint32_t i = tid; i < a.vocab; i += BM_WG) sum += exp((double)row[i] - (double)top);
    sum = reduce(sum, sums, [](double x, double y) { return x + y; });
    const double lse = (double)top + log(sum);
    unsigned long long below = ~0ull;
    for (uint32_t k = 0; k < a.select; ++k) {
        unsigned long long best = 0;
        for (uint32_t i = tid; i < a.vocab; i += BM_WG) {
            const unsigned long long x = row[i] == -INFINITY ? 0 : key_of(row[i], i);
            best = x < below && x > best ? x : best;
        }
        best = reduce(best, keys, [](unsigned long long x, unsigned long long y) { return x > y ? x : y; });
        if (tid == 0) {
            value[k] = best ? (double)score + ((double)logit_of(best) - lse) : -INFINITY;
            id[k] = id_of(best);
        }
        below = best ? best : 1;
    }
}

/* A workgroup per group: the best of its rows' candidates, and the histories. */
__global__ __launch_bounds__(BM_WG) void k_beam_join(BeamArgs a, const double *value, const uint32_t *id) {
    extern __shared__ double lds[]; /* beams * select values */
    __shared__ double best[64];
    __shared__ uint32_t which[64];
    const uint32_t g = blockIdx.x, tid = threadIdx.x, n = a.beams * a.select;
    const size_t at = (size_t)g * n;
    for (uint32_t i = tid; i < n; i += BM_WG) lds[i] = value[at + i];
    if (tid < 64) which[tid] = NONE;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += BM_WG) {
        const double v = lds[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += lds[j] > v || (lds[j] == v && j < i);
        if (rank < a.select && v > -INFINITY) {
            best[rank] = v;
            which[rank] = i;
        }
    }
    __syncthreads();
    for (uint32_t k = 0; k < a.select; ++k) {
        const uint32_t w = which[k], o = g * a.select + k;
        const bool none = w == NONE;
        const uint32_t r = none ? 0 : g * a.beams + w / a.select, token = none ? NONE : id[at + w];
        const bool over = !none && a.done && a.done[r];
        if (tid == 0) {
            a.parent[o] = none ? -1 : (int)r;
            a.token[o] = token;
            a.score_out[o] = none ? -INFINITY : (float)best[k];
            if (a.done_out) a.done_out[o] = none || over || (a.eos != NONE && token == a.eos);
        }
        if (!a.history) continue;
        const int have = none ? 0 : a.length[r];
        uint32_t len = (uint32_t)min(max(have, 0), (int)a.history_stride);
        const bool more = !none && !over && len < a.history_stride;
        if (tid == 0) {
            if (have < 0 || have > (int)a.history_stride || (!none && !over && !more)) *a.flag = 1;
            a.length_out[o] = (int)(len + more);
        }
        for (uint32_t i = tid; i < a.history_stride; i += BM_WG)
            a.history_out[(size_t)o * a.history_stride + i] =
                i < len ? a.history[(size_t)r * a.history_stride + i] : i == len && more ? token : NONE;
    }
}

}  // namespace

size_t beam_workspace(const BeamArgs &a) { return (size_t)a.groups * a.beams * a.select * 12 + 16; }

hipError_t launch_beam(const BeamArgs &a, void *ws, hipStream_t s) {
    const uint32_t rows = a.groups * a.beams;
    double *value = (double *)ws;
    uint32_t *id = (uint32_t *)(value + (size_t)rows * a.select);
    hipLaunchKernelGGL(k_beam_rows, dim3(rows), dim3(BM_WG), 0, s, a, value, id);
    hipLaunchKernelGGL(k_beam_join, dim3(a.groups), dim3(BM_WG), a.beams * a.select * 8, s, a, value, id);
    return hipGetLastError();
}

}  // namespace smq
