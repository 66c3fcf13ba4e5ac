/* A step of a beam search on gfx950: of each group of beams the best continuations over the vocabulary, and the histories
 * that go on from them (include/smq.h has the rules).
 *
 * Three launches. The first goes over the logits once: of each block of 64 ids the largest, of each wave's ids the sum of
 * exponentials. The second, a workgroup per row, joins the sums; a row's best `select` ids lie in the `select` blocks whose
 * largest logits are the largest (on equal ones the lower block: each of them has an id that comes before any id of another
 * block), so it reads those again, lists what is no smaller than the last of these maxima, and sorts the list's best. The
 * third does the same with the candidates of a group's rows, and writes histories. No list can overflow, whatever the
 * logits are, and the lists' orders do not show: no two keys are equal. */
#include "smq_device.h"

namespace smq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
constexpr uint32_t BM_WG = 256, BM_WAVES = BM_WG / 64, NONE = 0xffffffffu;
constexpr uint32_t BM_BLOCK = 64, BM_LANES = BM_BLOCK / 4; /* ids of a block, lanes that have four each */

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
/* Keys of a group's candidates: the larger value, then the lower number. v 0: none. */
struct Cand {
    uint64_t v;
    uint64_t i; /* ~number */
    __device__ __forceinline__ bool operator>(const Cand &o) const { return v > o.v || (v == o.v && i > o.i); }
};
__device__ __forceinline__ bool some(uint64_t k) { return k != 0; }
__device__ __forceinline__ bool some(const Cand &k) { return k.v != 0; }
__device__ __forceinline__ uint64_t order_of(double x) { /* as key_of; not 0 */
    const uint64_t b = __double_as_longlong(x == 0.0 ? 0.0 : x);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(uint64_t v) { return __longlong_as_double(v >> 63 ? v & ~(1ull << 63) : ~v); }

/* 2^(x log2 e), x <= 0: the polynomial of 2^f on [-1/2, 1/2] with the least relative error of its degree, 1.4e-14. 16
 * instructions on 64 bits, which run at the rate of those on 32; the library's exp takes over twice as many. */
__device__ __forceinline__ double exp_of(double x) {
    const double t = fmax(x * 0x1.71547652b82fep+0, -1100.0), n = __builtin_rint(t), f = t - n;
    double p = 0x1.b4014c1ff3fbep-24;
    p = __builtin_fma(p, f, 0x1.63ee359dfa9f3p-20);
    p = __builtin_fma(p, f, 0x1.ffce18ebcfb6cp-17);
    p = __builtin_fma(p, f, 0x1.43088f9609f89p-13);
    p = __builtin_fma(p, f, 0x1.5d87fd93161f0p-10);
    p = __builtin_fma(p, f, 0x1.3b2ab72a268b1p-7);
    p = __builtin_fma(p, f, 0x1.c6b08d70d1248p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff81568ap-3);
    p = __builtin_fma(p, f, 0x1.62e42fefa374fp-1);
    p = __builtin_fma(p, f, 0x1.0000000000039p+0);
    return __builtin_ldexp(p, (int)n);
}

template <typename T, typename F>
__device__ __forceinline__ T reduce(T x, T *lds, F f) { /* over the workgroup */
    for (int off = 1; off < 64; off *= 2) x = f(x, __shfl_xor(x, off));
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    x = lds[0];
    for (uint32_t w = 1; w < BM_WAVES; ++w) x = f(x, lds[w]);
    return x;
}

/* What the first launch leaves of a row: block maxima (NaN where an id's logit is NaN or +inf), and of each wave of its
 * spans the sum of exp(l - the largest of the wave's blocks). */
struct Sums {
    float *top;
    double *sum;
    uint32_t blocks, sums, per; /* of a row; blocks a wave */
};

/* A wave takes U times 256 ids of the span: no exchange with the others. */
template <uint32_t U, bool WIDE>
__global__ __launch_bounds__(BM_WG) void k_beam_sums(BeamArgs a, Sums s) {
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = blockIdx.x * BM_WAVES + tid / 64, r = blockIdx.y;
    const uint32_t v0 = wave * U * 256;
    if (v0 >= a.vocab || (a.done && a.done[r])) return;
    const float *row = a.logits + (size_t)r * a.stride;
    f4 l[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t i = v0 + u * 256 + 4 * lane;
        if (WIDE && i + 4 <= a.vocab) {
            l[u] = *(const f4 *)(row + i);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) l[u][e] = i + e < a.vocab ? row[i + e] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        float m = fmaxf(fmaxf(l[u][0], l[u][1]), fmaxf(l[u][2], l[u][3]));
        bool bad = false;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) bad = bad || !(l[u][e] < INFINITY);
#pragma unroll
        for (int off = 1; off < (int)BM_LANES; off *= 2) m = fmaxf(m, __shfl_xor(m, off));
        const uint64_t those = __ballot(bad);
        const uint32_t block = (wave * U + u) * (64 / BM_LANES) + lane / BM_LANES;
        if (lane % BM_LANES == 0 && block < s.blocks) s.top[(size_t)r * s.blocks + block] = those ? __builtin_nanf("") : m;
        top = fmaxf(top, m);
    }
#pragma unroll
    for (int off = BM_LANES; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
    const double off = top == -INFINITY ? 0.0 : (double)top;
    double sum = 0.0;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) sum += exp_of((double)l[u][e] - off);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) s.sum[(size_t)r * s.sums + wave] = sum;
}

/* The `most` largest keys of list[0 .. m), descending, into best; returns their number. Until a list has 256 keys: of each
 * thread's keys the largest, of these the most-th largest, and only keys that are no smaller go on: those of `most` threads
 * at most, to the other of two lists (list, other) in turn. Then each key is put where its rank says. */
template <typename K>
__device__ __forceinline__ uint32_t best_of(K *list, K *other, uint32_t m, uint32_t most, K *keys, K *best, uint32_t *count) {
    const uint32_t tid = threadIdx.x;
    const K zero = {};
    while (m > BM_WG) {
        K mine = zero;
        for (uint32_t i = tid; i < m; i += BM_WG) mine = list[i] > mine ? list[i] : mine;
        __syncthreads();
        keys[tid] = mine;
        if (tid == 0) {
            *count = 0;
            best[0] = zero;
        }
        __syncthreads();
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < BM_WG; ++i) rank += keys[i] > mine;
        if (rank == most - 1 && some(mine)) best[0] = mine;
        __syncthreads();
        const K least = best[0];
        for (uint32_t i = tid; i < m; i += BM_WG)
            if (some(list[i]) && !(least > list[i])) other[atomicAdd(count, 1u)] = list[i];
        __syncthreads();
        m = *count;
        K *x = list;
        list = other;
        other = x;
    }
    __syncthreads();
    keys[tid] = tid < m ? list[tid] : zero;
    if (tid == 0) *count = 0;
    __syncthreads();
    const K mine = keys[tid];
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < BM_WG; ++i) rank += keys[i] > mine;
    if (some(mine) && rank < most) {
        best[rank] = mine;
        atomicMax(count, rank + 1);
    }
    __syncthreads();
    return *count;
}
/* LDS of the lists: the first one's keys, and what of it can go on. */
__host__ __device__ inline uint32_t list_next(uint32_t first, uint32_t most) { return most * ((first + BM_WG - 1) / BM_WG); }

/* A workgroup per row: its `select` best ids and their values. */
__global__ __launch_bounds__(BM_WG) void k_beam_rows(BeamArgs a, Sums s, double *value, uint32_t *id) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ double sums[BM_WAVES];
    __shared__ float tops[BM_WAVES];
    __shared__ int bads[BM_WAVES];
    __shared__ uint64_t keys[BM_WG], best[MAX_SELECT], blocks[MAX_SELECT];
    __shared__ uint32_t count;
    uint64_t *list = (uint64_t *)lds, *other = list + a.select * BM_BLOCK;
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const float *row = a.logits + (size_t)r * a.stride, *bt = s.top + (size_t)r * s.blocks;
    const float score = a.score[r];
    value += (size_t)r * a.select;
    id += (size_t)r * a.select;
    const bool done = a.done && a.done[r];
    float top = -INFINITY;
    int bad = !(score < INFINITY);
    if (!done)
        for (uint32_t i = tid; i < s.blocks; i += BM_WG) {
            bad |= !(bt[i] < INFINITY);
            top = fmaxf(top, bt[i]);
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
    for (uint32_t i = tid; i < s.sums; i += BM_WG) {
        float m = -INFINITY;
        for (uint32_t k = 0; k < s.per; ++k)
            if (i * s.per + k < s.blocks) m = fmaxf(m, bt[i * s.per + k]);
        if (m > -INFINITY) sum += s.sum[(size_t)r * s.sums + i] * exp_of((double)m - (double)top);
    }
    sum = reduce(sum, sums, [](double x, double y) { return x + y; });
    const double lse = (double)top + log(sum);
    /* the blocks: of each thread's the largest, and those that are no smaller than the select-th of these */
    uint64_t mine = 0;
    for (uint32_t i = tid; i < s.blocks; i += BM_WG) {
        const uint64_t k = bt[i] == -INFINITY ? 0 : key_of(bt[i], i);
        mine = k > mine ? k : mine;
    }
    keys[tid] = mine;
    if (tid == 0) {
        count = 0;
        best[0] = 1;
    }
    __syncthreads();
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < BM_WG; ++i) rank += keys[i] > mine;
    if (rank == a.select - 1 && mine) best[0] = mine;
    __syncthreads();
    const uint64_t least = best[0];
    for (uint32_t i = tid; i < s.blocks; i += BM_WG) {
        const uint64_t k = bt[i] == -INFINITY ? 0 : key_of(bt[i], i);
        if (k >= least) list[atomicAdd(&count, 1u)] = k;
    }
    __syncthreads();
    const uint32_t nb = best_of(list, other, count, a.select, keys, blocks, &count);
    /* their ids */
    __syncthreads();
    if (tid == 0) count = 0;
    const float low = nb == a.select ? logit_of(blocks[nb - 1]) : -FLT_MAX;
    __syncthreads();
    for (uint32_t b = tid / BM_LANES; b < nb; b += BM_WG / BM_LANES) {
        const uint32_t i = id_of(blocks[b]) * BM_BLOCK + 4 * (tid % BM_LANES);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const float l = i + e < a.vocab ? row[i + e] : -INFINITY;
            if (l >= low) list[atomicAdd(&count, 1u)] = key_of(l, i + e);
        }
    }
    __syncthreads();
    const uint32_t n = best_of(list, other, count, a.select, keys, best, &count);
    for (uint32_t k = tid; k < a.select; k += BM_WG) {
        const uint64_t b = k < n ? best[k] : 0;
        value[k] = b ? (double)score + ((double)logit_of(b) - lse) : -INFINITY;
        id[k] = id_of(b);
    }
}

/* A workgroup per result where there are histories, else per group: the best of the group's candidates, and its results. */
__global__ __launch_bounds__(BM_WG) void k_beam_join(BeamArgs a, const double *value, const uint32_t *id, uint32_t per) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[]; /* the lists */
    __shared__ Cand keys[BM_WG], best[MAX_SELECT];
    __shared__ uint32_t count;
    const uint32_t g = blockIdx.x / per, tid = threadIdx.x, n = a.beams * a.select;
    const size_t at = (size_t)g * n;
    Cand *list = (Cand *)lds, *other = list + (n > BM_WG ? list_next(n, a.select) : BM_WG);
    auto cand = [&](uint32_t i) {
        const double v = value[at + i];
        return v > -INFINITY ? Cand{order_of(v), ~(uint64_t)i} : Cand{0, 0};
    };
    uint32_t m = n;
    if (n > BM_WG) {
        Cand mine = {0, 0};
        for (uint32_t i = tid; i < n; i += BM_WG) {
            const Cand c = cand(i);
            mine = c > mine ? c : mine;
        }
        keys[tid] = mine;
        if (tid == 0) {
            count = 0;
            best[0] = Cand{1, 0};
        }
        __syncthreads();
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < BM_WG; ++i) rank += keys[i] > mine;
        if (rank == a.select - 1 && some(mine)) best[0] = mine;
        __syncthreads();
        const Cand least = best[0];
        for (uint32_t i = tid; i < n; i += BM_WG) {
            const Cand c = cand(i);
            if (!(least > c)) list[atomicAdd(&count, 1u)] = c;
        }
        __syncthreads();
        m = count;
    } else if (tid < n) {
        list[tid] = cand(tid);
    }
    __syncthreads();
    const uint32_t found = best_of(list, other, m, a.select, keys, best, &count);
    for (uint32_t k = blockIdx.x % per; k < a.select; k += per) {
        const uint32_t o = g * a.select + k, w = k < found ? (uint32_t)~best[k].i : 0;
        const bool none = k >= found;
        const uint32_t r = none ? 0 : g * a.beams + w / a.select, token = none ? NONE : id[at + w];
        const bool over = !none && a.done && a.done[r];
        if (tid == 0) {
            a.parent[o] = none ? -1 : (int)r;
            a.token[o] = token;
            a.score_out[o] = none ? -INFINITY : (float)value_of(best[k].v);
            if (a.done_out) a.done_out[o] = none || over || (a.eos != NONE && token == a.eos);
        }
        if (!a.history) continue;
        const int have = none ? 0 : a.length[r];
        const uint32_t len = (uint32_t)min(max(have, 0), (int)a.history_stride);
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

/* Blocks a wave of the first launch: eight where the rows fill the card with them. */
uint32_t wave_loads(const BeamArgs &a) {
    const uint64_t ids = (uint64_t)a.groups * a.beams * a.vocab;
    return ids >= (uint64_t)1024 * 4096 ? 4 : ids >= (uint64_t)1024 * 2048 ? 2 : 1;
}
Sums sums_of(const BeamArgs &a) {
    Sums s;
    s.top = nullptr;
    s.sum = nullptr;
    s.per = 64 / BM_LANES * wave_loads(a);
    s.blocks = (a.vocab + BM_BLOCK - 1) / BM_BLOCK;
    s.sums = (s.blocks + s.per - 1) / s.per;
    return s;
}

}  // namespace

size_t beam_workspace(const BeamArgs &a) {
    const Sums s = sums_of(a);
    const size_t rows = (size_t)a.groups * a.beams;
    return rows * ((size_t)a.select * 12 + s.sums * 8 + s.blocks * 4);
}

hipError_t launch_beam(const BeamArgs &a, void *ws, hipStream_t st) {
    const uint32_t rows = a.groups * a.beams, U = wave_loads(a);
    Sums s = sums_of(a);
    double *value = (double *)ws;
    s.sum = value + (size_t)rows * a.select;
    s.top = (float *)(s.sum + (size_t)rows * s.sums);
    uint32_t *id = (uint32_t *)(s.top + (size_t)rows * s.blocks);
    const bool wide = !(((uintptr_t)a.logits | (rows > 1 ? a.stride * 4 : 0)) & 15);
    const dim3 grid((s.sums + BM_WAVES - 1) / BM_WAVES, rows);
#define SMQ_BEAM(U)                                                                                        \
    do {                                                                                                   \
        if (wide) hipLaunchKernelGGL((k_beam_sums<U, true>), grid, dim3(BM_WG), 0, st, a, s);              \
        else hipLaunchKernelGGL((k_beam_sums<U, false>), grid, dim3(BM_WG), 0, st, a, s);                  \
    } while (0)
    if (U == 4) SMQ_BEAM(4);
    else if (U == 2) SMQ_BEAM(2);
    else SMQ_BEAM(1);
#undef SMQ_BEAM
    const uint32_t first = a.select * BM_BLOCK, n = a.beams * a.select;
    hipLaunchKernelGGL(k_beam_rows, dim3(rows), dim3(BM_WG), (first + list_next(first, a.select)) * 8, st, a, s, value, id);
    const uint32_t per = a.history ? a.select : 1, list = n > BM_WG ? list_next(n, a.select) : BM_WG;
    hipLaunchKernelGGL(k_beam_join, dim3(a.groups * per), dim3(BM_WG), (list + list_next(list, a.select)) * sizeof(Cand), st, a,
                       value, id, per);
    return hipGetLastError();
}

}  // namespace smq
