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
constexpr uint32_t BM_BLOCK = 64, BM_LANES = 16; /* ids of a block, lanes that have four each */

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

/* e^x, x <= 0 (below -700, -infinity too, as at -700: nothing beside the largest term, 1): x log2 e to a whole number, which
 * the sum with 1.5 * 2^52 leaves in its low bits, and f in [-1/2, 1/2], whose 2^f is the polynomial with the least relative
 * error of its degree, 7.8e-13 (a term may have 1e-12: one of these, not a product of two). 14 instructions on 64 bits, which
 * run at the rate of those on 32. lead: the polynomial's first coefficient, in vector registers (an instruction takes one
 * scalar operand). */
constexpr double EXP_LEAD = 0x1.61af6ea7cb2d7p-20;
__device__ __forceinline__ double exp_of(double x, double lead) {
    x = fmax(x, -700.0);
    const double log2e = 0x1.71547652b82fep+0, magic = 0x1.8p+52;
    const double r = __builtin_fma(x, log2e, magic), f = __builtin_fma(x, log2e, -(r - magic));
    double p = __builtin_fma(lead, f, 0x1.00dad0d6f5ff9p-16);
    p = __builtin_fma(p, f, 0x1.430accf559f5cp-13);
    p = __builtin_fma(p, f, 0x1.5d87483a5a42cp-10);
    p = __builtin_fma(p, f, 0x1.3b2ab5c4fcf88p-7);
    p = __builtin_fma(p, f, 0x1.c6b08dd46bc16p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff931c07p-3);
    p = __builtin_fma(p, f, 0x1.62e42fef8615ep-1);
    p = __builtin_fma(p, f, 0x1.ffffffffff7a6p-1);
    return __hiloint2double(__double2hiint(p) + (__double2loint(r) << 20), __double2loint(p));
}
/* The largest of three in one instruction (the compiler's fmaxf makes every input canonical first). A NaN loses. */
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}

/* x with its neighbour's by a rotation in rows of 16 lanes. */
template <int N>
__device__ __forceinline__ int turned(int x) {
    return __builtin_amdgcn_mov_dpp(x, 0x120 + N, 0xf, 0xf, false);
}
template <int N>
__device__ __forceinline__ float turned(float x) {
    return __int_as_float(turned<N>(__float_as_int(x)));
}
template <int N>
__device__ __forceinline__ double turned(double x) {
    return __hiloint2double(turned<N>(__double2hiint(x)), turned<N>(__double2loint(x)));
}
__device__ __forceinline__ float max_row(float x) { /* of 16 lanes */
    x = max3(x, turned<8>(x), x);
    x = max3(x, turned<4>(x), x);
    x = max3(x, turned<2>(x), x);
    return max3(x, turned<1>(x), x);
}
__device__ __forceinline__ double sum_wave(double x) {
    x += turned<8>(x);
    x += turned<4>(x);
    x += turned<2>(x);
    x += turned<1>(x);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

/* What the first launch leaves of a row: block maxima (NaN where an id's logit is NaN or +inf), and of each wave the largest
 * logit and the sum of exp(l - that one). */
struct WaveSum {
    double sum, top;
};
struct Sums {
    float *top;
    WaveSum *sum;
    uint32_t blocks, sums; /* of a row */
};

/* A wave takes U times 256 ids of the row: no exchange with the others. 128 rows of 151936, 78 MB, 20 us, 3.9 TB/s: 13 us of VALU
 * work, most of it on 64 bits, beside 13.8 of reading alone, which waves in several rounds overlap in part. */
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
        float m = max3(max3(l[u][0], l[u][1], l[u][2]), l[u][3], l[u][3]);
        bool bad = false;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) bad = bad || !(l[u][e] < INFINITY);
        m = max_row(m);
        const uint64_t those = __ballot(bad);
        const uint32_t block = (wave * U + u) * (64 / BM_LANES) + lane / BM_LANES;
        if (lane % BM_LANES == 0 && block < s.blocks) s.top[(size_t)r * s.blocks + block] = those ? __builtin_nanf("") : m;
        top = fmaxf(top, m);
    }
#pragma unroll
    for (int off = BM_LANES; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
    const double off = top == -INFINITY ? 0.0 : (double)top; /* all masked: as at -700 each, and next to nothing in the row */
    double sum = 0.0, lead = EXP_LEAD;
    asm("" : "+v"(lead));
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) sum += exp_of((double)l[u][e] - off, lead);
    sum = sum_wave(sum);
    if (lane == 0) s.sum[(size_t)r * s.sums + wave] = WaveSum{sum, (double)top};
}

/* The `most`-th largest of some keys of which no two are equal but zeros: of keys[0 .. n), which all threads have written; 0 if
 * there are fewer. Every wave finds it for itself: no barrier. */
template <typename K>
__device__ __forceinline__ K kth_of(const K *keys, uint32_t n, uint32_t most) {
    K found = {};
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        const K mine = keys[i0 + threadIdx.x % 64];
        uint32_t rank = 0;
#pragma unroll 16
        for (uint32_t i = 0; i < n; ++i) rank += keys[i] > mine;
        const uint64_t hit = __ballot(rank == most - 1 && some(mine));
        if (hit) found = keys[i0 + __ffsll((unsigned long long)hit) - 1];
    }
    return found;
}

/* The `most` largest keys of list[0 .. m), descending, into best; returns their number. Until a list has BM_WG keys: of each
 * thread's keys the largest, of these the most-th largest, and only keys that are no smaller go on: those of `most` threads
 * at most, to the other of two lists (list, other) in turn. Then each key is put where its rank says. Begins with a
 * barrier, and ends with one. */
template <typename K>
__device__ __forceinline__ uint32_t best_of(K *list, K *other, uint32_t m, uint32_t most, K *keys, K *best, uint32_t *count) {
    const uint32_t tid = threadIdx.x;
    const K zero = {};
    __syncthreads();
    while (m > BM_WG) {
        K mine = zero;
        for (uint32_t i = tid; i < m; i += BM_WG) mine = list[i] > mine ? list[i] : mine;
        keys[tid] = mine;
        if (tid == 0) *count = 0;
        __syncthreads();
        const K least = kth_of(keys, BM_WG, most);
        for (uint32_t i = tid; i < m; i += BM_WG)
            if (!(least > list[i])) other[atomicAdd(count, 1u)] = list[i];
        __syncthreads();
        m = *count;
        K *x = list;
        list = other;
        other = x;
        __syncthreads();
    }
    if (tid < m) {
        const K mine = list[tid];
        uint32_t rank = 0;
#pragma unroll 16
        for (uint32_t i = 0; i < m; ++i) rank += list[i] > mine;
        if (rank < most) best[rank] = mine;
    }
    __syncthreads();
    return min(m, most);
}
/* LDS of the lists: the first one's keys, and what of it can go on. */
__host__ __device__ inline uint32_t list_next(uint32_t first, uint32_t most) { return most * ((first + BM_WG - 1) / BM_WG); }
/* Columns that a row's blocks are dealt to, and of whose maxima the select-th largest bounds the list: 64, one per lane, where
 * that keeps lists short. */
__host__ __device__ inline uint32_t columns_of(uint32_t blocks, uint32_t select) { return select <= 32 && blocks <= 4096 ? 64 : BM_WG; }

/* A workgroup per row: its `select` best ids and their values. What the row's blocks have is requested at once; the best
 * blocks' logits are on their way while the sums are joined. Bound by its chain of two trips to memory, eight barriers and
 * three rankings: 8 us, for 4 rows or 128. */
__global__ __launch_bounds__(BM_WG) void k_beam_rows(BeamArgs a, Sums s, double *value, uint32_t *id) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ double sums[BM_WAVES];
    __shared__ uint64_t keys[BM_WG], best[MAX_SELECT], blocks[MAX_SELECT];
    __shared__ uint32_t counts[3];
    uint64_t *list = (uint64_t *)lds, *other = list + a.select * BM_BLOCK;
    const uint32_t r = blockIdx.x, tid = threadIdx.x, columns = columns_of(s.blocks, a.select);
    const float *row = a.logits + (size_t)r * a.stride, *bt = s.top + (size_t)r * s.blocks;
    const float score = a.score[r];
    value += (size_t)r * a.select;
    id += (size_t)r * a.select;
    const bool done = a.done && a.done[r];
    int bad = !(score < INFINITY);
    /* the thread's blocks, BT of them in registers, and sums: one trip to memory for vocabularies of up to 262144 ids */
    constexpr uint32_t BT = 16, ST = 3;
    float t[BT];
    WaveSum ws[ST];
    const WaveSum *sum_row = s.sum + (size_t)r * s.sums;
#pragma unroll
    for (uint32_t k = 0; k < BT; ++k) t[k] = !done && tid + k * BM_WG < s.blocks ? bt[tid + k * BM_WG] : -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < ST; ++k) ws[k] = !done && tid + k * BM_WG < s.sums ? sum_row[tid + k * BM_WG] : WaveSum{0.0, -INFINITY};
    auto block_key = [](float x, uint32_t i) { return x == -INFINITY ? 0 : key_of(x, i); };
    uint64_t mine = 0;
    auto look = [&](float x, uint32_t i) {
        bad |= !(x < INFINITY);
        const uint64_t k = block_key(x, i);
        mine = k > mine ? k : mine;
    };
#pragma unroll
    for (uint32_t k = 0; k < BT; ++k) look(t[k], tid + k * BM_WG);
    if (!done)
        for (uint32_t i = tid + BT * BM_WG; i < s.blocks; i += BM_WG) look(bt[i], i);
    keys[tid] = mine;
    if (tid < 3) counts[tid] = 0;
    bad = __syncthreads_or(bad);
    if (columns == 64 && tid < 64) {
#pragma unroll
        for (uint32_t w = 1; w < BM_WAVES; ++w) mine = keys[w * 64 + tid] > mine ? keys[w * 64 + tid] : mine;
        keys[tid] = mine;
    }
    __syncthreads();
    if (bad && tid == 0) *a.flag = 1;
    auto finish = [&](bool some) { /* without a choice: the one of a row that is done, or none */
        for (uint32_t k = tid; k < a.select; k += BM_WG) {
            value[k] = some && k == 0 ? (double)score : -INFINITY;
            id[k] = a.pad;
        }
    };
    if (bad || score == -INFINITY || done) return finish(!bad && score > -INFINITY);
    /* the blocks that are no smaller than the select-th of the columns' maxima, and the best of them */
    const uint64_t least = max(kth_of(keys, columns, a.select), (uint64_t)1);
    auto put = [&](float x, uint32_t i) {
        const uint64_t k = block_key(x, i);
        if (k >= least) list[atomicAdd(&counts[0], 1u)] = k;
    };
#pragma unroll
    for (uint32_t k = 0; k < BT; ++k) put(t[k], tid + k * BM_WG);
    for (uint32_t i = tid + BT * BM_WG; i < s.blocks; i += BM_WG) put(bt[i], i);
    __syncthreads();
    const uint32_t listed = counts[0], nb = best_of(list, other, listed, a.select, keys, blocks, &counts[2]);
    if (!nb) return finish(false); /* all masked */
    const double top = (double)logit_of(blocks[0]);
    /* their ids, BM_WG / BM_LANES blocks at a time, a lane four */
    const float low = nb == a.select ? logit_of(blocks[nb - 1]) : -FLT_MAX;
    auto load = [&](uint32_t b, float(&l)[4]) {
        const uint32_t i = b < nb ? id_of(blocks[b]) * BM_BLOCK + 4 * (tid % BM_LANES) : a.vocab;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) l[e] = i + e < a.vocab ? row[i + e] : -INFINITY;
        return i;
    };
    float l[4];
    uint32_t i = load(tid / BM_LANES, l);
    double sum = 0.0;
    auto add = [&](const WaveSum &w) { sum += w.sum * exp(w.top - top); }; /* a second exp_of would double its error */
#pragma unroll
    for (uint32_t k = 0; k < ST; ++k) add(ws[k]);
    for (uint32_t i = tid + ST * BM_WG; i < s.sums; i += BM_WG) add(sum_row[i]);
    sum = sum_wave(sum);
    if (tid % 64 == 0) sums[tid / 64] = sum;
    for (uint32_t b = tid / BM_LANES; b < nb; b += BM_WG / BM_LANES) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (l[e] >= low) list[atomicAdd(&counts[1], 1u)] = key_of(l[e], i + e);
        i = load(b + BM_WG / BM_LANES, l);
    }
    __syncthreads();
    sum = sums[0];
#pragma unroll
    for (uint32_t w = 1; w < BM_WAVES; ++w) sum += sums[w];
    const uint32_t n = best_of(list, other, counts[1], a.select, keys, best, &counts[2]);
    if (tid < a.select) {
        const uint64_t b = tid < n ? best[tid] : 0;
        value[tid] = b ? (double)score + ((double)logit_of(b) - (top + log(sum))) : -INFINITY;
        id[tid] = id_of(b);
    }
}

/* A workgroup per result where there are histories, else per group: the best of the group's candidates, and its results. What the
 * results may need of the candidates and rows is requested with their values. Bound by two trips to memory and the ranking: 4.2 us
 * for 32 candidates, 7.2 for 128 of each of 16 groups. */
template <bool MANY> /* more than BM_WG candidates */
__global__ __launch_bounds__(BM_WG) void k_beam_join(BeamArgs a, const double *value, const uint32_t *id, uint32_t per) {
    __shared__ uint64_t values[BM_WG], best[MAX_SELECT];
    __shared__ uint32_t which[MAX_SELECT], ids[BM_WG];
    __shared__ int lengths[MAX_BEAMS];
    __shared__ uint8_t over_rows[MAX_BEAMS];
    const uint32_t g = blockIdx.x / per, tid = threadIdx.x, n = a.beams * a.select;
    const size_t at = (size_t)g * n;
    if (tid < a.beams) {
        over_rows[tid] = a.done ? a.done[g * a.beams + tid] : 0;
        lengths[tid] = a.history ? a.length[g * a.beams + tid] : 0;
    }
    uint32_t found;
    if constexpr (!MANY) {
        const double x = tid < n ? value[at + tid] : -INFINITY;
        const uint64_t mine = x > -INFINITY ? order_of(x) : 0;
        values[tid] = mine;
        if (tid < n) ids[tid] = id[at + tid];
        const int all = __syncthreads_count(mine != 0);
        if (mine) {
            uint32_t rank = 0;
#pragma unroll 16
            for (uint32_t i = 0; i < n; ++i) rank += values[i] > mine || (values[i] == mine && i < tid);
            if (rank < a.select) {
                which[rank] = tid;
                best[rank] = mine;
            }
        }
        __syncthreads();
        found = min((uint32_t)all, a.select);
    } else {
        extern __shared__ __attribute__((aligned(16))) unsigned char lds[]; /* the lists */
        __shared__ Cand keys[BM_WG], most[MAX_SELECT];
        __shared__ uint32_t count;
        if (tid == 0) count = 0;
        Cand *list = (Cand *)lds, *other = list + list_next(n, a.select);
        const auto cand = [&](uint32_t i) {
            const double v = value[at + i];
            return v > -INFINITY ? Cand{order_of(v), ~(uint64_t)i} : Cand{0, 0};
        };
        Cand mine = {0, 0};
        for (uint32_t i = tid; i < n; i += BM_WG) {
            const Cand c = cand(i);
            mine = c > mine ? c : mine;
        }
        keys[tid] = mine;
        __syncthreads();
        const Cand kth = kth_of(keys, BM_WG, a.select), least = some(kth) ? kth : Cand{1, 0};
        for (uint32_t i = tid; i < n; i += BM_WG) {
            const Cand c = cand(i);
            if (!(least > c)) list[atomicAdd(&count, 1u)] = c;
        }
        __syncthreads();
        found = best_of(list, other, count, a.select, keys, most, &count);
        if (tid < found) {
            which[tid] = (uint32_t)~most[tid].i;
            best[tid] = most[tid].v;
        }
        __syncthreads();
    }
    for (uint32_t k = blockIdx.x % per; k < a.select; k += per) {
        const uint32_t o = g * a.select + k, w = k < found ? which[k] : 0, row = w / a.select;
        const bool none = k >= found;
        const uint32_t r = none ? 0 : g * a.beams + row, token = none ? NONE : MANY ? id[at + w] : ids[w];
        const bool over = !none && over_rows[row];
        if (tid == 0) {
            a.parent[o] = none ? -1 : (int)r;
            a.token[o] = token;
            a.score_out[o] = none ? -INFINITY : (float)value_of(best[k]);
            if (a.done_out) a.done_out[o] = none || over || (a.eos != NONE && token == a.eos);
        }
        if (!a.history) continue;
        const int have = none ? 0 : lengths[row];
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

/* Loads of four ids a lane in the first launch. 128 rows of 151936: 1 24.6 us, 2 21.2, 4 21.0; 4 rows: 3.2, 3.3, 3.7. */
uint32_t wave_loads(const BeamArgs &a) { return (uint64_t)a.groups * a.beams * a.vocab >= (1u << 21) ? 2 : 1; }
Sums sums_of(const BeamArgs &a) {
    Sums s;
    s.top = nullptr;
    s.sum = nullptr;
    const uint32_t per = 256 * wave_loads(a);
    s.blocks = (a.vocab + BM_BLOCK - 1) / BM_BLOCK;
    s.sums = (a.vocab + per - 1) / per;
    return s;
}

}  // namespace

size_t beam_workspace(const BeamArgs &a) {
    const size_t rows = (size_t)a.groups * a.beams; /* sums of one load each: enough for fewer rows or ids too */
    return rows * ((size_t)a.select * 12 + (a.vocab + 255) / 256 * sizeof(WaveSum) + sums_of(a).blocks * 4);
}

hipError_t launch_beam(const BeamArgs &a, void *ws, hipStream_t st) {
    const uint32_t rows = a.groups * a.beams, U = wave_loads(a);
    Sums s = sums_of(a);
    double *value = (double *)ws;
    s.sum = (WaveSum *)(value + (size_t)rows * a.select);
    s.top = (float *)(s.sum + (size_t)rows * s.sums);
    uint32_t *id = (uint32_t *)(s.top + (size_t)rows * s.blocks);
    const bool wide = !(((uintptr_t)a.logits | (rows > 1 ? a.stride * 4 : 0)) & 15);
    const dim3 grid((s.sums + BM_WAVES - 1) / BM_WAVES, rows);
#define SMQ_BEAM(U)                                                                                        \
    do {                                                                                                   \
        if (wide) hipLaunchKernelGGL((k_beam_sums<U, true>), grid, dim3(BM_WG), 0, st, a, s);              \
        else hipLaunchKernelGGL((k_beam_sums<U, false>), grid, dim3(BM_WG), 0, st, a, s);                  \
    } while (0)
    if (U == 2) SMQ_BEAM(2);
    else SMQ_BEAM(1);
#undef SMQ_BEAM
    const uint32_t first = a.select * BM_BLOCK, n = a.beams * a.select;
    hipLaunchKernelGGL(k_beam_rows, dim3(rows), dim3(BM_WG), (first + list_next(first, a.select)) * 8, st, a, s, value, id);
    const uint32_t per = a.history ? a.select : 1, list = list_next(n, a.select);
    const dim3 joins(a.groups * per);
    if (n > BM_WG)
        hipLaunchKernelGGL((k_beam_join<true>), joins, dim3(BM_WG), (list + list_next(list, a.select)) * sizeof(Cand), st, a, value,
                           id, per);
    else
        hipLaunchKernelGGL((k_beam_join<false>), joins, dim3(BM_WG), 0, st, a, value, id, per);
    return hipGetLastError();
}

}  // namespace smq
