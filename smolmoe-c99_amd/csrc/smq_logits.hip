/* Rows of logits before the choice of a token on gfx950: penalties over a history, biases, grammar masks, and the
 * greedy choice (include/smq.h has the formulas).
 *
 * One pass: a workgroup takes a span of ids of one row, requests its logits, counts the row's whole history (and adds up
 * its biases) in LDS where they fall into the span meanwhile, and writes the adjusted logits with the span's best
 * candidate; a second launch, a wave per row, joins the candidates. */
#include "smq_device.h"

namespace smq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr uint32_t LG_WG = 256, LG_WAVES = LG_WG / 64;
constexpr uint32_t NONE = 0xffffffffu;

/* Of some ids that may be taken: the lowest one and whether its logit is a NaN, and the lowest one of the largest logit
 * above -inf. The choice: the lowest if its logit is a NaN or none is above -inf, else the largest. */
struct Part {
    float best;
    uint32_t id, first, first_nan;
};
__device__ __forceinline__ void join(Part &a, const Part &b) {
    const bool take = b.best > a.best || (b.best == a.best && b.id < a.id);
    a.best = take ? b.best : a.best;
    a.id = take ? b.id : a.id;
    a.first_nan = b.first < a.first ? b.first_nan : a.first_nan;
    a.first = min(a.first, b.first);
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
__device__ __forceinline__ Part nothing() { return {-INFINITY, NONE, NONE, 0}; }

/* [begin[r], begin[r + 1]) cut to the list's count entries. */
__device__ __forceinline__ void list_range(const int32_t *begin, uint32_t r, uint32_t count, uint32_t &b, uint32_t &e) {
    const int x = begin[r], y = begin[r + 1];
    b = x < 0 ? 0 : min((uint32_t)x, count);
    e = y < 0 ? 0 : min((uint32_t)y, count);
}

/* A thread has ids v0 + 1024 u + 4 tid .. + 3 of the span, u < SPAN / 1024. WIDE: rows of 16-byte aligned quadruples;
 * else single words.
 *
 * Two round trips to memory: the row's list bounds, penalties and mask (and the logits, which need none of them), then the
 * lists' first entries and the mask's words; everything after works in LDS and registers. The history is counted with
 * integers (no order); the thread that counts an id first puts it on a list, and the ids of the list, few, are adjusted by
 * a thread each: in the pass over all ids some lane of almost every wave would divide.
 *
 * 64 rows of 151936, 79 MB, 31 us, 2.5 TB/s with the second launch (4 us): bound by the latency of these trips in three
 * rounds of workgroups; histories of 2000, biases and masks are 4 us of it. One row: 9 us, two launches. */
template <uint32_t SPAN, bool WIDE>
__global__ __launch_bounds__(LG_WG) void k_logits(LogitArgs a, Part *parts) {
    constexpr uint32_t U = SPAN / (4 * LG_WG), AHEAD = 2;
    __shared__ __attribute__((aligned(16))) uint32_t count[SPAN]; /* then, of counted ids, the adjusted logit's bits + 1 */
    __shared__ __attribute__((aligned(16))) float add[SPAN];
    __shared__ uint16_t list[SPAN];
    __shared__ uint32_t ids[LG_WG], found[LG_WAVES], listed;
    __shared__ float vals[LG_WG];
    __shared__ Part best[LG_WAVES];
    const uint32_t tid = threadIdx.x, r = blockIdx.y, v0 = blockIdx.x * SPAN, left = a.vocab - v0; /* ids from v0 on */
    const float *row = a.logits + (size_t)r * a.stride + v0;
    f4 l[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t i = u * 4 * LG_WG + 4 * tid;
        if (WIDE && i + 4 <= left) {
            l[u] = *(const f4 *)(row + i);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) l[u][e] = i + e < left ? row[i + e] : 0.0f;
        }
    }
    uint32_t hb = 0, he = 0, bb = 0, be = 0;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (a.history) {
        list_range(a.history_begin, r, a.history_count, hb, he);
        rep = a.penalty[3 * (size_t)r];
        pres = a.penalty[3 * (size_t)r + 1];
        freq = a.penalty[3 * (size_t)r + 2];
    }
    if (a.bias_ids) list_range(a.bias_begin, r, a.bias_count, bb, be);
    bool masked = false, none = false;
    uint32_t may[U]; /* the mask's words of the quadruples */
    if (a.allowed) {
        const int m = a.mask_row ? a.mask_row[r] : (int)r;
        none = m >= 0 && (uint32_t)m >= a.allowed_rows;
        if (none && tid == 0) *a.flag = 1;
        masked = m >= 0 && !none;
        const uint32_t *mask = a.allowed + (size_t)(masked ? m : 0) * ((a.vocab + 31) / 32) + v0 / 32;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = u * 4 * LG_WG + 4 * tid;
            may[u] = masked && i < left ? mask[i / 32] : 0;
        }
    }
    /* a quadruple of the history; the last one may be shorter */
    const uint32_t quads = he > hb ? (he - hb + 3) / 4 : 0;
    auto history = [&](uint32_t i) {
        u4 v;
        if (hb + 4 * i + 4 <= he) {
            v = *(const u4u *)(a.history + hb + 4 * i);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = hb + 4 * i + e < he ? a.history[hb + 4 * i + e] : NONE;
        }
        return v;
    };
    u4 h[AHEAD];
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (tid + k * LG_WG < quads) h[k] = history(tid + k * LG_WG);
    uint32_t bias_id = NONE;
    float bias = 0.0f;
    if (tid < be - bb && be > bb) {
        bias_id = a.bias_ids[bb + tid];
        bias = a.bias[bb + tid];
    }
    if (tid == 0) listed = 0;
    if (quads) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) *(u4 *)&count[u * 4 * LG_WG + 4 * tid] = u4{};
        __syncthreads();
        auto tally = [&](const u4 &v) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t i = v[e] - v0;
                if (i < SPAN && v[e] < a.vocab && !atomicAdd(&count[i], 1u)) list[atomicAdd(&listed, 1u)] = (uint16_t)i;
            }
        };
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k)
            if (tid + k * LG_WG < quads) tally(h[k]);
        for (uint32_t i = tid + AHEAD * LG_WG; i < quads; i += LG_WG) tally(history(i));
        __syncthreads();
        for (uint32_t k = tid; k < listed; k += LG_WG) {
            const uint32_t i = list[k];
            const float x = row[i], y = x > 0.0f ? x / rep : x * rep, t = (float)count[i] * freq;
            const float z = y - (t + pres);
            count[i] = z == z ? __float_as_uint(z) + 1 : 0x7fc00001u;
        }
    }
    if (be > bb) {
        /* 256 entries at a time, those of the span put together in the order of the list; the first one of an id adds up
         * the later ones, so that the same id twice gives the same bits on every run */
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) *(f4 *)&add[u * 4 * LG_WG + 4 * tid] = f4{};
        for (uint32_t i0 = bb; i0 < be; i0 += LG_WG) {
            if (i0 != bb) {
                bias_id = i0 + tid < be ? a.bias_ids[i0 + tid] : NONE;
                bias = i0 + tid < be ? a.bias[i0 + tid] : 0.0f;
            }
            const uint32_t id = bias_id - v0;
            const bool in = id < SPAN && bias_id < a.vocab;
            const uint64_t those = __ballot(in);
            __syncthreads();
            if (tid % 64 == 0) found[tid / 64] = (uint32_t)__popcll(those);
            __syncthreads();
            uint32_t at = (uint32_t)__popcll(those & ((1ull << tid % 64) - 1)), total = 0;
#pragma unroll
            for (uint32_t w = 0; w < LG_WAVES; ++w) {
                at += w < tid / 64 ? found[w] : 0;
                total += found[w];
            }
            if (!total) continue; /* uniform */
            if (in) {
                ids[at] = id;
                vals[at] = bias;
            }
            __syncthreads();
            if (tid < total) {
                const uint32_t mine = ids[tid];
                bool first = true;
                for (uint32_t j = 0; j < tid; ++j) first = first & (ids[j] != mine);
                if (first) {
                    float sum = add[mine] + vals[tid];
                    for (uint32_t j = tid + 1; j < total; ++j)
                        if (ids[j] == mine) sum += vals[j];
                    add[mine] = sum;
                }
            }
        }
    }
    __syncthreads();
    Part p = nothing();
    float *out = a.out ? a.out + (size_t)r * a.out_stride + v0 : nullptr;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t i = u * 4 * LG_WG + 4 * tid;
        f4 x = l[u];
        if (quads) {
            const u4 c = *(const u4 *)&count[i];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = c[e] ? __uint_as_float(c[e] - 1) : x[e];
        }
        if (be > bb) x += *(const f4 *)&add[i];
        uint32_t ok = none ? 0 : i + 4 <= left ? 15 : i < left ? (1u << (left - i)) - 1 : 0;
        if (masked) ok &= may[u] >> (i % 32);
        if (ok != 15) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = ok >> e & 1 ? x[e] : -INFINITY;
        }
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const bool take = x[e] > p.best; /* ids ascend: the lowest of equal ones stays; a NaN is not above */
            p.best = take ? x[e] : p.best;
            p.id = take ? v0 + i + e : p.id;
        }
        if (p.first == NONE && ok) {
            const uint32_t e = (uint32_t)__ffs(ok) - 1;
            const float y = e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3];
            p.first = v0 + i + e;
            p.first_nan = y != y;
        }
        if (out) {
            if (WIDE && i + 4 <= left) {
                __builtin_nontemporal_store(x, (f4 *)(out + i));
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (i + e < left) out[i + e] = x[e];
            }
        }
    }
    if (!parts) return;
    p = join_wave(p);
    if (tid % 64 == 0) best[tid / 64] = p;
    __syncthreads();
    if (tid == 0) {
        for (uint32_t w = 1; w < LG_WAVES; ++w) join(p, best[w]);
        parts[(size_t)r * gridDim.x + blockIdx.x] = p;
    }
}

__global__ __launch_bounds__(64) void k_logits_pick(const Part *parts, uint32_t n, uint32_t *token) {
    Part p = nothing();
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += 64) join(p, parts[(size_t)blockIdx.x * n + i]);
    p = join_wave(p);
    if (threadIdx.x == 0) token[blockIdx.x] = p.first_nan || p.id == NONE ? p.first : p.id;
}

/* Spans of 2048 where there are four or more a CU, else of 1024: each reads the row's whole history, and holds 23 KiB of LDS
 * where one of 1024 holds 13. 64 rows of 151936 with histories of up to 2000: spans of 1024 46 us, 2048 32, 4096 34. One row
 * with one of 600: 9 us with either. */
constexpr uint32_t WIDE_SPAN = 2048;
uint32_t span_of(uint32_t rows, uint32_t vocab) {
    return (uint64_t)rows * ((vocab + WIDE_SPAN - 1) / WIDE_SPAN) >= 1024 ? WIDE_SPAN : 1024;
}

}  // namespace

/* Enough for fewer rows or ids too, which may have more spans: below the line they are of half the size, 2046 at most. */
size_t logits_workspace(uint32_t rows, uint32_t vocab) {
    const uint32_t span = span_of(rows, vocab);
    const size_t parts = (size_t)rows * ((vocab + span - 1) / span);
    return (span == WIDE_SPAN && parts < 2046 ? 2046 : parts) * sizeof(Part);
}

hipError_t launch_logits(const LogitArgs &a, uint32_t *token, void *ws, hipStream_t s) {
    const uint32_t span = span_of(a.rows, a.vocab), n = (a.vocab + span - 1) / span;
    const bool wide = !(((uintptr_t)a.logits | (uintptr_t)a.out | (a.rows > 1 ? (a.stride | a.out_stride) * 4 : 0)) & 15);
    Part *parts = token ? (Part *)ws : nullptr;
    const dim3 grid(n, a.rows);
    if (span == WIDE_SPAN) {
        if (wide) hipLaunchKernelGGL((k_logits<WIDE_SPAN, true>), grid, dim3(LG_WG), 0, s, a, parts);
        else hipLaunchKernelGGL((k_logits<WIDE_SPAN, false>), grid, dim3(LG_WG), 0, s, a, parts);
    } else {
        if (wide) hipLaunchKernelGGL((k_logits<1024, true>), grid, dim3(LG_WG), 0, s, a, parts);
        else hipLaunchKernelGGL((k_logits<1024, false>), grid, dim3(LG_WG), 0, s, a, parts);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !token) return e;
    hipLaunchKernelGGL(k_logits_pick, dim3(a.rows), dim3(64), 0, s, parts, n, token);
    return hipGetLastError();
}

}  // namespace smq
