/* Paged KV cache on gfx950: RoPE and the store of new tokens (f32, f16, Q8), rows read back, and the attention of a
 * ragged batch of new tokens over the pages (include/smq.h has the layout of a page). */
#include <hip/hip_fp16.h>
#include <float.h>

#include "smq_device.h"

namespace smq {
namespace {

/* A page id of the table or -1 with the flag raised where it names no page. */
__device__ __forceinline__ int page_of(const PagedArgs &a, uint32_t s, uint32_t pos) {
    const int id = a.table[(size_t)s * a.table_stride + (pos >> a.shift)];
    if ((uint32_t)id < a.pages) return id;
    *a.flag = 1;
    return -1;
}

/* Sequence s's new tokens: rows begin .. begin + n at positions first .. first + n, of `length` positions. False, with
 * the flag raised, where begin does not ascend within 0 .. tokens. */
struct Seq {
    int begin, n, length;
    int64_t first;
};
__device__ __forceinline__ bool sequence(const PagedArgs &a, uint32_t s, Seq &q) {
    const int b0 = a.begin[s], b1 = a.begin[s + 1];
    if (b0 < 0 || b1 < b0 || (uint32_t)b1 > a.tokens) {
        *a.flag = 1;
        return false;
    }
    const int len = a.length[s];
    q.begin = b0;
    q.n = b1 - b0;
    q.length = len < 0 ? 0 : (uint32_t)len > a.limit ? (int)a.limit : len;
    q.first = (int64_t)len - q.n;
    return true;
}

/* Raises the flag where begin does not ascend within 0 .. tokens (rows may then belong to no sequence); by one workgroup
 * of a launch. */
__device__ __forceinline__ void check_begin(const PagedArgs &a, uint32_t tid, uint32_t threads) {
    for (uint32_t s = tid; s < a.seqs; s += threads) {
        const int b0 = a.begin[s], b1 = a.begin[s + 1];
        if (b0 < 0 || b1 < b0 || (uint32_t)b1 > a.tokens) *a.flag = 1;
    }
}

/* The sequence and position of row r; false where the row is padding or has no place (then with the flag). */
__device__ __forceinline__ bool place_of(const PagedArgs &a, uint32_t r, uint32_t &s, uint32_t &pos) {
    uint32_t lo = 0, hi = a.seqs; /* the first sequence that begins past r */
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.begin[mid] <= (int)r) lo = mid + 1;
        else hi = mid;
    }
    Seq q;
    if (!lo || a.begin[lo] <= (int)r) return false; /* behind the last sequence (lo == seqs) */
    s = lo - 1;
    if (!sequence(a, s, q)) return false;
    const int64_t p = q.first + (int)(r - (uint32_t)q.begin);
    if (p < 0 || p >= (int64_t)a.limit) {
        *a.flag = 1;
        return false;
    }
    pos = (uint32_t)p;
    return true;
}

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

/* One wave per row and head: 64 positions at a time, a running maximum and sum of the softmax in one pass. */
template <uint32_t TYPE>
__global__ __launch_bounds__(64) void k_paged_attend(PagedArgs a, const float *q, float *att) {
    __shared__ float qs[MAX_HEAD_DIM], ps[64];
    __shared__ size_t at_v[64];
    const uint32_t r = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, h = head / (a.heads / a.kv_heads);
    const uint32_t P = 1u << a.shift, hd = a.head_dim;
    uint32_t s, pos;
    float *out = att + ((size_t)r * a.heads + head) * hd;
    if (r == 0 && head == 0) check_begin(a, lane, 64);
    if (!place_of(a, r, s, pos)) {
        if ((int)r < a.begin[a.seqs])
            for (uint32_t d = lane; d < hd; d += 64) out[d] = 0.0f;
        return;
    }
    for (uint32_t d = lane; d < hd; d += 64) qs[d] = q[((size_t)r * a.heads + head) * hd + d];
    const float scale = 1.0f / sqrtf((float)hd);
    float m = -INFINITY, l = 0.0f, o[MAX_HEAD_DIM / 64] = {};
    const uint32_t low = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 <= pos; j0 += 64) {
        if (j0 + 64 <= low && j0 >= a.sinks) continue;
        const uint32_t j = j0 + lane;
        bool sees = j <= pos && (j >= low || j < a.sinks);
        const int page = sees ? page_of(a, s, j) : -1;
        sees = page >= 0;
        float x = -INFINITY;
        if (sees) {
            const uint32_t slot = j & (P - 1);
            const size_t ph = (size_t)page * a.kv_heads + h;
            float dot = 0.0f;
            for (uint32_t d = 0; d < hd; ++d)
                dot += qs[d] * element<TYPE>(a.keys, (ph * P + slot) * hd + d, a.ks, (ph * a.nb + d / 32) * P + slot);
            x = dot * scale;
            at_v[lane] = ph * hd * P + slot;
        }
        float mx = x;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        const float mn = fmaxf(m, mx);
        if (mn == -INFINITY) continue; /* nothing seen so far: uniform */
        const float alpha = __expf(m - mn), p = sees ? __expf(x - mn) : 0.0f;
        float sum = p;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
        l = l * alpha + sum;
        m = mn;
        ps[lane] = sees ? p : -1.0f;
        __syncthreads();
        for (uint32_t u = 0; u * 64 + lane < hd; ++u) {
            const uint32_t d = u * 64 + lane;
            float acc = o[u] * alpha;
            for (uint32_t i = 0; i < 64; ++i) {
                if (ps[i] < 0.0f) continue; /* not seen: its value never matters */
                const size_t sh = at_v[i] / ((size_t)hd * P), slot = at_v[i] % P;
                acc += ps[i] * element<TYPE>(a.values, at_v[i] + (size_t)d * P, a.vs, (sh * a.nb + d / 32) * P + slot);
            }
            o[u] = acc;
        }
        __syncthreads();
    }
    for (uint32_t u = 0; u * 64 + lane < hd; ++u) out[u * 64 + lane] = l > 0.0f ? o[u] / l : m == -INFINITY ? 0.0f : l;
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

size_t paged_attention_workspace(const PagedArgs &) { return 0; }

hipError_t launch_paged_attention(const PagedArgs &a, const float *q, float *att, void *, size_t, hipStream_t s) {
    SMQ_PAGED(k_paged_attend, dim3(a.tokens, a.heads), dim3(64), q, att);
    return hipGetLastError();
}

}  // namespace smq
