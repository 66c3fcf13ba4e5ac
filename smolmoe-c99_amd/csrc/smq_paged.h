/* Device helpers of the paged KV cache's kernels: sequences, rows and pages of a checked batch. */
#ifndef SMQ_PAGED_H
#define SMQ_PAGED_H

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

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

/* Tile t of the batch: sequence and first row. Uniform; false behind the last tile. */
__device__ __forceinline__ bool find_tile(const PagedArgs &a, uint32_t t, uint32_t tile_rows, uint32_t &seq, uint32_t &row0) {
    const uint32_t lane = threadIdx.x % 64, G = a.heads / a.kv_heads;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
        const uint32_t s = s0 + lane;
        uint32_t n = 0;
        if (s < a.seqs) {
            const int b0 = a.begin[s], b1 = a.begin[s + 1];
            if (b0 < 0 || b1 < b0 || (uint32_t)b1 > a.tokens) *a.flag = 1;
            else n = ((uint32_t)(b1 - b0) * G + tile_rows - 1) / tile_rows;
        }
        uint32_t sum = n;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const uint32_t x = __shfl_up(sum, off);
            sum += (int)lane >= off ? x : 0;
        }
        const uint64_t past = __ballot(before + sum > t);
        if (past) {
            const int w = __ffsll((unsigned long long)past) - 1;
            const uint32_t upto = before + __builtin_amdgcn_readlane(sum, w) - __builtin_amdgcn_readlane(n, w);
            seq = s0 + (uint32_t)w;
            row0 = (t - upto) * tile_rows;
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

/* Row r of a sequence and KV head, in q and att. */
__device__ __forceinline__ size_t row_at(const PagedArgs &a, const Seq &sq, uint32_t kh, uint32_t r) {
    const uint32_t G = a.heads / a.kv_heads;
    return ((size_t)(sq.begin + (int)(r / G)) * a.heads + (size_t)kh * G + r % G) * a.head_dim;
}

}  // namespace
}  // namespace smq

#endif
