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

/* Sequence s's new tokens: rows begin .. begin + n at positions first .. first + n. False, with the flag raised, where
 * begin does not ascend within 0 .. tokens. */
struct Seq {
    int begin, n, first;
};
/* length - n without overflow: what no position of the n tokens (below 2^23) can make a place (0 .. 2^20) stays none. */
__device__ __forceinline__ int first_position(int length, int n) { return min(max(length, -(1 << 25)), 1 << 30) - n; }
__device__ __forceinline__ bool sequence(const PagedArgs &a, uint32_t s, Seq &q) {
    const int b0 = a.begin[s], b1 = a.begin[s + 1];
    if (b0 < 0 || b1 < b0 || (uint32_t)b1 > a.tokens) {
        *a.flag = 1;
        return false;
    }
    q.begin = b0;
    q.n = b1 - b0;
    q.first = first_position(a.length[s], q.n);
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

/* The sequence and position of row r (of a whole wave: uniform); false where the row is padding or has no place (then with the flag). */
__device__ __forceinline__ bool place_of(const PagedArgs &a, uint32_t r, uint32_t &s, uint32_t &pos) {
    uint32_t lo = 0, hi = a.seqs; /* the first sequence that begins past r: halved to 64, which the lanes look at */
    while (hi - lo > 64) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.begin[mid] <= (int)r) lo = mid + 1;
        else hi = mid;
    }
    const uint32_t lane = threadIdx.x % 64;
    lo += (uint32_t)__popcll(__ballot(lo + lane < hi && a.begin[lo + min(lane, hi - lo - 1)] <= (int)r));
    Seq q;
    if (!lo || a.begin[lo] <= (int)r) return false; /* behind the last sequence (lo == seqs) */
    s = lo - 1;
    if (!sequence(a, s, q)) return false;
    const int p = q.first + (int)(r - (uint32_t)q.begin);
    if ((uint32_t)p >= a.limit) {
        *a.flag = 1;
        return false;
    }
    pos = (uint32_t)p;
    return true;
}

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

/* Row r of a sequence (its first token: begin) and KV head, in q and att. */
__device__ __forceinline__ size_t row_at(const PagedArgs &a, int begin, uint32_t kh, uint32_t r) {
    const uint32_t G = a.heads / a.kv_heads;
    return ((size_t)(begin + (int)(r / G)) * a.heads + (size_t)kh * G + r % G) * a.head_dim;
}

}  // namespace
}  // namespace smq

#endif
