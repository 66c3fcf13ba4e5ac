/* Pages of the paged KV cache on gfx950: the next tables of a set of sequences (shared, copied, fresh and freed pages), the
 * copies over all layers, and accepted drafts moved to the front of their sequence's new tokens (include/smq.h). */
#include "smq_paged.h"

namespace smq {
namespace {

constexpr uint32_t PG_WG = 256, PG_CHUNK = 1024; /* pages of a chunk */

/* New row d, cut to what the tables hold. */
struct NewRow {
    int parent;
    uint32_t full, part, held; /* full pages, positions of the next one, entries */
};
__device__ __forceinline__ NewRow new_row(const ForkArgs &a, uint32_t d, bool flag) {
    NewRow r;
    bool bad = false;
    r.parent = a.parent[d];
    if (r.parent < -1 || r.parent >= (int)a.old_seqs) {
        bad = true;
        r.parent = -1;
    }
    const uint64_t most = (uint64_t)a.table_stride << a.shift;
    const int have = r.parent >= 0 ? min(max(a.held[r.parent], 0), (int)a.table_stride) : 0;
    int keep = a.keep[d], room = a.room[d];
    bad = bad || keep < 0 || room < 0 || keep > room || (uint64_t)(uint32_t)max(room, 0) > most ||
          (uint64_t)(uint32_t)max(keep, 0) > (uint64_t)have << a.shift;
    keep = (int)min((uint64_t)(uint32_t)max(keep, 0), (uint64_t)have << a.shift);
    room = (int)min((uint64_t)(uint32_t)max(max(room, keep), 0), most);
    const uint32_t P = 1u << a.shift;
    r.full = (uint32_t)keep >> a.shift;
    r.part = (uint32_t)keep & (P - 1);
    r.held = (uint32_t)(((uint64_t)(uint32_t)room + P - 1) >> a.shift);
    if (bad && flag) *a.flag = 1;
    return r;
}
/* Entries of old row s. */
__device__ __forceinline__ uint32_t old_held(const ForkArgs &a, uint32_t s, bool flag) {
    const int held = a.held[s];
    if (flag && (held < 0 || held > (int)a.table_stride)) *a.flag = 1;
    return (uint32_t)min(max(held, 0), (int)a.table_stride);
}
template <uint32_t WAVES, typename T>
__device__ __forceinline__ T block_sum(T x, T *lds) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2) x += __shfl_xor(x, off);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    T t = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) t += lds[w];
    return t;
}
/* The sum of x over the threads before this one; all: over all. */
template <uint32_t WAVES>
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *lds, uint32_t &all) {
    uint32_t upto = x;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const uint32_t y = __shfl_up(upto, off);
        upto += (int)(threadIdx.x % 64) >= off ? y : 0;
    }
    __syncthreads();
    if (threadIdx.x % 64 == 63) lds[threadIdx.x / 64] = upto;
    __syncthreads();
    uint32_t before = upto - x;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        before += w < threadIdx.x / 64 ? lds[w] : 0;
        all += lds[w];
    }
    return before;
}

/* Few rows and pages: one workgroup, the pages' holders in LDS. Bound by three trips to memory (row arrays, holders and old
 * entries; the parents' entries; the results) and ten barriers: four rows 6.8 us, where the four launches below take 11; 64 rows
 * of 14 entries 9.1, 15; 256 of 32, 7118 pages 13.9, 14.2; but 256 of 63 18.6, 14.6. */
constexpr uint32_t SMALL_WG = 1024, SMALL_WAVES = SMALL_WG / 64, SMALL_PAGES = 8192, SMALL_ROWS = 256, SMALL_ENTRIES = 8192;
__global__ __launch_bounds__(SMALL_WG) void k_fork_small(ForkArgs a) {
    __shared__ int holders[SMALL_PAGES];
    __shared__ uint32_t in_part[SMALL_PAGES / 32], free_words[SMALL_PAGES / 32], word_rank[SMALL_PAGES / 32];
    __shared__ int parents[SMALL_ROWS], last[SMALL_ROWS];
    __shared__ uint32_t olds[SMALL_ROWS], full[SMALL_ROWS], held[SMALL_ROWS], from[SMALL_ROWS], rank[SMALL_ROWS + 1];
    __shared__ uint32_t lds[SMALL_WAVES];
    const uint32_t tid = threadIdx.x, words = (a.pages + 31) / 32, entries = a.old_seqs * a.table_stride;
    constexpr uint32_t EARLY = 4; /* old entries of a thread that are requested with the row arrays */
    uint32_t early[EARLY];
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k) early[k] = tid + k * SMALL_WG < entries ? (uint32_t)a.table[tid + k * SMALL_WG] : 0;
    NewRow row = {};
    if (tid < a.old_seqs) olds[tid] = old_held(a, tid, true);
    if (tid < a.seqs) {
        row = new_row(a, tid, true);
        parents[tid] = row.parent;
        full[tid] = row.full;
        held[tid] = row.held;
        last[tid] = -1;
    }
    for (uint32_t i = tid; i < a.pages; i += SMALL_WG) {
        const int n = a.refs[i];
        holders[i] = n;
        if (n < 0) *a.flag = 1;
    }
    if (tid < words) in_part[tid] = 0;
    __syncthreads();
    const float inv = 1.0f / (float)a.table_stride;
    auto row_of = [&](uint32_t i) { return (uint32_t)(((float)i + 0.5f) * inv); }; /* i / stride: below 2^14, where this is exact */
    auto give_up = [&](uint32_t i, uint32_t id) {
        const uint32_t s = row_of(i), x = i - s * a.table_stride;
        if (x >= olds[s]) return;
        if (id < a.pages) atomicSub(&holders[id], 1);
        else *a.flag = 1;
    };
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k)
        if (tid + k * SMALL_WG < entries) give_up(tid + k * SMALL_WG, early[k]);
    for (uint32_t i = tid + EARLY * SMALL_WG; i < entries; i += SMALL_WG) give_up(i, (uint32_t)a.table[i]);
    __syncthreads();
    for (uint32_t i = tid; i < a.pages; i += SMALL_WG)
        if (holders[i] < 0) {
            *a.flag = 1;
            holders[i] = 0;
        }
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = tid; i < a.seqs * a.table_stride; i += SMALL_WG) {
        const uint32_t d = row_of(i), x = i - d * a.table_stride;
        const uint32_t id = x < full[d] ? (uint32_t)a.table[(size_t)parents[d] * a.table_stride + x] : a.pages;
        if (id < a.pages) atomicAdd(&holders[id], 1);
        if (x < full[d] || x >= held[d]) a.table_out[i] = id < a.pages ? (int)id : -1;
    }
    if (tid < a.seqs && row.part) {
        const uint32_t id = (uint32_t)a.table[(size_t)row.parent * a.table_stride + row.full];
        if (id < a.pages) {
            last[tid] = (int)id;
            atomicOr(&in_part[id / 32], 1u << (id % 32));
        }
    }
    __syncthreads();
    /* rows: the first one that takes a page in part keeps it, if nothing else holds it (the most of SMALL_ROWS - row there) */
    uint32_t need = 0;
    bool mine = tid < a.seqs && last[tid] >= 0 && holders[last[tid]] == 0;
    __syncthreads();
    if (mine) atomicMax(&holders[last[tid]], (int)(SMALL_ROWS - tid));
    __syncthreads();
    mine = mine && holders[last[tid]] == (int)(SMALL_ROWS - tid);
    if (tid < a.seqs) {
        from[tid] = row.full + mine;
        need = row.held - from[tid]; /* a page in part is one of them */
    }
    uint32_t wanted, spare, count = 0;
    /* pages, a word of 32 a thread */
    if (tid < words) {
        uint32_t bits = 0;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            const uint32_t k = (i + tid) % 32, id = tid * 32 + k; /* 32 banks a step */
            bits |= id < a.pages && holders[id] == 0 ? 1u << k : 0;
        }
        bits &= ~in_part[tid];
        free_words[tid] = bits;
        count = (uint32_t)__popc(bits);
    }
    const uint32_t before = block_scan<SMALL_WAVES>(need, lds, wanted), below = block_scan<SMALL_WAVES>(count, lds, spare);
    if (tid < a.seqs) rank[tid] = before;
    if (tid < words) word_rank[tid] = below;
    __syncthreads();
    if (mine) {
        holders[last[tid]] = 1;
        a.table_out[(size_t)tid * a.table_stride + row.full] = last[tid];
    }
    if (tid < a.seqs) {
        a.held_out[tid] = (int)row.held;
        if (!(last[tid] >= 0 && !mine && before < spare)) { /* else with the page below */
            a.copies[3 * tid] = a.copies[3 * tid + 1] = -1;
            a.copies[3 * tid + 2] = 0;
        }
    }
    if (tid == 0) {
        *a.free_out = (int)(spare - wanted);
        if (wanted > spare) *a.flag = 1;
    }
    /* number k of the wanted pages: the last row that begins at k or before, the last word */
    auto last_of = [](const uint32_t *x, uint32_t n, uint32_t k) {
        uint32_t at = 0;
        for (uint32_t step = n > 1 ? 1u << (31 - __builtin_clz(n - 1)) : 0; step; step /= 2)
            if (at + step < n && x[at + step] <= k) at += step;
        return at;
    };
    for (uint32_t k = tid; k < wanted; k += SMALL_WG) {
        const uint32_t d = last_of(rank, a.seqs, k), x = from[d] + k - rank[d];
        int id = -1;
        if (k < spare) {
            const uint32_t w = last_of(word_rank, words, k);
            uint32_t bits = free_words[w];
            for (uint32_t i = word_rank[w]; i < k; ++i) bits &= bits - 1;
            id = (int)(w * 32) + __ffs(bits) - 1;
            holders[id] = 1;
            if (x == full[d] && last[d] >= 0) {
                a.copies[3 * d] = last[d];
                a.copies[3 * d + 1] = id;
                a.copies[3 * d + 2] = a.keep[d] & ((1 << a.shift) - 1);
            }
        }
        a.table_out[(size_t)d * a.table_stride + x] = id;
    }
    __syncthreads();
    for (uint32_t i = tid; i < a.pages; i += SMALL_WG) a.refs_out[i] = holders[i];
}

/* The workspace: per page what its holders change by; as bits, which pages new rows take in part and which are free; the
 * free ones counted by chunks; per new row the page that it takes in part (-1: none), its first entry that needs a page and
 * how many do. */
struct ForkSpace {
    int *change;
    uint32_t *part, *bits, *chunk, *need, *from;
    int32_t *last;
};
inline uint32_t chunks_of(uint32_t pages) { return (pages + PG_CHUNK - 1) / PG_CHUNK; }
inline ForkSpace fork_space(void *ws, uint32_t pages, uint32_t rows) {
    const size_t chunks = chunks_of(pages), words = chunks * (PG_CHUNK / 32);
    ForkSpace s;
    s.change = (int *)ws;
    s.part = (uint32_t *)(s.change + chunks * PG_CHUNK);
    s.bits = s.part + words;
    s.chunk = s.bits + words;
    s.need = s.chunk + chunks;
    s.from = s.need + rows;
    s.last = (int32_t *)(s.from + rows);
    return s;
}

/* change and part, which follow it. */
__global__ __launch_bounds__(PG_WG) void k_fork_clear(uint4 *p, uint32_t n) {
    const uint32_t i = blockIdx.x * PG_WG + threadIdx.x;
    if (i < n) p[i] = uint4{0, 0, 0, 0};
}

/* The row scans of this kernel and the next two grow with the rows' square: 1000 rows of 8 pages 21 us, 4000 48, 16000 295, 65535
 * 3.7 ms.
 *
 * A workgroup per old row: its first new row (the first one that names it as its parent) takes its holders over, so that only
 * entries behind that one's are given up: a change costs an atomic across the XCDs' L2s, of 256 rows of 2000 pages 29 us when
 * each entry was counted out and in. Then a workgroup per new row: those that are not the first add themselves. */
__global__ __launch_bounds__(PG_WG) void k_fork_count(ForkArgs a, ForkSpace w) {
    __shared__ uint32_t lds[PG_WG / 64], least;
    const uint32_t tid = threadIdx.x;
    const bool old = blockIdx.x < a.old_seqs;
    const uint32_t d = blockIdx.x - a.old_seqs;
    NewRow r = {};
    if (!old) r = new_row(a, d, tid == 0);
    const int s = old ? (int)blockIdx.x : r.parent;
    if (tid == 0) least = a.seqs;
    __syncthreads();
    uint32_t first = a.seqs;
    for (uint32_t i = tid; i < (old ? a.seqs : d); i += PG_WG)
        if (a.parent[i] == s) {
            first = i;
            break;
        }
    if (first < a.seqs) atomicMin(&least, first);
    __syncthreads();
    first = least;
    const int32_t *row = a.table + (size_t)max(s, 0) * a.table_stride;
    if (old) {
        const uint32_t n = old_held(a, (uint32_t)s, tid == 0), kept = first < a.seqs ? new_row(a, first, false).full : 0;
        for (uint32_t x = tid; x < n; x += PG_WG) {
            const uint32_t id = (uint32_t)row[x];
            if (id >= a.pages || a.refs[id] < 1) *a.flag = 1;
            else if (x >= kept) atomicSub(&w.change[id], 1);
        }
        return;
    }
    if (first < a.seqs) /* a lower row has the same parent */
        for (uint32_t x = tid; x < r.full; x += PG_WG) {
            const uint32_t id = (uint32_t)row[x];
            if (id < a.pages && a.refs[id] >= 1) atomicAdd(&w.change[id], 1);
        }
    if (tid == 0) {
        const uint32_t id = r.part ? (uint32_t)row[r.full] : a.pages;
        if (id < a.pages) atomicOr(&w.part[id / 32], 1u << (id % 32));
        w.last[d] = id < a.pages ? (int)id : -1;
    }
}

/* Holders of a page beside the rows that take it in part. */
__device__ __forceinline__ int holders_of(const ForkArgs &a, const ForkSpace &w, uint32_t id, bool flag) {
    const int refs = a.refs[id], n = refs + w.change[id];
    if (flag && (n < 0 || refs < 0)) *a.flag = 1;
    return max(n, 0);
}

/* Chunks of pages: their holders but for fresh ones, and the free ones. Then a workgroup per new row: whether it keeps the page
 * that it takes in part, and the pages that it needs. */
__global__ __launch_bounds__(PG_WG) void k_fork_rows(ForkArgs a, ForkSpace w, uint32_t chunks) {
    __shared__ uint32_t lds[PG_WG / 64];
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < chunks) {
        uint32_t free = 0;
#pragma unroll
        for (uint32_t k = 0; k < PG_CHUNK / PG_WG; ++k) {
            const uint32_t id = blockIdx.x * PG_CHUNK + k * PG_WG + tid;
            bool none = false;
            if (id < a.pages) {
                const int n = holders_of(a, w, id, true);
                const bool kept = n == 0 && (w.part[id / 32] >> (id % 32) & 1);
                none = n == 0 && !kept;
                a.refs_out[id] = n + kept;
            }
            const uint64_t those = __ballot(none);
            if (tid % 64 < 2) w.bits[id / 64 * 2 + tid % 64] = (uint32_t)(those >> (32 * (tid % 64)));
            free += none;
        }
        free = block_sum<PG_WG / 64>(free, lds);
        if (tid == 0) w.chunk[blockIdx.x] = free;
        return;
    }
    const uint32_t d = blockIdx.x - chunks;
    const NewRow r = new_row(a, d, false);
    const int last = w.last[d];
    bool lower = false;
    if (last >= 0)
        for (uint32_t i = tid; i < d; i += PG_WG) lower = lower || w.last[i] == last;
    const uint32_t any = block_sum<PG_WG / 64>((uint32_t)lower, lds);
    if (tid == 0) {
        const bool mine = last >= 0 && !any && holders_of(a, w, (uint32_t)last, false) == 0;
        w.from[d] = r.full + mine;
        w.need[d] = r.held - (r.full + mine); /* a page in part is one of them */
    }
}

/* A workgroup per new row: its entries. Its fresh pages are the free ones of the numbers that the rows before it leave off at:
 * the chunk where they begin, then the words of eight chunks at a time. What the rows need is summed in 64 bits (65535 of 2^20
 * entries); numbers past the free pages are all alike. */
__global__ __launch_bounds__(PG_WG) void k_fork_assign(ForkArgs a, ForkSpace w, uint32_t chunks) {
    __shared__ unsigned long long wide[PG_WG / 64];
    __shared__ uint32_t lds[PG_WG / 64], begin[2];
    const uint32_t tid = threadIdx.x, d = blockIdx.x;
    const bool row_there = d < a.seqs;
    const NewRow r = row_there ? new_row(a, d, false) : NewRow{-1, 0, 0, 0};
    const uint32_t from = row_there ? w.from[d] : 0, need = row_there ? w.need[d] : 0;
    const int last = row_there ? w.last[d] : -1;
    const int32_t *row = a.table + (size_t)max(r.parent, 0) * a.table_stride;
    int32_t *out = a.table_out + (size_t)d * a.table_stride;
    if (row_there) {
#pragma unroll 4
        for (uint32_t x = tid; x < a.table_stride; x += PG_WG) {
            if (x < from) {
                const int id = row[x];
                out[x] = (uint32_t)id < a.pages ? id : -1;
            } else if (x >= from + need) {
                out[x] = -1;
            }
        }
        if (tid == 0) a.held_out[d] = (int)r.held;
    }
    const bool copies = last >= 0 && from == r.full;
    bool copied = false;
    if (need || d == 0) {
        unsigned long long needed = 0; /* by the rows before; row 0: by all */
        uint32_t sum = 0;
        for (uint32_t i = tid; i < (d == 0 ? a.seqs : d); i += PG_WG) needed += w.need[i];
        needed = block_sum<PG_WG / 64>(needed, wide);
        const uint32_t each = (chunks + PG_WG - 1) / PG_WG, c0 = tid * each, c1 = min(c0 + each, chunks);
        for (uint32_t c = c0; c < c1; ++c) sum += w.chunk[c];
        uint32_t spare, at = block_scan<PG_WG / 64>(sum, lds, spare);
        const uint32_t before = d == 0 ? 0 : (uint32_t)min(needed, (unsigned long long)spare);
        if (before >= at && before < at + sum) /* one thread, if any */
            for (uint32_t c = c0; c < c1; at += w.chunk[c++])
                if (before < at + w.chunk[c]) {
                    begin[0] = c;
                    begin[1] = at;
                    break;
                }
        if (d == 0 && tid == 0) {
            *a.free_out = (int)max((long long)spare - (long long)needed, -(1ll << 31));
            if (needed > spare) *a.flag = 1;
        }
        __syncthreads();
        const uint32_t end = min(before + need, spare), words = chunks * (PG_CHUNK / 32);
        copied = copies && before < spare;
        if (before < end) {
            uint32_t number = begin[1], total;
            for (uint32_t w0 = begin[0] * (PG_CHUNK / 32); number < end && w0 < words; w0 += PG_WG, number += total) {
                uint32_t bits = w0 + tid < words ? w.bits[w0 + tid] : 0;
                uint32_t k = number + block_scan<PG_WG / 64>((uint32_t)__popc(bits), lds, total);
                for (; bits && k < end; bits &= bits - 1, ++k) {
                    if (k < before) continue;
                    const int id = (int)((w0 + tid) * 32) + __ffs(bits) - 1;
                    out[from + k - before] = id;
                    a.refs_out[id] = 1;
                    if (k == before && copies) {
                        a.copies[3 * d] = last;
                        a.copies[3 * d + 1] = id;
                        a.copies[3 * d + 2] = (int)r.part;
                    }
                }
            }
        }
        for (uint32_t k = max(before, spare) + tid; k < before + need; k += PG_WG) out[from + k - before] = -1;
    }
    if (row_there && !copied && tid == 0) {
        a.copies[3 * d] = a.copies[3 * d + 1] = -1;
        a.copies[3 * d + 2] = 0;
    }
}

/* ---- copies and moves in every pool --------------------------------------------- */

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
/* i / n of numbers below 2^20 with a quotient below 2^12. */
struct Divide {
    uint32_t n;
    float inv;
    __device__ __forceinline__ Divide(uint32_t n_) : n(n_), inv(1.0f / (float)n_) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t i, uint32_t &rest) const {
        uint32_t q = (uint32_t)((float)i * inv);
        int r = (int)i - (int)(q * n);
        if (r < 0) { /* the estimate is off by one at most */
            --q;
            r += (int)n;
        } else if (r >= (int)n) {
            ++q;
            r -= (int)n;
        }
        rest = (uint32_t)r;
        return q;
    }
};

/* A workgroup per row of `copies`, pool, KV head and kind (keys, values). Keys are one run of bytes; of a value dim's row the
 * first positions, 16 bytes at a time and a shorter end. Scales go with their codes. CP_BATCH pieces a thread are requested
 * before the first is written. Bound by three trips to memory where pages are few (four beams of 24 Q8 layers 4.8 us), by bytes
 * else: 20 pages of 128 in 12 f16 layers of 2 KV heads of 128, 24 MB read and written, 6.9 us, 3.5 TB/s (4 bytes a piece, keys
 * and values in one workgroup: 42). */
constexpr uint32_t CP_BATCH = 4;
template <typename T, typename At>
__device__ __forceinline__ void copy_pieces(uint32_t n, const void *from, void *to, At at) {
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += CP_BATCH * PG_WG) {
        T x[CP_BATCH];
#pragma unroll
        for (uint32_t u = 0; u < CP_BATCH; ++u)
            if (i0 + u * PG_WG < n) x[u] = *(const T *)((const char *)from + at(i0 + u * PG_WG));
#pragma unroll
        for (uint32_t u = 0; u < CP_BATCH; ++u)
            if (i0 + u * PG_WG < n) *(T *)((char *)to + at(i0 + u * PG_WG)) = x[u];
    }
}
/* Of each of `rows` rows, `stride` bytes apart, the first `bytes`, which are whole elements of `unit` bytes. */
__device__ __forceinline__ void copy_rows(const void *from, void *to, uint32_t rows, uint32_t stride, uint32_t bytes, uint32_t unit) {
    const uint32_t whole = bytes / 16, rest = bytes % 16;
    if (whole) {
        const Divide by(whole);
        copy_pieces<u4>(rows * whole, from, to, [&](uint32_t i) {
            uint32_t x;
            const uint32_t r = by(i, x);
            return (size_t)r * stride + 16 * x;
        });
    }
    if (rest) {
        const uint32_t n = rest / unit;
        const Divide by(n);
        auto at = [&](uint32_t i) {
            uint32_t x;
            const uint32_t r = by(i, x);
            return (size_t)r * stride + 16 * whole + x * unit;
        };
        if (unit == 4) copy_pieces<uint32_t>(rows * n, from, to, at);
        else if (unit == 2) copy_pieces<uint16_t>(rows * n, from, to, at);
        else copy_pieces<uint8_t>(rows * n, from, to, at);
    }
}
__global__ __launch_bounds__(PG_WG) void k_paged_copy(PagedArgs a, Pools pools, const int32_t *copies) {
    const uint32_t kind = blockIdx.x & 1, y = blockIdx.x >> 1, h = y % a.kv_heads, l = y / a.kv_heads % pools.n;
    const int32_t *c = copies + 3 * (size_t)(y / a.kv_heads / pools.n);
    const int from = c[0], to = c[1], n = c[2];
    if (n == 0) return;
    if ((uint32_t)from >= a.pages || (uint32_t)to >= a.pages || n < 0 || n > 1 << a.shift) {
        *a.flag = 1;
        return;
    }
    const uint32_t EB = 4 >> a.type;
    const Pool &p = pools.p[l];
    if (pools.again >> l & 1) return;
    const size_t f = (size_t)from * a.kv_heads + h, t = (size_t)to * a.kv_heads + h;
    char *x = (char *)(kind ? p.values : p.keys), *w = (char *)(kind ? p.vs : p.ks);
    const size_t head = ((size_t)a.head_dim << a.shift) * EB, scales = ((size_t)a.nb << a.shift) * 4;
    if (a.type == 2) copy_rows(w + f * scales, w + t * scales, a.nb, 4u << a.shift, (uint32_t)n * 4, 4);
    if (kind) copy_rows(x + f * head, x + t * head, a.head_dim, EB << a.shift, (uint32_t)n * EB, EB);
    else copy_pieces<u4>((uint32_t)n * a.head_dim * EB / 16, x + f * head, x + t * head, [](uint32_t i) { return (size_t)i * 16; });
}

/* A workgroup per sequence, pool and KV head: 16 of the path's tokens at a time into registers, then to their places. The places of one round lie before the next rounds' tokens, since the path ascends. A thread has one token: of its
 * key every 16th piece of 16 bytes, of its value every 16th dim (lanes next to each other have the path's tokens of one dim,
 * which lie in the same lines of memory).
 *
 * Bound by four trips to memory (batch, path, page ids, tokens): 8 paths in 24 Q8 layers 5.2 us; then by the lines that hold a
 * value dim's tokens, 64 bytes for two each way: 64 paths of up to 12 of 60 drafts, four f16 layers of 8 KV heads of 128, 12 us
 * (through LDS, a workgroup's tokens one pass after another: 15; keys and values in workgroups of their own: 19). */
constexpr uint32_t CM_TOKENS = 16;
template <uint32_t EB>
struct Element;
template <>
struct Element<4> {
    typedef uint32_t T;
};
template <>
struct Element<2> {
    typedef uint16_t T;
};
template <>
struct Element<1> {
    typedef uint8_t T;
};
/* n pieces of `step` bytes, N at most, of a token: requested, then written. */
template <typename T, uint32_t N>
struct Piece {
    T x[N];
    __device__ __forceinline__ void load(const char *from, uint32_t n, uint32_t step) {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            if (j < n) x[j] = *(const T *)(from + j * step);
    }
    __device__ __forceinline__ void store(char *to, uint32_t n, uint32_t step) const {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            if (j < n) *(T *)(to + j * step) = x[j];
    }
};
/* A token's move: its page and slot before and after. in: it does move. */
struct Move {
    bool in;
    int fp, tp;
    uint32_t fs, ts;
};
__device__ __forceinline__ Move move_of(const PagedArgs &a, uint32_t s, const Seq &sq, int x, uint32_t k, bool there) {
    const int f = sq.first + x, t = sq.first + (int)k;
    const uint32_t P = 1u << a.shift;
    Move m = {false, -1, -1, (uint32_t)f & (P - 1), (uint32_t)t & (P - 1)};
    if (!there || f == t) return m;
    if (f < 0 || t < 0 || (uint32_t)f >= a.limit) {
        *a.flag = 1;
        return m;
    }
    m.fp = page_of(a, s, (uint32_t)f);
    m.tp = page_of(a, s, (uint32_t)t);
    m.in = m.fp >= 0 && m.tp >= 0;
    return m;
}
template <uint32_t EB>
__global__ __launch_bounds__(PG_WG) void k_paged_compact(PagedArgs a, Pools pools, const int32_t *accepted, uint32_t stride,
                                                         const int32_t *count, int32_t *length_out) {
    typedef typename Element<EB>::T T;
    const uint32_t tid = threadIdx.x, h = blockIdx.x % a.kv_heads, y = blockIdx.x / a.kv_heads, s = y / pools.n;
    const Pool &p = pools.p[y % pools.n];
    const uint32_t kt = tid / 16, kx = tid % 16, vt = tid % 16, vx = tid / 16; /* token and part, of keys and of values */
    const int32_t *path = accepted + (size_t)s * stride;
    /* of the first round, requested with the count */
    const int entry = tid < stride ? path[tid] : 0, m = count[s];
    int k_at = kt < stride ? path[kt] : 0, v_at = vt < stride ? path[vt] : 0;
    Seq sq;
    const bool ok = sequence(a, s, sq);
    bool good = ok && m >= 0 && m <= sq.n && (uint32_t)m <= stride, moved = false;
    if (good)
        for (uint32_t k = tid; k < (uint32_t)m; k += PG_WG) {
            const int at = k == tid ? entry : path[k];
            if (at < 0 || at >= sq.n || (k && at <= path[k - 1])) good = false;
            moved = moved || at != (int)k;
        }
    good = __syncthreads_and(good);
    if (tid == 0 && !good) *a.flag = 1;
    if (length_out && y % pools.n == 0 && h == 0 && tid == 0) length_out[s] = good ? sq.first + m : a.length[s];
    if (!good || !__syncthreads_or(moved) || (pools.again >> y % pools.n & 1)) return;
    const uint32_t hd = a.head_dim, shift = a.shift, nb = a.nb, pieces = hd * EB / 16;
    const uint32_t kn = pieces > kx ? (pieces - kx + 15) / 16 : 0, vn = hd / 16, vstep = 16 * EB << shift;
    for (uint32_t k0 = 0; k0 < (uint32_t)m; k0 += CM_TOKENS) {
        if (k0) {
            k_at = k0 + kt < (uint32_t)m ? path[k0 + kt] : 0;
            v_at = k0 + vt < (uint32_t)m ? path[k0 + vt] : 0;
        }
        const Move km = move_of(a, s, sq, k_at, k0 + kt, k0 + kt < (uint32_t)m), vm = move_of(a, s, sq, v_at, k0 + vt, k0 + vt < (uint32_t)m);
        auto head = [&](int page) { return (size_t)page * a.kv_heads + h; };
        auto key = [&](int page, uint32_t slot) { return (char *)p.keys + ((head(page) << shift) + slot) * hd * EB + 16 * kx; };
        auto value = [&](int page, uint32_t slot) { return (char *)p.values + (((head(page) * hd + vx) << shift) + slot) * EB; };
        auto scale = [&](float *w, int page, uint32_t slot) { return w + ((head(page) * nb + vx) << shift) + slot; };
        Piece<u4, 4> kp;
        Piece<T, 16> vp;
        float ks = 0.0f, vs = 0.0f;
        if (km.in) kp.load(key(km.fp, km.fs), kn, 256);
        if (vm.in) {
            vp.load(value(vm.fp, vm.fs), vn, vstep);
            if (EB == 1 && vx < nb) {
                ks = *scale(p.ks, vm.fp, vm.fs);
                vs = *scale(p.vs, vm.fp, vm.fs);
            }
        }
        __syncthreads(); /* what is read here may be another's place */
        if (km.in) kp.store(key(km.tp, km.ts), kn, 256);
        if (vm.in) {
            vp.store(value(vm.tp, vm.ts), vn, vstep);
            if (EB == 1 && vx < nb) {
                *scale(p.ks, vm.tp, vm.ts) = ks;
                *scale(p.vs, vm.tp, vm.ts) = vs;
            }
        }
    }
}

}  // namespace

size_t fork_workspace(uint32_t pages, uint32_t rows) {
    const ForkSpace s = fork_space(nullptr, pages, rows);
    return (size_t)((char *)(s.last + rows) - (char *)nullptr);
}

hipError_t launch_fork(const ForkArgs &a, void *ws, hipStream_t s) {
    const uint64_t rows = max(a.old_seqs, a.seqs);
    if (a.pages <= SMALL_PAGES && rows <= SMALL_ROWS && rows * a.table_stride <= SMALL_ENTRIES) {
        hipLaunchKernelGGL(k_fork_small, dim3(1), dim3(SMALL_WG), 0, s, a);
        return hipGetLastError();
    }
    const ForkSpace w = fork_space(ws, a.pages, a.seqs);
    const uint32_t chunks = chunks_of(a.pages), clear = chunks * (PG_CHUNK / 4 + PG_CHUNK / 128);
    hipLaunchKernelGGL(k_fork_clear, dim3((clear + PG_WG - 1) / PG_WG), dim3(PG_WG), 0, s, (uint4 *)ws, clear);
    if (a.old_seqs + a.seqs)
        hipLaunchKernelGGL(k_fork_count, dim3(a.old_seqs + a.seqs), dim3(PG_WG), 0, s, a, w);
    hipLaunchKernelGGL(k_fork_rows, dim3(chunks + a.seqs), dim3(PG_WG), 0, s, a, w, chunks);
    hipLaunchKernelGGL(k_fork_assign, dim3(a.seqs ? a.seqs : 1), dim3(PG_WG), 0, s, a, w, chunks);
    return hipGetLastError();
}

/* As many pools a launch as its arguments hold and its grid's threads allow. */
uint32_t pools_at_once(const PagedArgs &a, uint32_t rows) {
    const uint64_t most = (1u << 22) / ((uint64_t)rows * a.kv_heads);
    return most < POOLS_AT_ONCE ? (most ? (uint32_t)most : 1) : POOLS_AT_ONCE;
}
template <typename F>
hipError_t each_pools(const PagedArgs &a, const Pool *pools, uint32_t n, uint32_t rows, F launch) {
    const uint32_t step = pools_at_once(a, rows);
    for (uint32_t i = 0; i < n; i += step) {
        Pools p;
        p.n = n - i < step ? n - i : step;
        p.again = 0;
        for (uint32_t k = 0; k < p.n; ++k) {
            p.p[k] = pools[i + k];
            p.again |= (uint64_t)!pools[i + k].keys << k;
        }
        launch(p, i == 0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_paged_copy(const PagedArgs &a, const Pool *pools, uint32_t n, const int32_t *copies, uint32_t rows,
                             hipStream_t s) {
    return each_pools(a, pools, n, rows, [&](const Pools &p, bool) {
        hipLaunchKernelGGL(k_paged_copy, dim3(2 * rows * p.n * a.kv_heads), dim3(PG_WG), 0, s, a, p, copies);
    });
}

hipError_t launch_paged_compact(const PagedArgs &a, const Pool *pools, uint32_t n, const int32_t *accepted, uint32_t stride,
                                const int32_t *count, int32_t *length_out, hipStream_t s) {
    return each_pools(a, pools, n, a.seqs, [&](const Pools &p, bool first) {
        const dim3 grid(a.seqs * p.n * a.kv_heads);
        int32_t *const tells = first ? length_out : nullptr;
        if (a.type == 0) hipLaunchKernelGGL((k_paged_compact<4>), grid, dim3(PG_WG), 0, s, a, p, accepted, stride, count, tells);
        else if (a.type == 1) hipLaunchKernelGGL((k_paged_compact<2>), grid, dim3(PG_WG), 0, s, a, p, accepted, stride, count, tells);
        else hipLaunchKernelGGL((k_paged_compact<1>), grid, dim3(PG_WG), 0, s, a, p, accepted, stride, count, tells);
    });
}

}  // namespace smq
