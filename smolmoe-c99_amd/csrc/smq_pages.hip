/* Pages of the paged KV cache on gfx950: the next tables of a set of sequences (shared, copied, fresh and freed pages), the
 * copies over all layers, and accepted drafts moved to the front of their sequence's new tokens (include/smq.h). */
#include "smq_paged.h"

namespace smq {
namespace {

constexpr uint32_t PG_WG = 256, PG_CHUNK = 1024; /* pages of a chunk */
constexpr uint32_t PART = 1u << 31;              /* of a page's claims: some new row takes it in part */

/* The workspace: per page the old table's entries and the new one's claims; per chunk its free pages; per new row the page
 * that it takes in part (-1: none), its first entry that needs a page and how many do. */
struct ForkSpace {
    uint32_t *gone, *claims, *chunk, *need;
    int32_t *last;
    uint32_t *from;
};
__host__ __device__ inline ForkSpace fork_space(void *ws, uint32_t pages, uint32_t rows) {
    const uint32_t chunks = (pages + PG_CHUNK - 1) / PG_CHUNK;
    ForkSpace s;
    s.gone = (uint32_t *)ws;
    s.claims = s.gone + pages;
    s.chunk = s.claims + pages;
    s.need = s.chunk + chunks;
    s.last = (int32_t *)(s.need + rows);
    s.from = (uint32_t *)(s.last + rows);
    return s;
}

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
__device__ __forceinline__ uint32_t block_sum(uint32_t x, uint32_t *lds) {
    for (int off = 1; off < 64; off *= 2) x += __shfl_xor(x, off);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    uint32_t t = 0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) t += lds[w];
    return t;
}

__global__ __launch_bounds__(PG_WG) void k_fork_clear(ForkArgs a, ForkSpace w) {
    const uint32_t i = blockIdx.x * PG_WG + threadIdx.x;
    if (i < a.pages) {
        w.gone[i] = 0;
        w.claims[i] = 0;
    }
}

/* A workgroup per old row, then one per new row: how often each page was named, and is. */
__global__ __launch_bounds__(PG_WG) void k_fork_count(ForkArgs a, ForkSpace w) {
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < a.old_seqs) {
        const int held = a.held[blockIdx.x];
        if ((held < 0 || held > (int)a.table_stride) && tid == 0) *a.flag = 1;
        const uint32_t n = (uint32_t)min(max(held, 0), (int)a.table_stride);
        for (uint32_t x = tid; x < n; x += PG_WG) {
            const uint32_t id = (uint32_t)a.table[(size_t)blockIdx.x * a.table_stride + x];
            if (id < a.pages) atomicAdd(&w.gone[id], 1u);
            else *a.flag = 1;
        }
        return;
    }
    const uint32_t d = blockIdx.x - a.old_seqs;
    const NewRow r = new_row(a, d, tid == 0);
    const int32_t *row = a.table + (size_t)max(r.parent, 0) * a.table_stride;
    for (uint32_t x = tid; x < r.full; x += PG_WG) {
        const uint32_t id = (uint32_t)row[x];
        if (id < a.pages) atomicAdd(&w.claims[id], 1u);
    }
    if (tid == 0) {
        const uint32_t id = r.part ? (uint32_t)row[r.full] : a.pages;
        if (id < a.pages) atomicOr(&w.claims[id], PART);
        w.last[d] = id < a.pages ? (int)id : -1;
    }
}

/* What holds page id beside the old table's rows and the rows that take it in part. */
__device__ __forceinline__ uint32_t others(const ForkArgs &a, const ForkSpace &w, uint32_t id, bool flag) {
    const int refs = a.refs[id];
    const uint32_t gone = w.gone[id];
    if (flag && (refs < 0 || (uint32_t)refs < gone)) *a.flag = 1;
    return (refs > 0 && (uint32_t)refs > gone ? (uint32_t)refs - gone : 0) + (w.claims[id] & ~PART);
}

/* Chunks of pages: their holders but for fresh ones, and the free ones counted. Then a workgroup per new row: whether it
 * keeps the page that it takes in part, and the pages it needs. */
__global__ __launch_bounds__(PG_WG) void k_fork_rows(ForkArgs a, ForkSpace w, uint32_t chunks) {
    __shared__ uint32_t lds[PG_WG / 64];
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < chunks) {
        uint32_t free = 0;
        for (uint32_t k = 0; k < PG_CHUNK / PG_WG; ++k) {
            const uint32_t id = blockIdx.x * PG_CHUNK + k * PG_WG + tid;
            if (id >= a.pages) break;
            const uint32_t n = others(a, w, id, true), kept = n == 0 && (w.claims[id] & PART);
            a.refs_out[id] = (int)(n + kept);
            free += n + kept == 0;
        }
        free = block_sum(free, lds);
        if (tid == 0) w.chunk[blockIdx.x] = free;
        return;
    }
    const uint32_t d = blockIdx.x - chunks;
    const NewRow r = new_row(a, d, false);
    const int last = w.last[d];
    bool lower = false;
    if (last >= 0)
        for (uint32_t i = tid; i < d; i += PG_WG) lower = lower || w.last[i] == last;
    const uint32_t any = block_sum(lower, lds);
    if (tid == 0) {
        const bool mine = last >= 0 && !any && others(a, w, (uint32_t)last, false) == 0;
        w.from[d] = r.full + mine;
        w.need[d] = r.held - min(r.held, r.full + mine);
    }
}

/* Chunks of pages: each free one to the row and entry whose number it has. Then a workgroup per new row: the other
 * entries. */
__global__ __launch_bounds__(PG_WG) void k_fork_assign(ForkArgs a, ForkSpace w, uint32_t chunks) {
    __shared__ uint32_t lds[PG_WG / 64], scan[PG_WG];
    const uint32_t tid = threadIdx.x;
    uint32_t need = 0, free = 0, mine = 0;
    const uint32_t d = blockIdx.x - chunks;
    for (uint32_t i = tid; i < a.seqs; i += PG_WG) {
        need += w.need[i];
        if (blockIdx.x >= chunks && i < d) mine += w.need[i];
    }
    for (uint32_t i = tid; i < chunks; i += PG_WG) {
        free += w.chunk[i];
        if (blockIdx.x < chunks && i < blockIdx.x) mine += w.chunk[i];
    }
    need = block_sum(need, lds);
    free = block_sum(free, lds);
    mine = block_sum(mine, lds);
    if (blockIdx.x == 0 && tid == 0) {
        *a.free_out = (int)(free - need);
        if (need > free) *a.flag = 1;
    }
    if (blockIdx.x < chunks) {
        for (uint32_t k = 0; k < PG_CHUNK / PG_WG; ++k) {
            const uint32_t id = blockIdx.x * PG_CHUNK + k * PG_WG + tid;
            const bool ok = id < a.pages && a.refs_out[id] == 0 && w.claims[id] == 0;
            scan[tid] = ok;
            __syncthreads();
            uint32_t at = mine, all = 0;
            for (uint32_t i = 0; i < PG_WG; ++i) {
                at += i < tid ? scan[i] : 0;
                all += scan[i];
            }
            __syncthreads();
            if (ok && at < need) {
                uint32_t row = 0;
                while (at >= w.need[row]) at -= w.need[row++];
                const uint32_t x = w.from[row] + at;
                a.table_out[(size_t)row * a.table_stride + x] = (int)id;
                a.refs_out[id] = 1;
                const NewRow r = new_row(a, row, false);
                if (r.part && w.last[row] >= 0 && x == r.full) {
                    a.copies[3 * row] = w.last[row];
                    a.copies[3 * row + 1] = (int)id;
                    a.copies[3 * row + 2] = (int)r.part;
                }
            }
            mine += all;
        }
        return;
    }
    const NewRow r = new_row(a, d, false);
    const uint32_t from = w.from[d], end = from + w.need[d], have = mine < free ? min(w.need[d], free - mine) : 0;
    const int32_t *row = a.table + (size_t)max(r.parent, 0) * a.table_stride;
    int32_t *out = a.table_out + (size_t)d * a.table_stride;
    for (uint32_t x = tid; x < a.table_stride; x += PG_WG) {
        if (x < from) {
            const int id = row[x];
            out[x] = (uint32_t)id < a.pages ? id : -1;
        } else if (x >= from + have || x >= end) {
            out[x] = -1;
        }
    }
    if (tid == 0) {
        a.held_out[d] = (int)r.held;
        if (!(r.part && w.last[d] >= 0 && from == r.full && have)) {
            a.copies[3 * d] = a.copies[3 * d + 1] = -1;
            a.copies[3 * d + 2] = 0;
        }
    }
}

/* ---- copies and moves in every pool --------------------------------------------- */

template <typename T>
__device__ __forceinline__ void copy_run(T *to, const T *from, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += PG_WG) to[i] = from[i];
}

/* A workgroup per row of `copies`, pool and KV head. */
__global__ __launch_bounds__(PG_WG) void k_paged_copy(PagedArgs a, Pools pools, const int32_t *copies) {
    const uint32_t h = blockIdx.x % a.kv_heads, l = blockIdx.x / a.kv_heads % pools.n;
    const int32_t *c = copies + 3 * (size_t)(blockIdx.x / a.kv_heads / pools.n);
    const int from = c[0], to = c[1], n = c[2];
    if (n == 0) return;
    if ((uint32_t)from >= a.pages || (uint32_t)to >= a.pages || n < 0 || n > 1 << a.shift) {
        *a.flag = 1;
        return;
    }
    const uint32_t EB = 4 >> a.type;
    const Pool &p = pools.p[l];
    const size_t head = (size_t)a.head_dim << a.shift, f = ((size_t)from * a.kv_heads + h) * head * EB,
                 t = ((size_t)to * a.kv_heads + h) * head * EB;
    copy_run((uint32_t *)((char *)p.keys + t), (const uint32_t *)((const char *)p.keys + f), (uint32_t)n * a.head_dim * EB / 4);
    for (uint32_t i = threadIdx.x; i < a.head_dim * (uint32_t)n * EB; i += PG_WG) {
        const uint32_t d = i / (n * EB), x = i % (n * EB);
        ((char *)p.values)[t + ((size_t)d * EB << a.shift) + x] = ((const char *)p.values)[f + ((size_t)d * EB << a.shift) + x];
    }
    if (a.type == 2)
        for (uint32_t i = threadIdx.x; i < a.nb * (uint32_t)n; i += PG_WG) {
            const uint32_t b = i / n, x = i % n;
            const size_t sf = ((((size_t)from * a.kv_heads + h) * a.nb + b) << a.shift) + x,
                         st = ((((size_t)to * a.kv_heads + h) * a.nb + b) << a.shift) + x;
            p.ks[st] = p.ks[sf];
            p.vs[st] = p.vs[sf];
        }
}

/* A workgroup per sequence, pool and KV head: 16 of the path's tokens at a time into LDS, then to their places. The places
 * of one round lie before the next rounds' tokens, since the path ascends. */
constexpr uint32_t CP_AT_ONCE = 16;
__global__ __launch_bounds__(PG_WG) void k_paged_compact(PagedArgs a, Pools pools, const int32_t *accepted, uint32_t stride,
                                                         const int32_t *count, int32_t *length_out) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ int from_page[CP_AT_ONCE], to_page[CP_AT_ONCE];
    __shared__ uint32_t from_slot[CP_AT_ONCE], to_slot[CP_AT_ONCE];
    const uint32_t tid = threadIdx.x, h = blockIdx.x % a.kv_heads, l = blockIdx.x / a.kv_heads % pools.n;
    const uint32_t s = blockIdx.x / a.kv_heads / pools.n;
    const Pool &p = pools.p[l];
    const bool first_one = h == 0 && l == 0 && length_out;
    Seq sq;
    const int m = count[s];
    const int32_t *path = accepted + (size_t)s * stride;
    bool ok = sequence(a, s, sq);
    bool good = ok && m >= 0 && m <= sq.n && (uint32_t)m <= stride;
    if (good)
        for (uint32_t k = tid; k < (uint32_t)m; k += PG_WG)
            if (path[k] < 0 || path[k] >= sq.n || (k && path[k] <= path[k - 1])) good = false;
    good = __syncthreads_and(good);
    if (!good) {
        if (tid == 0) *a.flag = 1;
        if (tid == 0 && first_one) length_out[s] = a.length[s];
        return;
    }
    if (tid == 0 && first_one) length_out[s] = sq.first + m;
    const uint32_t EB = 4 >> a.type, hd = a.head_dim, P = 1u << a.shift, words = hd * EB / 4;
    uint32_t *keys = (uint32_t *)lds;
    unsigned char *values = lds + CP_AT_ONCE * hd * EB;
    float *scales = (float *)(values + CP_AT_ONCE * hd * EB);
    for (uint32_t k0 = 0; k0 < (uint32_t)m; k0 += CP_AT_ONCE) {
        const uint32_t n = min(CP_AT_ONCE, (uint32_t)m - k0);
        __syncthreads();
        if (tid < n) {
            const int f = sq.first + path[k0 + tid], t = sq.first + (int)(k0 + tid);
            from_page[tid] = to_page[tid] = -1;
            if (f != t) {
                if ((uint32_t)f < a.limit && (uint32_t)t < a.limit && f >= 0 && t >= 0) {
                    const int fp = page_of(a, s, (uint32_t)f), tp = page_of(a, s, (uint32_t)t);
                    from_page[tid] = fp;
                    to_page[tid] = fp < 0 ? -1 : tp;
                    from_slot[tid] = (uint32_t)f & (P - 1);
                    to_slot[tid] = (uint32_t)t & (P - 1);
                } else {
                    *a.flag = 1;
                }
            }
        }
        __syncthreads();
        for (int store = 0; store < 2; ++store) {
            auto place = [&](uint32_t k, size_t &page, uint32_t &slot) {
                const int pg = store ? to_page[k] : from_page[k];
                page = (size_t)max(pg, 0) * a.kv_heads + h;
                slot = store ? to_slot[k] : from_slot[k];
                return to_page[k] >= 0;
            };
            size_t page;
            uint32_t slot;
            for (uint32_t i = tid; i < n * words; i += PG_WG) {
                if (!place(i / words, page, slot)) continue;
                uint32_t *x = (uint32_t *)p.keys + ((page << a.shift) + slot) * words + i % words;
                if (store) *x = keys[i];
                else keys[i] = *x;
            }
            for (uint32_t i = tid; i < n * hd; i += PG_WG) {
                if (!place(i / hd, page, slot)) continue;
                const size_t at = ((page * hd + i % hd) << a.shift) + slot;
                unsigned char *x = (unsigned char *)p.values + at * EB, *y = values + (size_t)i * EB;
                unsigned char *to = store ? x : y, *from = store ? y : x;
                if (a.type == 0) *(uint32_t *)to = *(const uint32_t *)from;
                else if (a.type == 1) *(uint16_t *)to = *(const uint16_t *)from;
                else *to = *from;
            }
            if (a.type == 2)
                for (uint32_t i = tid; i < n * a.nb; i += PG_WG) {
                    if (!place(i / a.nb, page, slot)) continue;
                    const size_t at = ((page * a.nb + i % a.nb) << a.shift) + slot;
                    if (store) {
                        p.ks[at] = scales[2 * i];
                        p.vs[at] = scales[2 * i + 1];
                    } else {
                        scales[2 * i] = p.ks[at];
                        scales[2 * i + 1] = p.vs[at];
                    }
                }
            __syncthreads();
        }
    }
}

}  // namespace

size_t fork_workspace(uint32_t pages, uint32_t rows) {
    const ForkSpace s = fork_space(nullptr, pages, rows);
    return (size_t)((char *)(s.from + rows) - (char *)nullptr);
}

hipError_t launch_fork(const ForkArgs &a, void *ws, hipStream_t s) {
    const ForkSpace w = fork_space(ws, a.pages, a.seqs);
    const uint32_t chunks = (a.pages + PG_CHUNK - 1) / PG_CHUNK;
    hipLaunchKernelGGL(k_fork_clear, dim3((a.pages + PG_WG - 1) / PG_WG), dim3(PG_WG), 0, s, a, w);
    hipLaunchKernelGGL(k_fork_count, dim3(a.old_seqs + a.seqs), dim3(PG_WG), 0, s, a, w);
    hipLaunchKernelGGL(k_fork_rows, dim3(chunks + a.seqs), dim3(PG_WG), 0, s, a, w, chunks);
    hipLaunchKernelGGL(k_fork_assign, dim3(chunks + a.seqs), dim3(PG_WG), 0, s, a, w, chunks);
    return hipGetLastError();
}

/* As many pools a launch as its arguments hold and its grid's threads allow. */
uint32_t pools_at_once(const PagedArgs &a, uint32_t rows) {
    const uint64_t most = (1u << 23) / ((uint64_t)rows * a.kv_heads);
    return most < POOLS_AT_ONCE ? (most ? (uint32_t)most : 1) : POOLS_AT_ONCE;
}
template <typename F>
hipError_t each_pools(const PagedArgs &a, const Pool *pools, uint32_t n, uint32_t rows, F launch) {
    const uint32_t step = pools_at_once(a, rows);
    for (uint32_t i = 0; i < n; i += step) {
        Pools p;
        p.n = n - i < step ? n - i : step;
        for (uint32_t k = 0; k < p.n; ++k) p.p[k] = pools[i + k];
        launch(p, i == 0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_paged_copy(const PagedArgs &a, const Pool *pools, uint32_t n, const int32_t *copies, uint32_t rows,
                             hipStream_t s) {
    return each_pools(a, pools, n, rows, [&](const Pools &p, bool) {
        hipLaunchKernelGGL(k_paged_copy, dim3(rows * p.n * a.kv_heads), dim3(PG_WG), 0, s, a, p, copies);
    });
}

hipError_t launch_paged_compact(const PagedArgs &a, const Pool *pools, uint32_t n, const int32_t *accepted, uint32_t stride,
                                const int32_t *count, int32_t *length_out, hipStream_t s) {
    const uint32_t EB = 4 >> a.type, lds = CP_AT_ONCE * (2 * a.head_dim * EB + 8 * a.nb);
    return each_pools(a, pools, n, a.seqs, [&](const Pools &p, bool first) {
        hipLaunchKernelGGL(k_paged_compact, dim3(a.seqs * p.n * a.kv_heads), dim3(PG_WG), lds, s, a, p, accepted, stride, count,
                           first ? length_out : nullptr);
    });
}

}  // namespace smq
