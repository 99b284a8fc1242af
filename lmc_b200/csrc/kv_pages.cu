// kv_pages.cu - page bookkeeping of a paged KV cache on the device
// (lmc_kv_pages_fork, _reserve, _compact).
//
// The table and the counts are small (four bytes a page and entry), so the
// plans run in one CTA (reserve, compact) or in column stripes (fork) and are
// bound by latency; what costs bandwidth is copying pages, 2 x page_bytes x
// pools for each, done by one kernel for all pools of a call from the list of
// page pairs that the plan left in the workspace.
#include <algorithm>

#include "lmc_common.cuh"
#include "lmc_internal.h"

namespace {

__device__ int g_kv_pages_err;  // an index outside its range was met (lmc_device_status)

constexpr int PLAN_THREADS = 1024;
constexpr int COPY_VECS = 1024;  // 16-byte words that a CTA copies at a time, four loads a thread in flight
constexpr int MAX_POOLS = 256;  // pool addresses passed in one launch (2 KiB of parameters)

// Workspace: [0] pages to copy, then from WS_LIST on pairs (source, destination),
// then arrays of the plan.
constexpr int WS_LIST = 16;

struct Pools {
    uint4 *p[MAX_POOLS];
};

// Exclusive prefix sum of v over the CTA's 1024 threads; *total gets the sum.
// `part` holds 33 ints.
__device__ __forceinline__ int block_scan(int v, int *part, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // part's last use
    if (lane == 31) part[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int p = part[lane], s = p;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        part[lane] = s - p;
        if (lane == 31) part[32] = s;
    }
    __syncthreads();
    *total = part[32];
    return part[warp] + x - v;
}

// The pages of a plan are gone through in chunks of 1024 M: warp w has the 32 M
// from p0 + 32 M w on, 32 for each bit mask, so a chunk costs one round of
// loads and one prefix sum.  M = 16 for large pools (64 of 65536 pages reserved
// with the last 200 free: 23 us, a compaction of them 28, against 55 and 83
// with M = 1), M = 1 up to 4096 pages, where fewer warps would have all the
// work (1000 pages: 13 against 15 us).
constexpr int SMALL_POOL = 4096, MAX_PAGES = 1 << 30;

// This warp's pages of the chunk at p0 whose count passes `test`, as masks.
template <int M, class T> __device__ __forceinline__ void chunk_masks(const int *refs, int p0, int n_pages, unsigned (&mask)[M], T test) {
    const int p = p0 + (threadIdx.x >> 5) * (32 * M) + (threadIdx.x & 31);
    int r[M];
#pragma unroll
    for (int u = 0; u < M; u++) r[u] = p + 32 * u < n_pages ? refs[p + 32 * u] : 0;
#pragma unroll
    for (int u = 0; u < M; u++) mask[u] = __ballot_sync(0xffffffffu, p + 32 * u < n_pages && test(p + 32 * u, r[u]));
}
template <int M> __device__ __forceinline__ int count_masks(const unsigned (&mask)[M]) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < M; u++) n += __popc(mask[u]);
    return n;
}
// Calls use(i, page) for the masks' pages in order, the chunk's first being number i0; returns how many.
template <int M, class F> __device__ __forceinline__ int number_pages(const unsigned (&mask)[M], int p0, int i0, int *part, F use) {
    const int lane = threadIdx.x & 31;
    int total, i = block_scan(lane == 0 ? count_masks(mask) : 0, part, &total);
    i = i0 + __shfl_sync(0xffffffffu, i, 0);
#pragma unroll
    for (int u = 0; u < M; u++) {
        if (mask[u] >> lane & 1) use(i + __popc(mask[u] & ((1u << lane) - 1)), p0 + (int)(threadIdx.x >> 5) * (32 * M) + 32 * u + lane);
        i += __popc(mask[u]);
    }
    return total;
}

// Column stripe of the table: every row's entries of 2^cs columns are read
// before any is written, so parents may be any mapping.  What a call changes
// in the counts of row r's old entries is the same in every column: one more
// for each other row that copies r, one less when r itself is replaced; so one
// atomic addition per entry of a row where that is not 0 (and none per copy;
// 256 rows of 2048 entries 24 -> 7.5 us).  5 rows of 128: 3.0 us, latency.
__global__ void __launch_bounds__(256) k_pages_fork(int *pages, int n_seqs, int max_pages, int *refs, int n_pages,
                                                    const int *parent, int cs) {
    extern __shared__ int tile[];  // [n_seqs][2^cs], then parent[n_seqs], change[n_seqs]
    int *const par = tile + ((size_t)n_seqs << cs), *const change = par + n_seqs;
    pdl_wait();
    pdl_launch_dependents();
    const int c0 = blockIdx.x << cs, nc = min(1 << cs, max_pages - c0), mask = (1 << cs) - 1;
    const int p0 = threadIdx.x < n_seqs ? parent[threadIdx.x] : 0;  // (on its way beside the table)
#pragma unroll 8
    for (int i = threadIdx.x; i < n_seqs << cs; i += 256)
        if ((i & mask) < nc) tile[i] = pages[(size_t)(i >> cs) * max_pages + c0 + (i & mask)];
    for (int b = threadIdx.x; b < n_seqs; b += 256) {
        int p = b < 256 ? p0 : parent[b];
        if (p >= n_seqs || p < -1) {
            atomicExch(&g_kv_pages_err, 1);
            p = b;
        }
        par[b] = p;
        change[b] = p == b ? 0 : -1;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < n_seqs; b += 256)
        if (par[b] >= 0 && par[b] != b) atomicAdd(change + par[b], 1);
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < n_seqs << cs; i += 256) {
        const int b = i >> cs, j = i & mask, p = par[b], was = tile[i], d = change[b];
        if (j >= nc) continue;
        if (was >= n_pages) atomicExch(&g_kv_pages_err, 1);
        if (d != 0 && was >= 0 && was < n_pages) atomicAdd(refs + was, d);
        if (p != b) {
            const int now = p < 0 ? -1 : tile[(p << cs) + j];
            if (now != was) pages[(size_t)b * max_pages + c0 + j] = now;
        }
    }
}

// Reserve, the plan.  Workspace after the list: entry[n_seqs] (the page that
// sequence b writes, -1 none, -2 nothing to do), rank[n_seqs] (its number
// among those that need a page, or -1).
template <int M> __global__ void __launch_bounds__(PLAN_THREADS) k_reserve_plan(int *pages, int n_seqs, int max_pages, int page_shift,
                                                               int *refs, int n_pages, const int *pos, int *d_short,
                                                               int *ws) {
    __shared__ int part[33], n_copy;
    pdl_wait();
    pdl_launch_dependents();
    int *const list = ws + WS_LIST, *const entry = list + 2 * n_seqs, *const rank = entry + n_seqs;
    const int tid = threadIdx.x;
    if (tid == 0) n_copy = 0;
    for (int b = tid; b < n_seqs; b += PLAN_THREADS) {
        const int p = pos[b];
        int e = -2;
        if (p >= 0) {
            const int j = p >> page_shift;
            if (j < max_pages) e = pages[(size_t)b * max_pages + j];
            if (j >= max_pages || e >= n_pages) {
                atomicExch(&g_kv_pages_err, 1);
                e = -2;
            } else if (e < 0) {
                e = -1;
            }
        }
        entry[b] = e;
    }
    __syncthreads();
    int need_total = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        bool need = false;
        if (b < n_seqs) {
            const int e = entry[b];
            need = e == -1;
            if (e >= 0) {  // the i-th writer of a page copies it while more than i + 1 entries name it
                const int r = refs[e];
                if (r > 1) {
                    int before = 0;
                    for (int i = 0; i < b; i++) before += entry[i] == e;
                    need = before < r - 1;
                }
            }
        }
        int total;
        const int k = block_scan(need ? 1 : 0, part, &total);
        if (b < n_seqs) rank[b] = need ? need_total + k : -1;
        need_total += total;
    }
    // the lowest free ids, into the destinations of the list
    int found = 0;
    for (int p0 = 0; p0 < n_pages && found < need_total; p0 += PLAN_THREADS * M) {
        unsigned mask[M];
        chunk_masks(refs, p0, n_pages, mask, [](int, int r) { return r == 0; });
        found += number_pages(mask, p0, found, part, [&](int i, int p) {
            if (i < need_total) list[2 * i + 1] = p;
        });
    }
    const int missing = max(need_total - found, 0);
    __syncthreads();
    if (missing == 0) {
        // the destinations move into rank first: the list is rewritten as pairs to copy
        for (int b = tid; b < n_seqs; b += PLAN_THREADS)
            if (rank[b] >= 0) rank[b] = list[2 * rank[b] + 1];
        __syncthreads();
        for (int b = tid; b < n_seqs; b += PLAN_THREADS) {
            const int p = rank[b], e = entry[b];
            if (p < 0) continue;
            pages[(size_t)b * max_pages + (pos[b] >> page_shift)] = p;
            refs[p] = 1;
            if (e >= 0) {
                atomicSub(refs + e, 1);
                const int k = atomicAdd(&n_copy, 1);
                list[2 * k] = e;
                list[2 * k + 1] = p;
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        *d_short = missing;
        ws[0] = n_copy;
    }
}

// Compact, the plan.  Workspace: the list, then map[n_pages] (new id of a
// page at or above n_live, -1 for a free one).
template <int M> __global__ void __launch_bounds__(PLAN_THREADS) k_compact_plan(int *refs, int n_pages, int *d_n_live, int *ws) {
    __shared__ int part[33];
    pdl_wait();
    pdl_launch_dependents();
    int *const list = ws + WS_LIST, *const map = list + n_pages + 2;
    const int tid = threadIdx.x;
    int n_live = 0;
    for (int p0 = 0; p0 < n_pages; p0 += PLAN_THREADS * M) {
        unsigned live[M];
        chunk_masks(refs, p0, n_pages, live, [](int, int r) { return r > 0; });
        int total;
        block_scan((tid & 31) == 0 ? count_masks(live) : 0, part, &total);
        n_live += total;
    }
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < n_pages; p0 += PLAN_THREADS * M) {
        unsigned mask[M];
        if (p0 < n_live) {
            chunk_masks(refs, p0, n_live, mask, [](int, int r) { return r <= 0; });
            holes += number_pages(mask, p0, holes, part, [&](int i, int p) { list[2 * i + 1] = p; });
        }
        if (p0 + PLAN_THREADS * M > n_live) {
            chunk_masks(refs, p0, n_pages, mask, [&](int p, int r) {
                if (p >= n_live) map[p] = -1;
                return p >= n_live && r > 0;
            });
            movers += number_pages(mask, p0, movers, part, [&](int i, int p) { list[2 * i] = p; });
        }
    }
    __syncthreads();
    for (int k = tid; k < movers; k += PLAN_THREADS) {
        const int src = list[2 * k], dst = list[2 * k + 1];
        map[src] = dst;
        refs[dst] = refs[src];
        refs[src] = 0;
    }
    if (tid == 0) {
        *d_n_live = n_live;
        ws[0] = movers;
    }
}

// Renames the table's entries by the plan's map.
__device__ __forceinline__ void rename_entry(int *entry, int n_live, int n_pages, const int *map) {
    const int e = *entry;
    if (e < n_live) return;
    const int to = e < n_pages ? map[e] : -1;
    if (to < 0) atomicExch(&g_kv_pages_err, 1);  // no such page, or its count says it is free
    else *entry = to;
}

// Copies the listed pages in every pool; pages != NULL: renames the table too.
// HBM bounds it: 1024 pages of 32 KiB in 64 pools, 600 in use, are compacted in
// 183 us, the plan's 7 included, 87% of a plain copy's rate.  Copies on write of
// pages that eight sequences share read them from L2: 128 sequences, 42 us.
__global__ void __launch_bounds__(256) k_pages_copy(Pools pools, int n_pools, int vecs, const int *ws, int *pages,
                                                    long long entries, const int *d_n_live, int n_pages) {
    pdl_wait();
    pdl_launch_dependents();
    const int n = ws[0];
    const long long tid = (long long)blockIdx.x * 256 + threadIdx.x, nthr = (long long)gridDim.x * 256;
    if (pages) {
        const int n_live = *d_n_live;
        for (long long i = tid; i < entries; i += nthr) rename_entry(pages + i, n_live, n_pages, ws + WS_LIST + n_pages + 2);
    }
    // piece = COPY_VECS neighbouring 16-byte words of one page in one pool; pools innermost, so that the
    // CTAs at work spread over the memory
    const int pieces = (vecs + COPY_VECS - 1) / COPY_VECS;
    const long long items = (long long)n * pieces * n_pools;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int pool = (int)(item % n_pools), at = (int)(item / n_pools % pieces) * COPY_VECS, k = (int)(item / n_pools / pieces);
        const uint4 *src = pools.p[pool] + (size_t)ws[WS_LIST + 2 * k] * vecs + at;
        uint4 *dst = pools.p[pool] + (size_t)ws[WS_LIST + 2 * k + 1] * vecs + at;
        const int m = min(COPY_VECS, vecs - at);
        uint4 v[COPY_VECS / 256];
#pragma unroll
        for (int u = 0; u < COPY_VECS / 256; u++)
            if (threadIdx.x + 256 * u < m) v[u] = __ldg(src + threadIdx.x + 256 * u);
#pragma unroll
        for (int u = 0; u < COPY_VECS / 256; u++)
            if (threadIdx.x + 256 * u < m) dst[threadIdx.x + 256 * u] = v[u];
    }
}

int check_pools(const char *name, void *const *h_pools, int n_pools, size_t page_bytes) {
    if (!h_pools || n_pools <= 0 || page_bytes == 0 || page_bytes % 16 || page_bytes / 16 > (1u << 30))
        return lmc_set_error(LMC_ERR_INVALID, "%s: %d pools, pages of %zu bytes (need a multiple of 16)", name, n_pools,
                             page_bytes);
    for (int i = 0; i < n_pools; i++)
        if (!h_pools[i] || ((uintptr_t)h_pools[i] & 15))
            return lmc_set_error(LMC_ERR_INVALID, "%s: pool %d is null or not 16-byte aligned", name, i);
    return LMC_OK;
}

// At most `most` pages are copied and `entries` table entries renamed: no more CTAs than that has work for.
int copy_launch(const char *name, void *const *h_pools, int n_pools, size_t page_bytes, int most, const int *ws, int *pages,
                long long entries, const int *d_n_live, int n_pages, cudaStream_t s) {
    const long long pieces = (long long)(page_bytes / 16 + COPY_VECS - 1) / COPY_VECS * std::min(n_pools, MAX_POOLS) * most;
    const int grid = (int)std::min<long long>(lmc_sm_count() * 8, std::max(pieces, (entries + 255) / 256));
    for (int p0 = 0; p0 < n_pools; p0 += MAX_POOLS) {
        Pools pools;
        const int n = n_pools - p0 < MAX_POOLS ? n_pools - p0 : MAX_POOLS;
        for (int i = 0; i < n; i++) pools.p[i] = (uint4 *)h_pools[p0 + i];
        LMC_LAUNCH(name, k_pages_copy, grid, 256, 0, s, pools, n, (int)(page_bytes / 16), ws, p0 ? nullptr : pages, entries,
                   d_n_live, n_pages);
    }
    return LMC_OK;
}

}  // namespace

extern "C" size_t lmc_kv_pages_workspace_bytes(int n_seqs, int n_pages) {
    if (n_seqs < 0 || n_pages < 0) return 0;
    return sizeof(int) * (64 + 4 * ((size_t)n_seqs + (size_t)n_pages));
}

extern "C" int lmc_kv_pages_fork(int *d_pages, int n_seqs, int max_pages, int *d_refs, int n_pages, const int *d_parent,
                                 void *stream) {
    if (!d_pages || !d_refs || !d_parent) return lmc_set_error(LMC_ERR_INVALID, "kv_pages_fork: null pointer");
    if (n_seqs <= 0 || max_pages <= 0 || n_pages <= 0 || n_seqs > 16384)
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_fork: %d sequences x %d entries, %d pages (at most 16384 "
                             "sequences)", n_seqs, max_pages, n_pages);
    // 32 columns (128 bytes of a row) to a CTA; down to 8 (a 32-byte sector)
    // while that gives fewer than two CTAs an SM, and as few as fit in 128 KiB,
    // with the parents and changes beside them in 200 (16384 sequences: one column, 192 KiB)
    constexpr size_t MOST = 200 * 1024;
    const size_t column = n_seqs * sizeof(int);
    int cs = 5;
    while (cs > 3 && (max_pages >> cs) < 2 * lmc_sm_count()) cs--;
    while (cs > 0 && (column << cs > 128 * 1024 || (column << cs) + 2 * column > MOST)) cs--;
    const size_t smem = (column << cs) + 2 * column;
    if (smem > 48 * 1024) LMC_CUDA_TRY(cudaFuncSetAttribute(k_pages_fork, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST));
    LMC_LAUNCH("kv pages fork", k_pages_fork, lmc_cdiv(max_pages, (size_t)1 << cs), 256, smem, lmc_stream(stream), d_pages,
               n_seqs, max_pages, d_refs, n_pages, d_parent, cs);
    return LMC_OK;
}

extern "C" int lmc_kv_pages_reserve(void *const *h_pools, int n_pools, size_t page_bytes, int *d_pages, int n_seqs,
                                    int max_pages, int page_size, int *d_refs, int n_pages, const int *d_pos,
                                    int *d_short, void *d_ws, size_t ws_bytes, void *stream) {
    const int rc = check_pools("kv_pages_reserve", h_pools, n_pools, page_bytes);
    if (rc != LMC_OK) return rc;
    if (!d_pages || !d_refs || !d_pos || !d_short || !d_ws)
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_reserve: null pointer");
    // (the plan compares each writer of a shared page with those before it)
    if (n_seqs <= 0 || n_seqs > 65536 || max_pages <= 0 || n_pages <= 0 || n_pages > MAX_PAGES || page_size < 16 || (page_size & (page_size - 1)))
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_reserve: %d sequences x %d entries, %d pages of %d positions",
                             n_seqs, max_pages, n_pages, page_size);
    if (ws_bytes < lmc_kv_pages_workspace_bytes(n_seqs, n_pages))
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_reserve: workspace %zu bytes < %zu needed", ws_bytes,
                             lmc_kv_pages_workspace_bytes(n_seqs, n_pages));
    int shift = 0;
    while ((1 << shift) < page_size) shift++;
    cudaStream_t s = lmc_stream(stream);
    LMC_LAUNCH("kv pages reserve", (n_pages <= SMALL_POOL ? k_reserve_plan<1> : k_reserve_plan<16>), 1, PLAN_THREADS, 0, s, d_pages, n_seqs, max_pages, shift, d_refs, n_pages,
               d_pos, d_short, (int *)d_ws);
    return copy_launch("kv pages copy", h_pools, n_pools, page_bytes, n_seqs, (const int *)d_ws, nullptr, 0, nullptr, n_pages, s);
}

extern "C" int lmc_kv_pages_compact(void *const *h_pools, int n_pools, size_t page_bytes, int *d_pages, int n_seqs,
                                    int max_pages, int *d_refs, int n_pages, int *d_n_live, void *d_ws, size_t ws_bytes,
                                    void *stream) {
    const int rc = check_pools("kv_pages_compact", h_pools, n_pools, page_bytes);
    if (rc != LMC_OK) return rc;
    if (!d_pages || !d_refs || !d_n_live || !d_ws)
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_compact: null pointer");
    if (n_seqs <= 0 || max_pages <= 0 || n_pages <= 0 || n_pages > MAX_PAGES)
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_compact: %d sequences x %d entries, %d pages", n_seqs, max_pages,
                             n_pages);
    if (ws_bytes < lmc_kv_pages_workspace_bytes(n_seqs, n_pages))
        return lmc_set_error(LMC_ERR_INVALID, "kv_pages_compact: workspace %zu bytes < %zu needed", ws_bytes,
                             lmc_kv_pages_workspace_bytes(n_seqs, n_pages));
    cudaStream_t s = lmc_stream(stream);
    LMC_LAUNCH("kv pages compact", (n_pages <= SMALL_POOL ? k_compact_plan<1> : k_compact_plan<16>), 1, PLAN_THREADS, 0, s, d_refs, n_pages, d_n_live, (int *)d_ws);
    return copy_launch("kv pages copy", h_pools, n_pools, page_bytes, n_pages / 2, (const int *)d_ws, d_pages,
                       (long long)n_seqs * max_pages, d_n_live, n_pages, s);
}

extern "C" int lmc_kv_pages_status(void) {
    int v = 0;
    LMC_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv_pages_err, sizeof(int)));
    if (!v) return LMC_OK;
    const int zero = 0;
    LMC_CUDA_TRY(cudaMemcpyToSymbol(g_kv_pages_err, &zero, sizeof(int)));
    return lmc_set_error(LMC_ERR_INVALID, "kv pages: a table entry, parent or position outside its range (left as it is)");
}
