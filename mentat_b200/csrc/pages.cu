// Pages of several sequences at once: batched fork, batched free, and compaction of
// sequences to kept tokens.
//
// The allocator's state after a batch is that of the single calls made one after
// another (kv_cache.cu).  For a fork that needs no order: every child takes its
// parent's table and every page's count rises.  A free does: a page joins the free
// FIFO where its last reference goes, in the order sequence, layer, table entry.
// All releases are subtracted at once; each also raises its block's word of
// `order` to its own index in that order, and the one whose index stands there
// after all of them, over a count of zero, is the release that frees the block.
// Positions in the FIFO are a scan over the rows (sequence, layer) of how many
// blocks each one frees.
//
// Compaction pops its fresh blocks in the same row order (the scan over the rows'
// demands), moves the kept rows there, one CTA per page, and then releases, in place,
// what the sequence held beyond its unchanged pages at the front.
//
// The steps of one call depend on one another across all rows.  Where they are small, one cluster
// of CTAs takes them all, with cluster barriers between them; else each step is a launch.
//
// Forks and frees are bound by latency: chains of dependent loads and barriers.  Fork and free of 64 x 3 children of 130
// to 160 pages in 32 layers: 32 us, against 1 us of bytes; of 6 of 30 pages: 17 us.  A compaction is bound by the
// rows that it moves.

#include <cooperative_groups.h>

#include "rotary.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

namespace mentat {

constexpr int PAGES_MAX_SEQS = 1024;

// workspace: [0] 1 = stop (an error, now or before), [1] fresh blocks of a compaction, [2..3] the FIFO's tail before
// a free, then order, the ids of fresh
// blocks, and per row the pages at the front that stay, the first of its fresh
// blocks, the freed (or, before that, the demanded) count, and its exclusive scan
struct PagesWs {
    int32_t* stop;
    uint32_t* order;
    int32_t* fresh;
    int32_t* lead;
    int32_t* first;
    int32_t* count;
    int32_t* base;
};

static int64_t pages_ws(const mentat_kv_cache* c, int64_t n, void* p, PagesWs* w) {
    const int64_t B = ((int64_t)c->num_blocks + 3) / 4 * 4, R = (n * c->num_layers + 3) / 4 * 4;
    if (w) {
        int32_t *x = reinterpret_cast<int32_t*>(p), *y = x + 4 + 2 * B;
        *w = PagesWs{x, reinterpret_cast<uint32_t*>(x + 4), x + 4 + B, y, y + R, y + 2 * R, y + 3 * R};
    }
    return (4 + 2 * B + 4 * R) * (int64_t)sizeof(int32_t);
}

// Whether the slots are in range and distinct, as a bitmap over max_seqs in shared
// memory (zeroed here); every thread of the CTA gets the answer.
__device__ __forceinline__ bool slots_distinct(const mentat_kv_cache& c, const int32_t* slots, int n, uint32_t* bits,
                                               int* bad) {
    for (int k = threadIdx.x; k < (c.max_seqs + 31) / 32; k += blockDim.x) bits[k] = 0;
    __syncthreads();
    int no = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = slots[i];
        if (s < 0 || s >= c.max_seqs || ((atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1)) {
            no = 1;
            *bad = s;  // any of them
        }
    }
    return !__syncthreads_or(no);
}
// Entries of a table, no more than it has room for: the counters of a KVCacheView are the caller's.
__device__ __forceinline__ int table_len(const mentat_kv_cache& c, int64_t si) { return min(c.nblocks[si], c.max_blocks_per_seq); }
__device__ __forceinline__ bool table_overflows(const mentat_kv_cache& c, int64_t si) {
    const int nb = c.nblocks[si], len = c.ntok[si];
    return nb > c.max_blocks_per_seq || len > (int64_t)c.max_blocks_per_seq * c.block_size;
}
__device__ __forceinline__ bool has_bit(const uint32_t* bits, int s) { return (bits[s >> 5] >> (s & 31)) & 1; }

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
// The batch is checked in a launch before: no CTA of the fork could see whether a child is empty, since another one may
// have filled it.  What is wrong is recorded, and the fork does nothing after an error.  CTA 0 looks at the slots, all of them at
// the counters.
constexpr int PAGES_THREADS = 256, PAGES_WARPS = PAGES_THREADS / 32;
__global__ void __launch_bounds__(PAGES_THREADS) k_fork_check(mentat_kv_cache c, const int32_t* parents,
                                                              const int32_t* children, int n) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
    griddep_launch();
    for (int64_t x = blockIdx.x * (int64_t)PAGES_THREADS + threadIdx.x; x < (int64_t)n * c.num_layers;
         x += (int64_t)gridDim.x * PAGES_THREADS) {
        const int s = children[x % n], p = parents[x % n], l = (int)(x / n);
        const bool child = s >= 0 && s < c.max_seqs, parent = p >= 0 && p < c.max_seqs;
        const int64_t si = seq_index(c, l, child ? s : 0), pi = seq_index(c, l, parent ? p : 0);
        const bool used = (c.nblocks[si] | c.ntok[si]) != 0, over = table_overflows(c, pi);
        if (child && used) set_error(c, MENTAT_DEV_BAD_SLOT, s);
        if (parent && over) set_error(c, MENTAT_DEV_TABLE_OVERFLOW, p);
    }
    if (blockIdx.x) return;
    if (!slots_distinct(c, children, n, bits, &s_bad)) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
        return;
    }
    for (int i = threadIdx.x; i < n; i += PAGES_THREADS) {
        const int p = parents[i];
        if (p < 0 || p >= c.max_seqs || has_bit(bits, p)) set_error(c, MENTAT_DEV_BAD_SLOT, p);
    }
}

// A warp takes one (layer, child) and every gridDim.z-th group of 128 pages.  Of a run of children of one parent that
// follow one another, the first one's warp raises each page's count by the run's length in one atomic.  (One warp for
// a whole run and table: 3 children of 2,048 pages in 32 layers took 43 us, 3 single forks 14.)
__global__ void __launch_bounds__(PAGES_THREADS) k_fork_batched(mentat_kv_cache c, const int32_t* parents,
                                                                const int32_t* children, int n) {
    __shared__ int s_stop;
    griddep_wait();
    griddep_launch();
    if (threadIdx.x == 0) s_stop = has_error(c);
    __syncthreads();
    if (s_stop) return;
    const int lane = threadIdx.x & 31, l = blockIdx.y, i = blockIdx.x * PAGES_WARPS + (threadIdx.x >> 5);
    if (i >= n) return;
    const int parent = parents[i], child = children[i];
    const int64_t ps = seq_index(c, l, parent), cs = seq_index(c, l, child);
    const int nb = c.nblocks[ps], ntok = c.ntok[ps], tail = c.tail[ps];
    int run = 0;  // of the children that this one is the first of
    if (i == 0 || parents[i - 1] != parent) {
        uint32_t same = 0xffffffffu;
        for (run = 1; same == 0xffffffffu; run += same == 0xffffffffu ? 32 : __ffs(~same) - 1)
            same = __ballot_sync(0xffffffffu, i + run + lane < n && parents[i + run + lane] == parent);
    }
    const int32_t* src = table_row(c, l, parent);
    int32_t* dst = table_row(c, l, child);
    for (int j0 = blockIdx.z * 128 + lane; j0 < nb; j0 += gridDim.z * 128) {
        int b[4], old[4];  // four entries of a lane on the way
#pragma unroll
        for (int u = 0; u < 4; ++u) b[u] = j0 + 32 * u < nb ? src[j0 + 32 * u] : -1;
        if (run) {
#pragma unroll
            for (int u = 0; u < 4; ++u) old[u] = (unsigned)b[u] < (unsigned)c.num_blocks ? atomicAdd(&c.refcounts[b[u]], run) : 1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j0 + 32 * u < nb) dst[j0 + 32 * u] = b[u];
        if (run) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (j0 + 32 * u >= nb) continue;
                if ((unsigned)b[u] >= (unsigned)c.num_blocks) set_error(c, MENTAT_DEV_BAD_BLOCK, b[u]);
                else if (old[u] <= 0) set_error(c, MENTAT_DEV_REF_FREE, b[u]);
            }
        }
    }
    if (blockIdx.z == 0 && lane == 0) {
        c.nblocks[cs] = nb;
        c.ntok[cs] = ntok;
        c.tail[cs] = tail;
    }
}

// ---------------------------------------------------------------------------
// check and reset: CTA 0 checks the batch, all of them clear `order`
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_pages_begin(mentat_kv_cache c, const int32_t* slots, int n, int groups,
                                                     PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < c.num_blocks; b += (int64_t)gridDim.x * blockDim.x)
        w.order[b] = 0;
    for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < groups; k += gridDim.x * blockDim.x) w.base[k] = 0;
    if (blockIdx.x) return;
    const bool ok = slots_distinct(c, slots, n, bits, &s_bad);
    if (threadIdx.x == 0) {
        if (!ok) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
        *w.stop = has_error(c) ? 1 : 0;
        *reinterpret_cast<long long*>(w.stop + 2) = c.ctrl[MENTAT_CTRL_TAIL];
    }
}

__global__ void __launch_bounds__(256) k_order_clear(mentat_kv_cache c, int groups, PagesWs w) {
    griddep_wait();
    for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < groups; k += gridDim.x * blockDim.x) w.base[k] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<long long*>(w.stop + 2) = c.ctrl[MENTAT_CTRL_TAIL];
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < c.num_blocks; b += (int64_t)gridDim.x * blockDim.x)
        w.order[b] = 0;
}

// ---------------------------------------------------------------------------
// free: rows are (sequence i, layer l), row index i * layers + l
// ---------------------------------------------------------------------------
// the order of a release: its row, then its table entry; 0 is "none"
__device__ __forceinline__ uint32_t release_index(const mentat_kv_cache& c, int row, int j) {
    return (uint32_t)row * (uint32_t)c.max_blocks_per_seq + (uint32_t)j + 1u;
}

// Entries j of up to MARK_SEQS sequences that follow one another, in one layer: siblings have the same blocks
// there, so a run of equal ones is one subtraction, and the last one's index is the run's.
constexpr int MARK_SEQS = 8;
template <bool LEAD>
__global__ void __launch_bounds__(256) k_free_mark(mentat_kv_cache c, const int32_t* slots, int n, PagesWs w) {
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    const int l = blockIdx.x % c.num_layers, i0 = blockIdx.x / c.num_layers * MARK_SEQS, count = min(MARK_SEQS, n - i0);
    int nb[MARK_SEQS], most = 0;
#pragma unroll
    for (int k = 0; k < MARK_SEQS; ++k) {
        const int64_t si = seq_index(c, l, slots[i0 + min(k, count - 1)]);
        nb[k] = k < count ? table_len(c, si) : 0;
        if (!LEAD && blockIdx.y == 0 && threadIdx.x == 0 && k < count && c.nblocks[si] > c.max_blocks_per_seq)
            set_error(c, MENTAT_DEV_TABLE_OVERFLOW, slots[i0 + k]);
        most = max(most, nb[k]);
    }
    for (int j = blockIdx.y * blockDim.x + threadIdx.x; j < most; j += gridDim.y * blockDim.x) {
        int b[MARK_SEQS];
#pragma unroll
        for (int k = 0; k < MARK_SEQS; ++k) {
            const bool mine = j < nb[k] && (!LEAD || j >= w.lead[(i0 + k) * c.num_layers + l]);
            b[k] = mine ? table_row(c, l, slots[i0 + k])[j] : -1;
            if (mine && (unsigned)b[k] >= (unsigned)c.num_blocks) {
                set_error(c, MENTAT_DEV_BAD_BLOCK, b[k]);
                b[k] = -1;
            }
        }
        int run = 0;
#pragma unroll
        for (int k = 0; k < MARK_SEQS; ++k) {
            if (b[k] < 0) continue;  // (a run goes on behind it only if the next block differs: its own atomic)
            ++run;
            if (k + 1 < MARK_SEQS && b[k + 1 < MARK_SEQS ? k + 1 : k] == b[k]) continue;
            if (atomicSub(&c.refcounts[b[k]], run) < run) {
                atomicAdd(&c.refcounts[b[k]], run);
                set_error(c, MENTAT_DEV_RELEASE_FREE, b[k]);
            } else {
                atomicMax(&w.order[b[k]], release_index(c, (i0 + k) * c.num_layers + l, j));
            }
            run = 0;
        }
    }
}

// whether entry j of a row frees its block
__device__ __forceinline__ bool frees(const mentat_kv_cache& c, const PagesWs& w, int b, int row, int j) {
    return (unsigned)b < (unsigned)c.num_blocks && c.refcounts[b] == 0 && w.order[b] == release_index(c, row, j);
}

template <bool LEAD>
__global__ void __launch_bounds__(PAGES_THREADS) k_free_count(mentat_kv_cache c, const int32_t* slots, int rows, PagesWs w) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, row = blockIdx.x * PAGES_WARPS + (threadIdx.x >> 5);
    if (row >= rows || *w.stop) return;
    const int i = row / c.num_layers, l = row - i * c.num_layers;
    const int nb = table_len(c, seq_index(c, l, slots[i]));
    const int32_t* t = table_row(c, l, slots[i]);
    int n = 0;
    for (int j0 = LEAD ? w.lead[row] : 0; j0 < nb; j0 += 128) {
        int b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) b[u] = j0 + 32 * u + lane < nb ? t[j0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) n += frees(c, w, b[u], row, j0 + 32 * u + lane);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) {
        w.count[row] = n;
        if (n) atomicAdd(&w.base[blockIdx.x], n);  // the CTA's rows together
    }
}

// a row's new table and counters after a compaction in place
__device__ __forceinline__ void install(const mentat_kv_cache& c, const PagesWs& w, int row, int m, int64_t si, int32_t* t,
                                        int first, int step) {
    const int pages = (m + c.block_size - 1) / c.block_size, lead = w.lead[row];
    const int32_t* fresh = w.fresh + w.first[row];
    for (int j = lead + first; j < pages; j += step) t[j] = fresh[j - lead];
    if (first == 0) {
        c.nblocks[si] = pages;
        c.ntok[si] = m;
        c.tail[si] = m ? m - (pages - 1) * c.block_size : 0;
    }
}

// push, and the rows' new counters (empty, or what compaction kept: cu); a warp a row.  A CTA adds up the totals of
// the CTAs before it (8 rows each).
template <bool LEAD>
__global__ void __launch_bounds__(PAGES_THREADS) k_free_push(mentat_kv_cache c, const int32_t* slots, const int32_t* cu,
                                                             int rows, PagesWs w) {
    __shared__ int s_sum[PAGES_WARPS], s_count[PAGES_WARPS];
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * PAGES_WARPS + warp;
    int before = 0;
    for (int k = threadIdx.x; k < (int)blockIdx.x; k += PAGES_THREADS) before += w.base[k];
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) {
        s_sum[warp] = before;
        s_count[warp] = row < rows ? w.count[row] : 0;
    }
    __syncthreads();
    long long at = *reinterpret_cast<const long long*>(w.stop + 2);  // the tail before the batch
    int all = 0;
    for (int k = 0; k < PAGES_WARPS; ++k) {
        at += s_sum[k] + (k < warp ? s_count[k] : 0);
        all += s_count[k];
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) c.ctrl[MENTAT_CTRL_TAIL] = at + all;
    if (row >= rows) return;
    const int i = row / c.num_layers, l = row - i * c.num_layers;
    const int64_t si = seq_index(c, l, slots[i]);
    int32_t* t = table_row(c, l, slots[i]);
    if (s_count[warp]) {
        const int nb = table_len(c, si);
        for (int j0 = LEAD ? w.lead[row] : 0; j0 < nb; j0 += 32) {
            const int j = j0 + lane, b = j < nb ? t[j] : -1;
            const bool go = frees(c, w, b, row, j);
            const uint32_t who = __ballot_sync(0xffffffffu, go);
            if (go) c.free_ring[(at + __popc(who & ((1u << lane) - 1))) % c.num_blocks] = b;
            at += __popc(who);
        }
    }
    __syncwarp();  // the old entries and counters have been read
    if (LEAD)
        install(c, w, row, cu[i + 1] - cu[i], si, t, lane, 32);
    else if (lane == 0)
        c.nblocks[si] = c.ntok[si] = c.tail[si] = 0;
}

// ---------------------------------------------------------------------------
// the same in one cluster
// ---------------------------------------------------------------------------
constexpr int CLUSTER_CTAS = 8, CLUSTER_THREADS = 1024, CLUSTER_WARPS = CLUSTER_THREADS / 32;
constexpr int CLUSTER_ALL_WARPS = CLUSTER_CTAS * CLUSTER_WARPS;

// the sum of s_total over the warps of the cluster before this one, and over all of them (a cluster barrier
// between the writes and this call)
__device__ __forceinline__ int before_warp(cg::cluster_group& cluster, int* s_total, int* all) {
    const int lane = threadIdx.x & 31, me = cluster.block_rank() * CLUSTER_WARPS + (threadIdx.x >> 5);
    int before = 0, total = 0;
    for (int w = lane; w < CLUSTER_ALL_WARPS; w += 32) {
        const int v = cluster.map_shared_rank(s_total, w / CLUSTER_WARPS)[w % CLUSTER_WARPS];
        total += v;
        before += w < me ? v : 0;
    }
    *all = __reduce_add_sync(0xffffffffu, total);
    return __reduce_add_sync(0xffffffffu, before);
}

// Items are 32 entries of a row (the last chunk of a row goes on to its end); a warp takes `per` items that
// follow one another, so a scan over the warps' totals orders the pushes.  Entries stay in shared memory
// between the steps: [CLUSTER_WARPS][per][32], negative once they are settled.
template <bool LEAD>
__global__ void __launch_bounds__(CLUSTER_THREADS) k_free_cluster(mentat_kv_cache c, const int32_t* slots, const int32_t* cu,
                                                                  int n, int chunks, int per, PagesWs w) {
    extern __shared__ uint32_t dyn[];
    __shared__ int s_bad, s_total[CLUSTER_WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster.block_rank();
    int* held = reinterpret_cast<int*>(dyn) + warp * per * 32 + lane;
    uint32_t* bits = dyn + CLUSTER_WARPS * per * 32;
    const int rows = n * c.num_layers, items = rows * chunks, me = rank * CLUSTER_WARPS + warp;
    const int y0 = min(items, me * per), y1 = min(items, y0 + per);
    // the entries are read while the batch is checked (a slot that is out of range has none)
    const long long tail0 = c.ctrl[MENTAT_CTRL_TAIL];
    bool stop = LEAD ? *w.stop != 0 : has_error(c);
    int over = -1;  // a slot whose table is longer than its room
    for (int y = y0; y < y1; ++y) {
        const int row = y / chunks, j = y % chunks * 32 + lane, i = row / c.num_layers, l = row - i * c.num_layers;
        const int slot = slots[i], lead = LEAD && !stop ? w.lead[row] : 0;
        int b = -1;
        if (slot >= 0 && slot < c.max_seqs) {
            const int nb = c.nblocks[seq_index(c, l, slot)];
            if (nb > c.max_blocks_per_seq) over = slot;
            if (j >= lead && j < min(nb, c.max_blocks_per_seq)) {
                b = table_row(c, l, slot)[j];
                if ((unsigned)b >= (unsigned)c.num_blocks) b = -2;  // recorded once all CTAs have looked at the error word
            }
        }
        held[(y - y0) * 32] = b;
    }
    if (!LEAD) {
        const bool bad = !slots_distinct(c, slots, n, bits, &s_bad);
        stop = __syncthreads_or(stop || bad);
        if (bad && threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
    }
    // an earlier error, or this one, stops every CTA: nothing of this call is recorded before all have looked
    if (stop) return;
    // entries past an item's first 32 (a table longer than the launch was sized for) are read again each time
    auto rest = [&](int y, auto&& f) {
        if (y % chunks != chunks - 1) return;
        const int row = y / chunks, i = row / c.num_layers, l = row - i * c.num_layers;
        const int nb = table_len(c, seq_index(c, l, slots[i])), lead = LEAD ? w.lead[row] : 0;
        const int32_t* t = table_row(c, l, slots[i]);
        for (int j0 = chunks * 32; j0 < nb; j0 += 32) {
            const int j = j0 + lane, b = j < nb && j >= lead ? t[j] : -1;
            f(row, j, (unsigned)b < (unsigned)c.num_blocks ? b : -1);
        }
    };
    for (int y = y0; y < y1; ++y) {
        const int b = held[(y - y0) * 32];
        if (b >= 0) w.order[b] = 0;
        rest(y, [&](int, int, int b) {
            if (b >= 0) w.order[b] = 0;
        });
    }
    cluster.sync();
    if (!LEAD && over >= 0 && lane == 0) set_error(c, MENTAT_DEV_TABLE_OVERFLOW, over);
    auto mark = [&](int row, int j, int b) {
        if (b < 0) return;
        if (atomicSub(&c.refcounts[b], 1) <= 0) {
            atomicAdd(&c.refcounts[b], 1);
            set_error(c, MENTAT_DEV_RELEASE_FREE, b);
            return;
        }
        atomicMax(&w.order[b], release_index(c, row, j));
    };
    for (int y = y0; y < y1; ++y) {
        const int row = y / chunks, j = y % chunks * 32 + lane, b = held[(y - y0) * 32];
        if (b == -2) set_error(c, MENTAT_DEV_BAD_BLOCK, table_row(c, row % c.num_layers, slots[row / c.num_layers])[j]);
        mark(row, j, b);
        rest(y, mark);
    }
    cluster.sync();
    auto freed = [&](int row, int j, int b) {
        return b >= 0 && __ldcg(&w.order[b]) == release_index(c, row, j) && __ldcg(&c.refcounts[b]) == 0;
    };
    int mine = 0;
    for (int y = y0; y < y1; ++y) {
        const int b = held[(y - y0) * 32];
        const bool go = freed(y / chunks, y % chunks * 32 + lane, b);
        if (!go) held[(y - y0) * 32] = -1;
        mine += __popc(__ballot_sync(0xffffffffu, go));
        rest(y, [&](int row, int j, int b) { mine += __popc(__ballot_sync(0xffffffffu, freed(row, j, b))); });
    }
    if (lane == 0) s_total[warp] = mine;
    cluster.sync();
    int all;
    long long at = tail0 + before_warp(cluster, s_total, &all);
    auto push = [&](int b) {
        const uint32_t who = __ballot_sync(0xffffffffu, b >= 0);
        if (b >= 0) c.free_ring[(at + __popc(who & ((1u << lane) - 1))) % c.num_blocks] = b;
        at += __popc(who);
    };
    for (int y = y0; y < y1; ++y) {
        push(held[(y - y0) * 32]);
        rest(y, [&](int row, int j, int b) { push(freed(row, j, b) ? b : -1); });
    }
    cluster.sync();  // every CTA has read the old tail, the others' totals and the tables
    if (rank == 0 && threadIdx.x == 0) c.ctrl[MENTAT_CTRL_TAIL] = tail0 + all;
    for (int row = me; row < rows; row += CLUSTER_ALL_WARPS) {
        const int i = row / c.num_layers, l = row - i * c.num_layers;
        const int64_t si = seq_index(c, l, slots[i]);
        if (LEAD)
            install(c, w, row, cu[i + 1] - cu[i], si, table_row(c, l, slots[i]), lane, 32);
        else if (lane == 0)
            c.nblocks[si] = c.ntok[si] = c.tail[si] = 0;
    }
}

// ---------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------
struct CompactArgs {
    const int32_t* src;
    const int32_t* dst;  // NULL: in place
    const int32_t* keep;
    int64_t keep_ls, total;
    const int32_t* cu;
    int n;
};

constexpr int PLAN_CHUNK = 512;  // kept positions of a warp's step; the last chunk goes on to the end of a list
// The plan, in one cluster, a warp a range of rows: the batch is checked, the kept positions are inside their
// sequences; how many pages at the front stay, and the fresh blocks of the others.  Bound by latency (the lists
// are a thousandth of the bytes that are moved): 12 us for 8 sequences in 4 layers, 21 for 12 of 16,000 tokens in 2;
// alone with cold caches 16 and 26.
__global__ void __launch_bounds__(CLUSTER_THREADS) k_compact_plan(mentat_kv_cache c, CompactArgs a, int chunks,
                                                                  PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad, s_list, s_is_list, s_total[CLUSTER_WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) s_is_list = 0;  // (slots_distinct synchronises)
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster.block_rank(), L = c.num_layers;
    // every CTA checks the whole batch
    const bool ok = slots_distinct(c, a.dst ? a.dst : a.src, a.n, bits, &s_bad);
    const bool before = has_error(c);
    int no = 0;
    if (a.dst && ok)  // sources in range, destinations empty in every layer (so none is a source with tokens)
        for (int64_t x = threadIdx.x; x < (int64_t)a.n * L; x += CLUSTER_THREADS) {
            const int i = (int)(x / L), l = (int)(x % L);
            if (a.src[i] < 0 || a.src[i] >= c.max_seqs || has_bit(bits, a.src[i])) {
                no = 1;
                s_bad = a.src[i];
            } else if (c.nblocks[seq_index(c, l, a.dst[i])] || c.ntok[seq_index(c, l, a.dst[i])]) {
                no = 1;
                s_bad = a.dst[i];
            }
        }
    for (int i = threadIdx.x; i < a.n; i += CLUSTER_THREADS)  // lists within keep: nothing of another is read
        if (a.cu[i] < 0 || a.cu[i + 1] < a.cu[i] || a.cu[i + 1] > a.total) {
            no = 1;
            s_list = a.cu[i + 1];
            s_is_list = 1;
        }
    bool stop = __syncthreads_or(no || !ok || before);
    if (stop && threadIdx.x == 0 && !before) {
        if (s_is_list) set_error(c, MENTAT_DEV_BAD_TOKEN, s_list);
        else set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
    }
    const int rows = a.n * L, per = (rows + CLUSTER_ALL_WARPS - 1) / CLUSTER_ALL_WARPS;
    const int r0 = min(rows, (rank * CLUSTER_WARPS + warp) * per), r1 = min(rows, r0 + per);
    if (!stop)
        for (int row = r0 + lane; row < r1; row += 32) w.count[row] = a.cu[row / L + 1] - a.cu[row / L];
    cluster.sync();  // all have looked at the error word before this call writes it
    // the first position that moves: chunks of the lists over all warps
    if (!stop)
        for (int64_t y = rank * CLUSTER_WARPS + warp; y < (int64_t)rows * chunks; y += CLUSTER_ALL_WARPS) {
            const int row = (int)(y / chunks), i = row / L, l = row - i * L;
            const int m = a.cu[i + 1] - a.cu[i], j0 = (int)(y % chunks) * PLAN_CHUNK, j1 = chunks - 1 == y % chunks ? m : min(m, j0 + PLAN_CHUNK);
            if (j0 >= j1) continue;
            const int len = c.ntok[seq_index(c, l, a.src[i])];
            const int32_t* keep = a.keep + l * a.keep_ls + a.cu[i];
            int first = m;
            for (int j = j0 + lane; j < j1; j += 256) {
                int t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] = j + 32 * u < j1 ? keep[j + 32 * u] : j + 32 * u;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (j + 32 * u < j1 && (t[u] < 0 || t[u] >= len)) set_error(c, MENTAT_DEV_BAD_TOKEN, t[u]);
                    if (t[u] != j + 32 * u) first = min(first, j + 32 * u);
                }
            }
            first = __reduce_min_sync(0xffffffffu, first);
            if (lane == 0 && first < m) atomicMin(&w.count[row], first);
        }
    cluster.sync();
    int demand = 0;
    if (!stop)
        for (int row = r0; row < r1; ++row) {
            const int i = row / L, l = row - i * L;
            const int m = a.cu[i + 1] - a.cu[i], len = c.ntok[seq_index(c, l, a.src[i])], first = __ldcg(&w.count[row]);
            const int pages = (m + c.block_size - 1) / c.block_size;
            // a page kept in part is copied even if its tokens stay in place: sequences whose tail is one
            // block have tails of one length (the batched append relies on it)
            const int lead = first == m && m == len ? pages : first / c.block_size;
            if (lane == 0) {
                if (pages > c.max_blocks_per_seq || table_overflows(c, seq_index(c, l, a.src[i])))
                    set_error(c, MENTAT_DEV_TABLE_OVERFLOW, a.src[i]);
                w.lead[row] = lead;
                w.first[row] = demand;  // within the warp, so far
                w.count[row] = pages - lead;
            }
            demand += pages - lead;
        }
    if (lane == 0) s_total[warp] = demand;
    const long long head = c.ctrl[MENTAT_CTRL_HEAD], tail = c.ctrl[MENTAT_CTRL_TAIL];
    __threadfence();
    cluster.sync();
    stop = stop || has_error(c);  // written before the barrier, if at all
    int all;
    const int base = before_warp(cluster, s_total, &all);
    const bool short_of = !stop && all > tail - head;
    cluster.sync();  // everyone has read the error word, the totals and the control words
    if (rank == 0 && threadIdx.x == 0) {
        if (short_of) set_error(c, MENTAT_DEV_OUT_OF_BLOCKS, c.num_blocks);
        w.stop[0] = stop || short_of;
        w.stop[1] = all;
        if (!stop && !short_of) {
            c.ctrl[MENTAT_CTRL_HEAD] = head + all;
            const long long used = c.num_blocks - (tail - head - all);
            if (used > c.ctrl[MENTAT_CTRL_PEAK]) c.ctrl[MENTAT_CTRL_PEAK] = used;
            c.ctrl[MENTAT_CTRL_ALLOCS] += all;
        }
    }
    if (stop || short_of) return;
    for (int row = r0; row < r1; ++row) {
        const int first = w.first[row] + base, count = w.count[row];
        __syncwarp();
        if (lane == 0) w.first[row] = first;
        for (int j = lane; j < count; j += 256) {
            int b[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) b[u] = j + 32 * u < count ? c.free_ring[(head + first + j + 32 * u) % c.num_blocks] : -1;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (b[u] >= 0) {
                    w.fresh[first + j + 32 * u] = b[u];
                    c.refcounts[b[u]] = 1;
                }
        }
    }
}

// What a compaction into new sequences leaves in their tables: shared pages with a reference more, fresh ones,
// counters; rows spread over the grid.
__device__ __forceinline__ void install_new(const mentat_kv_cache& c, const CompactArgs& a, const PagesWs& w, int step) {
    const int rows = a.n * c.num_layers;
    for (int row = blockIdx.x; row < rows; row += step) {
        const int i = row / c.num_layers, l = row - i * c.num_layers, lead = w.lead[row];
        const int32_t* s = table_row(c, l, a.src[i]);
        int32_t* to = table_row(c, l, a.dst[i]);
        for (int j = threadIdx.x; j < lead; j += blockDim.x) {
            const int b = s[j];
            to[j] = b;
            if ((unsigned)b >= (unsigned)c.num_blocks) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            else if (atomicAdd(&c.refcounts[b], 1) <= 0) set_error(c, MENTAT_DEV_REF_FREE, b);
        }
        install(c, w, row, a.cu[i + 1] - a.cu[i], seq_index(c, l, a.dst[i]), to, threadIdx.x, blockDim.x);
    }
}

// Where fresh page f goes: its row, found from the rows' first fresh pages, and its place in the row
struct FreshPage {
    int row, page;
};
__device__ __forceinline__ FreshPage fresh_page(const PagesWs& w, int rows, int f) {
    int lo = 0, hi = rows - 1;  // the last row that begins at or before f (rows without fresh pages begin where the next does)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (w.first[mid] <= f) lo = mid; else hi = mid - 1;
    }
    return FreshPage{lo, w.lead[lo] + f - w.first[lo]};
}

// The kept tokens of the fresh pages, element by element (heads that 16-byte accesses do not divide, or rows too
// long for the ring of k_compact_stream): a CTA a page, a warp a token.
constexpr int MOVE_THREADS = 256, MOVE_TOKENS = 16;
template <typename T, bool IL>
__global__ void __launch_bounds__(MOVE_THREADS) k_compact_move(mentat_kv_cache c, CompactArgs a, mentat_rotary r, PagesWs w) {
    extern __shared__ float cs[];  // [MOVE_TOKENS][2 pairs]
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    if (a.dst) install_new(c, a, w, gridDim.x);
    const int tid = threadIdx.x, lane = tid & 31, D = c.head_dim, H = c.num_kv_heads, bs = c.block_size, n = H * D;
    T* kp = reinterpret_cast<T*>(c.k_pool);
    T* vp = reinterpret_cast<T*>(c.v_pool);
    for (int f = blockIdx.x; f < w.stop[1]; f += gridDim.x) {
        const FreshPage fp = fresh_page(w, a.n * c.num_layers, f);
        const int i = fp.row / c.num_layers, l = fp.row - i * c.num_layers, m = a.cu[i + 1] - a.cu[i];
        const int32_t* keep = a.keep + l * a.keep_ls + a.cu[i];
        const int32_t* t = table_row(c, l, a.src[i]);
        const int64_t to = pool_row(c, l, w.fresh[f], 0);
        for (int j0 = fp.page * bs; j0 < min(m, (fp.page + 1) * bs); j0 += MOVE_TOKENS) {
            const int count = min(min(m, (fp.page + 1) * bs) - j0, MOVE_TOKENS);
            __syncthreads();
            for (int x = tid; x < count * r.pairs; x += MOVE_THREADS) {
                const int k = x / r.pairs, e = x - k * r.pairs;
                rotary_angle(r, e, j0 + k - keep[j0 + k], cs + k * 2 * r.pairs + e, cs + k * 2 * r.pairs + r.pairs + e);
            }
            __syncthreads();
            for (int k = tid >> 5; k < count; k += MOVE_THREADS / 32) {
                const int from = keep[j0 + k], b = t[from / bs];
                if ((unsigned)b >= (unsigned)c.num_blocks) {
                    if (lane == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
                    continue;
                }
                const int64_t src = pool_row(c, l, b, from % bs), dst = to + (int64_t)(j0 + k - fp.page * bs) * n;
                const float* tab = cs + k * 2 * r.pairs;
                for (int x = lane; x < n; x += 32) {
                    const int d = x % D - r.offset;
                    float v = Elem<T>::to_f(kp[src + x]);
                    if (from != j0 + k && d >= 0 && d < 2 * r.pairs) {
                        const bool low = IL ? !(d & 1) : d < r.pairs;  // first or second of its pair
                        const int e = IL ? d / 2 : low ? d : d - r.pairs, step = IL ? 1 : r.pairs;
                        const float o = Elem<T>::to_f(kp[src + (low ? x + step : x - step)]);
                        v = low ? v * tab[e] - o * tab[r.pairs + e] : o * tab[r.pairs + e] + v * tab[e];
                    }
                    kp[dst + x] = Elem<T>::from_f(v);
                    vp[dst + x] = vp[src + x];
                }
            }
        }
    }
}

// A token's heads turned in place in shared memory by a table (cosines, then sines), a warp.  Where the 32 lanes
// cover whole heads, a lane has the same pairs in every head and keeps their cosines and sines.
template <typename T, int VEC, bool IL>
__device__ __forceinline__ void turn_row(T* row, int H, int D, const mentat_rotary& r, const float* tab) {
    using P = Pack<T, VEC>;
    const int lane = threadIdx.x & 31, pairs = r.pairs, off = r.offset;
    const int tasks = IL ? 2 * pairs / VEC : pairs / VEC, total = H * tasks;
    constexpr int N = IL ? VEC / 2 : VEC;
    float co[N], sn[N];
    auto fetch = [&](int t) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            co[e] = tab[t * N + e];
            sn[e] = tab[pairs + t * N + e];
        }
    };
    const bool whole = 32 % tasks == 0;
    if (whole) fetch(lane % tasks);
    for (int x = lane; x < total; x += 32) {
        const int h = x / tasks, t = x - h * tasks;
        if (!whole) fetch(t);
        T* p = row + h * D + off + t * VEC;
        P a = *reinterpret_cast<const P*>(p);
        if (IL) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float u = Elem<T>::to_f(a.v[2 * e]), v = Elem<T>::to_f(a.v[2 * e + 1]);
                a.v[2 * e] = Elem<T>::from_f(u * co[e] - v * sn[e]);
                a.v[2 * e + 1] = Elem<T>::from_f(u * sn[e] + v * co[e]);
            }
        } else {
            P b = *reinterpret_cast<const P*>(p + pairs);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float u = Elem<T>::to_f(a.v[e]), v = Elem<T>::to_f(b.v[e]);
                a.v[e] = Elem<T>::from_f(u * co[e] - v * sn[e]);
                b.v[e] = Elem<T>::from_f(u * sn[e] + v * co[e]);
            }
            *reinterpret_cast<P*>(p + pairs) = b;
        }
        *reinterpret_cast<P*>(p) = a;
    }
}

// The same with the rows in shared memory: persistent CTAs take ranges of the fresh pages, `tokens` rows at a time
// through a ring of stages.  A producer warp looks up where the rows come from and copies them in with bulk
// copies, K and V, a stage ahead or more; eight warps turn K in place; the stage, which is contiguous in the
// fresh page, leaves as two bulk copies.  So the bytes pass through registers only where they change, and the
// next rows are always on the way.  Bound by memory: 1.3 GB in 229 us alone, 5.7 TB/s (through registers, a CTA a page: 3.0);
// 75 MB in 23 us with cold caches, 19 among other calls, of which the first and last stages, which nothing covers, are 6.
constexpr int STREAM_WORKERS = 256, STREAM_THREADS = STREAM_WORKERS + 32, STREAM_MAX_STAGES = 4;
template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(STREAM_THREADS) k_compact_stream(mentat_kv_cache c, CompactArgs a, mentat_rotary r,
                                                                   int tokens, int stages, PagesWs w) {
    extern __shared__ __align__(128) uint8_t ring[];  // [stages][K, V][tokens][row], then cosines and sines [tokens][2 pairs]
    __shared__ uint64_t s_full[STREAM_MAX_STAGES], s_empty[STREAM_MAX_STAGES];
    __shared__ int s_shift[STREAM_MAX_STAGES][MOVE_TOKENS], s_count[STREAM_MAX_STAGES], s_abort;
    __shared__ int64_t s_to[STREAM_MAX_STAGES];
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(smem_u32(s_full + s), 1);
            mbar_init(smem_u32(s_empty + s), 1);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    __syncthreads();
    if (a.dst) install_new(c, a, w, gridDim.x);
    const int D = c.head_dim, H = c.num_kv_heads, bs = c.block_size, rows = a.n * c.num_layers;
    const uint32_t row_bytes = H * D * sizeof(T), tile = tokens * row_bytes;
    const int64_t total = w.stop[1];
    const int f0 = (int)(total * blockIdx.x / gridDim.x), f1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
    const int groups = (bs + tokens - 1) / tokens, items = (f1 - f0) * groups;
    T* kp = reinterpret_cast<T*>(c.k_pool);
    T* vp = reinterpret_cast<T*>(c.v_pool);
    if (tid >= STREAM_WORKERS) {  // producer
        FreshPage fp = fresh_page(w, rows, min(f0, (int)total - 1 < 0 ? 0 : (int)total - 1));
        int row_end = 0, i = 0, l = 0, m = 0, it = 0;
        const int32_t *keep = nullptr, *t = nullptr;
        auto enter = [&]() {  // fp.row's data
            i = fp.row / c.num_layers;
            l = fp.row - i * c.num_layers;
            m = a.cu[i + 1] - a.cu[i];
            keep = a.keep + l * a.keep_ls + a.cu[i];
            t = table_row(c, l, a.src[i]);
            row_end = w.first[fp.row] + w.count[fp.row];
        };
        if (items) enter();
        for (; it < items; ++it) {
            const int f = f0 + it / groups, s = it % stages;
            if (it % groups == 0 && it) {
                ++fp.page;
                while (f >= row_end) {  // the next row with fresh pages
                    ++fp.row;
                    fp.page = w.lead[fp.row];
                    enter();
                }
            }
            const int j0 = fp.page * bs + it % groups * tokens;
            const int count = max(0, min(min(m, (fp.page + 1) * bs) - j0, tokens));
            int from = -1;
            int64_t src = -1;
            if (lane < count) {
                from = keep[j0 + lane];
                const int b = t[from / bs];
                if ((unsigned)b < (unsigned)c.num_blocks) src = pool_row(c, l, b, from % bs);
                else set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            }
            const int to = w.fresh[f];
            if (it >= stages && !__all_sync(0xffffffffu, mbar_wait(smem_u32(s_empty + s), (it / stages - 1) & 1))) {
                if (lane == 0) {
                    set_error(c, MENTAT_DEV_DECODE_TIMEOUT, 9);
                    *(volatile int*)&s_abort = 1;
                }
                break;
            }
            if (lane < tokens) s_shift[s][lane] = src >= 0 && r.pairs ? j0 + lane - from : 0;
            if (lane == 0) {
                s_count[s] = count;
                s_to[s] = pool_row(c, l, to, 0) + (int64_t)(j0 - fp.page * bs) * H * D;
            }
            const uint32_t good = __ballot_sync(0xffffffffu, src >= 0);
            __syncwarp();
            const uint32_t bar = smem_u32(s_full + s), dst = smem_u32(ring) + s * 2 * tile + lane * row_bytes;
            if (lane == 0) mbar_expect_tx(bar, 2 * row_bytes * __popc(good));
            __syncwarp();
            if (src >= 0) {
                bulk_load(dst, kp + src, row_bytes, bar);
                bulk_load(dst + tile, vp + src, row_bytes, bar);
            }
        }
        // every stage that was asked for has arrived before the CTA may end
        for (int k = max(0, it - stages); k < it; ++k) (void)mbar_wait(smem_u32(s_full + k % stages), (k / stages) & 1);
        return;
    }
    float* tab = reinterpret_cast<float*>(ring + (size_t)stages * 2 * tile);
    for (int it = 0; it < items; ++it) {
        const int s = it % stages;
        if (!mbar_wait(smem_u32(s_full + s), (it / stages) & 1)) {
            set_error(c, MENTAT_DEV_DECODE_TIMEOUT, 10);
            *(volatile int*)&s_abort = 1;
        }
        const int count = s_count[s];
        if (r.pairs) {
            for (int x = tid; x < count * r.pairs; x += STREAM_WORKERS) {
                const int k = x / r.pairs, e = x - k * r.pairs, shift = s_shift[s][k];
                // neighbours that moved together share the table of the first of them
                if (shift && (k == 0 || s_shift[s][k - 1] != shift))
                    rotary_angle(r, e, shift, tab + k * 2 * r.pairs + e, tab + k * 2 * r.pairs + r.pairs + e);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int k = tid >> 5; k < count; k += STREAM_WORKERS / 32) {
                const int shift = s_shift[s][k];
                if (!shift) continue;
                int own = k;
                while (own && s_shift[s][own - 1] == shift) --own;
                turn_row<T, VEC, IL>(reinterpret_cast<T*>(ring + (size_t)s * 2 * tile + k * row_bytes), H, D, r,
                                     tab + own * 2 * r.pairs);
            }
            fence_proxy_async();
        }
        // the workers leave together, whatever each has seen of the flag
        int gone;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\t"
                     "selp.s32 %0, 1, 0, q;\n\t}"
                     : "=r"(gone)
                     : "r"(*(volatile int*)&s_abort)
                     : "memory");
        if (gone) break;
        if (tid == 0) {
            if (count) {
                bulk_store(kp + s_to[s], smem_u32(ring) + s * 2 * tile, count * row_bytes);
                bulk_store(vp + s_to[s], smem_u32(ring) + s * 2 * tile + tile, count * row_bytes);
            } else {
                asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.commit_group;" ::: "memory");
            }
            // the stage before has been read by its copies: two groups a stage
            asm volatile("cp.async.bulk.wait_group.read 2;" ::: "memory");
            if (it) mbar_arrive(smem_u32(s_empty + (it - 1) % stages));
        }
    }
    if (tid == 0) bulk_wait_all();
}

}  // namespace mentat

using namespace mentat;

static bool bad_pages(const mentat_kv_cache* c, int32_t n) {
    return !c || c->num_layers <= 0 || c->num_layers > 65535 || c->num_blocks <= 0 || c->block_size <= 0 ||
           c->max_seqs <= 0 || c->max_blocks_per_seq <= 0 || !c->refcounts || !c->free_ring || !c->ctrl ||
           !c->tables || !c->nblocks || !c->ntok || !c->tail || n < 0 || n > PAGES_MAX_SEQS;
}
static size_t bitmap_bytes(const mentat_kv_cache* c) { return ((size_t)c->max_seqs + 31) / 32 * 4; }
// the bitmap fits in shared memory
static bool slots_fit(const mentat_kv_cache* c) { return bitmap_bytes(c) <= 48 * 1024; }
// and a release's index in 32 bits
static bool pages_fit(const mentat_kv_cache* c, int32_t n) {
    return slots_fit(c) && (int64_t)n * c->num_layers * c->max_blocks_per_seq < 0xffffffffll;
}
static int chunks_of(int64_t work, int64_t each, int64_t most) {
    const int64_t x = (work + each - 1) / each;
    return (int)(x < 1 ? 1 : x > most ? most : x);
}

// a kernel over one cluster of CLUSTER_CTAS
template <auto KERNEL, typename... Args>
static int launch_one_cluster(size_t smem, cudaStream_t s, Args... args) {
    return launch_cluster<KERNEL>(CLUSTER_CTAS, dim3(CLUSTER_CTAS), CLUSTER_THREADS, smem, s, args...);
}

// Releases are one cluster's work while a warp has at most this many groups of 32 table entries.  One launch instead
// of four saves the host 6 us (fork and free of 6 sequences: 16.5 and 22.4).  On the device both are as fast at 1 a
// warp (8 siblings of 30 pages in 32 layers: 15.3); at 3 the cluster takes 22 us and four launches 40 for 12
// sequences of 440 pages of their own, at 4 it is 25 and 17 for 16 siblings of 60 pages, which k_free_mark takes
// in runs; 32 of them, 8 a warp, 40 and 19.
constexpr int FREE_CLUSTER_PER = 4;

template <bool LEAD>
static int launch_free(const mentat_kv_cache* c, const int32_t* slots, const int32_t* cu, int32_t n, int32_t max_nb,
                       const PagesWs& w, cudaStream_t s) {
    if (max_nb > c->max_blocks_per_seq) max_nb = c->max_blocks_per_seq;
    const int rows = n * c->num_layers, chunks = max_nb < 1 ? 1 : (max_nb + 31) / 32;
    const int64_t per = ((int64_t)rows * chunks + CLUSTER_ALL_WARPS - 1) / CLUSTER_ALL_WARPS;
    const size_t held = (size_t)CLUSTER_WARPS * per * 32 * 4;
    if (per <= FREE_CLUSTER_PER && held + bitmap_bytes(c) <= 100 * 1024)
        return launch_one_cluster<k_free_cluster<LEAD>>(held + bitmap_bytes(c), s, *c, slots, cu, n, chunks, (int)per, w);
    const dim3 clear(chunks_of(c->num_blocks, 1024, 148)), by_row((rows + PAGES_WARPS - 1) / PAGES_WARPS);
    if (!LEAD)
        MENTAT_LAUNCH(k_pages_begin, clear, dim3(256), bitmap_bytes(c), s, *c, slots, n, (int)by_row.x, w);
    else
        MENTAT_LAUNCH(k_order_clear, clear, dim3(256), 0, s, *c, (int)by_row.x, w);
    const dim3 marks((n + MARK_SEQS - 1) / MARK_SEQS * c->num_layers, chunks_of(max_nb, 256, 64));
    MENTAT_LAUNCH(k_free_mark<LEAD>, marks, dim3(256), 0, s, *c, slots, n, w);
    MENTAT_LAUNCH(k_free_count<LEAD>, by_row, dim3(PAGES_THREADS), 0, s, *c, slots, rows, w);
    MENTAT_LAUNCH(k_free_push<LEAD>, by_row, dim3(PAGES_THREADS), 0, s, *c, slots, cu, rows, w);
    return MENTAT_OK;
}

namespace {
// The launch that moves the rows.  With `ready`, only what may refuse it: asked before the plan, whose fresh blocks
// would belong to no table if the rows could not be moved.
struct LaunchCompactMove {
    const mentat_kv_cache& c;
    const CompactArgs& a;
    const mentat_rotary& r;
    const PagesWs& w;
    int max_keep;
    cudaStream_t s;
    bool ready;
    template <auto KERNEL>
    static int reserve() {
        if (reserve_smem<KERNEL>() == cudaSuccess) return MENTAT_OK;
        (void)cudaGetLastError();
        return MENTAT_ERR_CUDA;
    }
    template <typename T, int VEC, bool IL>
    int operator()() {
        const int64_t rows = (int64_t)a.n * c.num_layers, most = rows * ((max_keep + c.block_size - 1) / c.block_size);
        const size_t table = (size_t)MOVE_TOKENS * 2 * r.pairs * sizeof(float);
        if constexpr (VEC > 1) {
            // stages of up to 16 tokens and 64 KB, three of them or four; several CTAs on an SM where they are small.
            // 12 sequences, 1.3 GB (64 KB for 16 tokens): 277 us with 16 tokens, 308 with 8, 320 with 4; 3 or 4
            // stages are alike, 2 take 438.
            const int64_t row = (int64_t)c.num_kv_heads * c.head_dim * sizeof(T);
            int tokens = c.block_size < MOVE_TOKENS ? c.block_size : MOVE_TOKENS;
            while (tokens > 1 && 2 * tokens * row > 64 * 1024) tokens /= 2;
            const int64_t room = 220 * 1024 - (int64_t)table - 1024, stage = 2 * tokens * row;
            int stages = (int)(room / stage < STREAM_MAX_STAGES ? room / stage : STREAM_MAX_STAGES);
            if (stages >= 2) {
                const size_t smem = stages * stage + table;
                int per_sm = (int)(220 * 1024 / (smem + 2048));
                per_sm = per_sm < 1 ? 1 : per_sm > 6 ? 6 : per_sm;
                if (ready) return reserve<k_compact_stream<T, VEC, IL>>();
                MENTAT_LAUNCH((k_compact_stream<T, VEC, IL>), dim3(chunks_of(most, 1, 148 * per_sm)), dim3(STREAM_THREADS), smem, s, c, a, r, tokens,
                              stages, w);
                return MENTAT_OK;
            }
        }
        if (ready) return reserve<k_compact_move<T, IL>>();
        MENTAT_LAUNCH((k_compact_move<T, IL>), dim3(chunks_of(most, 1, 148 * 8)), dim3(MOVE_THREADS), table, s, c, a, r, w);
        return MENTAT_OK;
    }
};
}  // namespace

extern "C" {

int64_t mentat_pages_workspace_bytes(const mentat_kv_cache* c, int32_t n) {
    return bad_pages(c, n) ? 0 : pages_ws(c, n, nullptr, nullptr);
}

int mentat_kv_fork_batched(const mentat_kv_cache* c, const int32_t* parents, const int32_t* children, int32_t n, cudaStream_t s) {
    if (bad_pages(c, n) || (n > 0 && (!parents || !children))) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!slots_fit(c)) return MENTAT_ERR_UNSUPPORTED;
    // two CTAs an SM at least, if the tables may be long enough (how long they are, only the device knows)
    const int by_child = (n + PAGES_WARPS - 1) / PAGES_WARPS;
    const int parts = 2 * 148 / (by_child * c->num_layers);
    const dim3 grid(by_child, c->num_layers, parts < 2 ? 1 : chunks_of(c->max_blocks_per_seq, 128, parts));
    MENTAT_LAUNCH(k_fork_check, dim3(chunks_of((int64_t)n * c->num_layers, PAGES_THREADS, 148)), dim3(PAGES_THREADS),
                  bitmap_bytes(c), s, *c, parents, children, n);
    MENTAT_LAUNCH(k_fork_batched, grid, dim3(PAGES_THREADS), 0, s, *c, parents, children, n);
    return MENTAT_OK;
}

int mentat_kv_free_batched(const mentat_kv_cache* c, const int32_t* slots, int32_t n, int32_t max_nb, void* workspace,
                           int64_t workspace_bytes, cudaStream_t s) {
    if (bad_pages(c, n) || max_nb < 0 || (n > 0 && (!slots || !workspace || ((uintptr_t)workspace & 15)))) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!pages_fit(c, n)) return MENTAT_ERR_UNSUPPORTED;
    PagesWs w;
    if (workspace_bytes < pages_ws(c, n, workspace, &w)) return MENTAT_ERR_ARG;
    return launch_free<false>(c, slots, nullptr, n, max_nb, w, s);
}

int mentat_kv_compact(const mentat_kv_cache* c, const int32_t* src, const int32_t* dst, int32_t n, const int32_t* keep,
                      int64_t keep_ls, int64_t total, const int32_t* cu, int32_t max_keep, int32_t max_nb,
                      const mentat_rotary* r, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
    if (bad_pages(c, n) || max_keep < 0 || max_nb < 0 || keep_ls < 0 || total < 0 || c->head_dim <= 0 || c->num_kv_heads <= 0 ||
        (n > 0 && (!src || !cu || !workspace || ((uintptr_t)workspace & 15) || !c->k_pool || !c->v_pool || (total > 0 && !keep))) ||
        (r && !rotary_ok(r, c->head_dim)))
        return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!pages_fit(c, n)) return MENTAT_ERR_UNSUPPORTED;
    PagesWs w;
    if (workspace_bytes < pages_ws(c, n, workspace, &w)) return MENTAT_ERR_ARG;
    const int vec = 16 / dtype_bytes(c->dtype);
    mentat_rotary turn{};
    if (r) {
        turn = *r;
        turn.scale = 1.0f;
    }
    const bool wide = c->head_dim % vec == 0 && (!r || rotary_aligned(r, c->head_dim, vec)) &&
                      ((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) % 16 == 0;
    const CompactArgs a{src, dst, keep, keep_ls, total, cu, n};
    const auto move = [&](bool ready) {
        return rotary_dispatch(c->dtype, wide, turn.interleaved != 0, LaunchCompactMove{*c, a, turn, w, max_keep, s, ready});
    };
    if (!dst && reserve_smem<k_free_cluster<true>>() != cudaSuccess) {
        (void)cudaGetLastError();
        return MENTAT_ERR_CUDA;
    }
    int st = move(true);
    if (st == MENTAT_OK)
        st = launch_one_cluster<k_compact_plan>(bitmap_bytes(c), s, *c, a, chunks_of(max_keep, PLAN_CHUNK, 1 << 20), w);
    if (st == MENTAT_OK) st = move(false);
    return st != MENTAT_OK || dst ? st : launch_free<true>(c, src, cu, n, max_nb, w, s);
}

}  // extern "C"
