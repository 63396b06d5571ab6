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

#include <cooperative_groups.h>

#include "rotary.cuh"

namespace cg = cooperative_groups;

namespace mentat {

constexpr int PAGES_MAX_SEQS = 1024;

// workspace: [0] 1 = stop (an error, now or before), then order, the ids of fresh
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
__device__ __forceinline__ bool has_bit(const uint32_t* bits, int s) { return (bits[s >> 5] >> (s & 31)) & 1; }

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
// Every CTA checks the whole batch for itself, so all of them agree whether to go on.  A warp takes one
// (layer, run of children of one parent that follow one another): the parent's table is read once and each
// page's count rises by the run's length in one atomic.
constexpr int PAGES_THREADS = 256, PAGES_WARPS = PAGES_THREADS / 32;
__global__ void __launch_bounds__(PAGES_THREADS) k_fork_batched(mentat_kv_cache c, const int32_t* parents,
                                                                const int32_t* children, int n) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
    griddep_launch();
    const bool ok = slots_distinct(c, children, n, bits, &s_bad);
    int no = 0;
    if (ok)
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int p = parents[i];
            if (p < 0 || p >= c.max_seqs || has_bit(bits, p)) {
                no = 1;
                s_bad = p;
            }
        }
    if (__syncthreads_or(no) || !ok) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
        return;
    }
    if (has_error(c)) return;
    const int lane = threadIdx.x & 31, l = blockIdx.y, i = blockIdx.x * PAGES_WARPS + (threadIdx.x >> 5);
    if (i >= n) return;
    const int parent = parents[i];
    if (i > 0 && parents[i - 1] == parent) return;  // in an earlier warp's run
    int run = 1;
    while (i + run < n && parents[i + run] == parent) ++run;
    const int64_t ps = seq_index(c, l, parent);
    const int nb = c.nblocks[ps], ntok = c.ntok[ps], tail = c.tail[ps];
    const int32_t* src = table_row(c, l, parent);
    for (int j0 = 0; j0 < nb; j0 += 128) {
        int b[4];  // four entries of a lane on the way
#pragma unroll
        for (int u = 0; u < 4; ++u) b[u] = j0 + 32 * u + lane < nb ? src[j0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (j0 + 32 * u + lane >= nb) continue;
            if ((unsigned)b[u] >= (unsigned)c.num_blocks) set_error(c, MENTAT_DEV_BAD_BLOCK, b[u]);
            else if (atomicAdd(&c.refcounts[b[u]], run) <= 0) set_error(c, MENTAT_DEV_REF_FREE, b[u]);
        }
        for (int k = 0; k < run; ++k) {
            int32_t* dst = table_row(c, l, children[i + k]) + j0 + lane;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (j0 + 32 * u + lane < nb) dst[32 * u] = b[u];
        }
    }
    for (int k = lane; k < run; k += 32) {
        const int64_t cs = seq_index(c, l, children[i + k]);
        c.nblocks[cs] = nb;
        c.ntok[cs] = ntok;
        c.tail[cs] = tail;
    }
}

// ---------------------------------------------------------------------------
// check and reset: CTA 0 checks the batch, all of them clear `order`
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_pages_begin(mentat_kv_cache c, const int32_t* slots, int n, PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < c.num_blocks; b += (int64_t)gridDim.x * blockDim.x)
        w.order[b] = 0;
    if (blockIdx.x) return;
    const bool ok = slots_distinct(c, slots, n, bits, &s_bad);
    if (threadIdx.x == 0) {
        if (!ok) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
        *w.stop = has_error(c) ? 1 : 0;
    }
}

__global__ void __launch_bounds__(256) k_order_clear(mentat_kv_cache c, PagesWs w) {
    griddep_wait();
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
        nb[k] = k < count ? c.nblocks[seq_index(c, l, slots[i0 + k])] : 0;
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
    const int nb = c.nblocks[seq_index(c, l, slots[i])];
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
    if (lane == 0) w.count[row] = n;
}

// exclusive scan of w.count into base by one CTA; returns the total
__device__ __forceinline__ int scan_rows(const PagesWs& w, int32_t* base, int rows, int* smem32) {
    int carry = 0;
    for (int r0 = 0; r0 < rows; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        int total;
        const int at = block_exclusive_scan(r < rows ? w.count[r] : 0, &total, smem32);
        if (r < rows) base[r] = carry + at;
        carry += total;
    }
    return carry;
}

// the scan, and the FIFO's new tail; base counts from the old tail
__global__ void __launch_bounds__(1024) k_free_scan(mentat_kv_cache c, int rows, PagesWs w) {
    __shared__ int smem32[32];
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    const int total = scan_rows(w, w.base, rows, smem32);
    if (threadIdx.x == 0) c.ctrl[MENTAT_CTRL_TAIL] += total;
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

// push, and the rows' new counters (empty, or what compaction kept: cu); a warp a row
template <bool LEAD>
__global__ void __launch_bounds__(PAGES_THREADS) k_free_push(mentat_kv_cache c, const int32_t* slots, const int32_t* cu,
                                                             int rows, PagesWs w) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, row = blockIdx.x * PAGES_WARPS + (threadIdx.x >> 5);
    if (row >= rows || *w.stop) return;
    const int i = row / c.num_layers, l = row - i * c.num_layers;
    const int64_t si = seq_index(c, l, slots[i]);
    int32_t* t = table_row(c, l, slots[i]);
    if (w.count[row]) {
        const int nb = c.nblocks[si];
        // base counts from the tail before the batch, which the scan has moved past all rows
        long long at = c.ctrl[MENTAT_CTRL_TAIL] - (w.base[rows - 1] + w.count[rows - 1]) + w.base[row];
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
// the same in one cluster: warps take ranges of rows, so a scan over the warps' totals orders the pushes
// ---------------------------------------------------------------------------
constexpr int CLUSTER_CTAS = 8, CLUSTER_THREADS = 512, CLUSTER_WARPS = CLUSTER_THREADS / 32;

// the sum of s_total over the warps of the cluster before this one, and over all of them (a cluster barrier
// between the writes and this call)
__device__ __forceinline__ int before_warp(cg::cluster_group& cluster, int* s_total, int* all) {
    const int lane = threadIdx.x & 31, me = cluster.block_rank() * CLUSTER_WARPS + (threadIdx.x >> 5);
    int before = 0, total = 0;
    for (int w = lane; w < CLUSTER_CTAS * CLUSTER_WARPS; w += 32) {
        const int v = cluster.map_shared_rank(s_total, w / CLUSTER_WARPS)[w % CLUSTER_WARPS];
        total += v;
        before += w < me ? v : 0;
    }
    *all = __reduce_add_sync(0xffffffffu, total);
    return __reduce_add_sync(0xffffffffu, before);
}

template <bool LEAD>
__global__ void __launch_bounds__(CLUSTER_THREADS) k_free_cluster(mentat_kv_cache c, const int32_t* slots, const int32_t* cu,
                                                                  int n, PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad, s_total[CLUSTER_WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster.block_rank();
    bool stop = LEAD ? *w.stop != 0 : !slots_distinct(c, slots, n, bits, &s_bad);
    if (!LEAD && stop && threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
    if (!LEAD) stop = __syncthreads_or(stop || has_error(c));
    // an earlier error, or this one, stops every CTA: nothing of this call is recorded before all have looked
    if (stop) return;
    const int rows = n * c.num_layers, per = (rows + CLUSTER_CTAS * CLUSTER_WARPS - 1) / (CLUSTER_CTAS * CLUSTER_WARPS);
    const int r0 = min(rows, (rank * CLUSTER_WARPS + warp) * per), r1 = min(rows, r0 + per);
    const long long tail0 = c.ctrl[MENTAT_CTRL_TAIL];
    auto each = [&](auto&& f) {  // f(row, entry, block) over the warp's rows, a lane an entry
        for (int row = r0; row < r1; ++row) {
            const int i = row / c.num_layers, l = row - i * c.num_layers;
            const int nb = c.nblocks[seq_index(c, l, slots[i])];
            const int32_t* t = table_row(c, l, slots[i]);
            for (int j0 = LEAD ? w.lead[row] : 0; j0 < nb; j0 += 32) {
                const int j = j0 + lane, b = j < nb ? t[j] : -1;
                f(row, j, (unsigned)b < (unsigned)c.num_blocks ? b : -1, j < nb);
            }
        }
    };
    each([&](int, int, int b, bool) {
        if (b >= 0) w.order[b] = 0;
    });
    cluster.sync();
    each([&](int row, int j, int b, bool have) {
        if (b < 0) {
            if (have) set_error(c, MENTAT_DEV_BAD_BLOCK, table_row(c, row % c.num_layers, slots[row / c.num_layers])[j]);
            return;
        }
        if (atomicSub(&c.refcounts[b], 1) <= 0) {
            atomicAdd(&c.refcounts[b], 1);
            set_error(c, MENTAT_DEV_RELEASE_FREE, b);
            return;
        }
        atomicMax(&w.order[b], release_index(c, row, j));
    });
    cluster.sync();
    auto freed = [&](int row, int j, int b) {
        return b >= 0 && __ldcg(&w.order[b]) == release_index(c, row, j) && __ldcg(&c.refcounts[b]) == 0;
    };
    int mine = 0;
    each([&](int row, int j, int b, bool) { mine += __popc(__ballot_sync(0xffffffffu, freed(row, j, b))); });
    if (lane == 0) s_total[warp] = mine;
    cluster.sync();
    int all;
    long long at = tail0 + before_warp(cluster, s_total, &all);
    each([&](int row, int j, int b, bool) {
        const bool go = freed(row, j, b);
        const uint32_t who = __ballot_sync(0xffffffffu, go);
        if (go) c.free_ring[(at + __popc(who & ((1u << lane) - 1))) % c.num_blocks] = b;
        at += __popc(who);
    });
    __syncwarp();
    for (int row = r0; row < r1; ++row) {
        const int i = row / c.num_layers, l = row - i * c.num_layers;
        const int64_t si = seq_index(c, l, slots[i]);
        if (LEAD)
            install(c, w, row, cu[i + 1] - cu[i], si, table_row(c, l, slots[i]), lane, 32);
        else if (lane == 0)
            c.nblocks[si] = c.ntok[si] = c.tail[si] = 0;
    }
    cluster.sync();  // every CTA has read the old tail and the others' totals
    if (rank == 0 && threadIdx.x == 0) c.ctrl[MENTAT_CTRL_TAIL] = tail0 + all;
}

// ---------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------
struct CompactArgs {
    const int32_t* src;
    const int32_t* dst;  // NULL: in place
    const int32_t* keep;
    int64_t keep_ls;
    const int32_t* cu;
    int n;
};

constexpr int PLAN_CHUNK = 1024;  // kept positions of a warp's step; the last chunk goes on to the end of a list
// The plan, in one cluster, a warp a range of rows: the batch is checked, the kept positions are inside their
// sequences; how many pages at the front stay, and the fresh blocks of the others.  (The lists are a
// thousandth of the bytes that are moved.)
__global__ void __launch_bounds__(CLUSTER_THREADS) k_compact_plan(mentat_kv_cache c, CompactArgs a, int chunks,
                                                                  PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad, s_total[CLUSTER_WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster.block_rank(), L = c.num_layers;
    // every CTA checks the whole batch
    bool ok = slots_distinct(c, a.dst ? a.dst : a.src, a.n, bits, &s_bad);
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
    ok = !__syncthreads_or(no) && ok;
    if (!ok && threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
    bool stop = __syncthreads_or(!ok || has_error(c));
    const int rows = a.n * L, per = (rows + CLUSTER_CTAS * CLUSTER_WARPS - 1) / (CLUSTER_CTAS * CLUSTER_WARPS);
    const int r0 = min(rows, (rank * CLUSTER_WARPS + warp) * per), r1 = min(rows, r0 + per);
    if (!stop)
        for (int row = r0 + lane; row < r1; row += 32) w.count[row] = a.cu[row / L + 1] - a.cu[row / L];
    cluster.sync();  // all have looked at the error word before this call writes it
    // the first position that moves: chunks of the lists over all warps
    if (!stop)
        for (int64_t y = rank * CLUSTER_WARPS + warp; y < (int64_t)rows * chunks; y += CLUSTER_CTAS * CLUSTER_WARPS) {
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
                if (m < 0 || pages > c.max_blocks_per_seq) set_error(c, MENTAT_DEV_TABLE_OVERFLOW, a.src[i]);
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
        *w.stop = stop || short_of;
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
        for (int j = lane; j < count; j += 32) {
            const int b = c.free_ring[(head + first + j) % c.num_blocks];
            w.fresh[first + j] = b;
            c.refcounts[b] = 1;
        }
    }
}

// One CTA per (row, page): the kept tokens of one fresh page, a warp a token.  The cosines and sines of a
// token's shift are computed once for all of its heads, and once for neighbours that moved together; K is
// turned and V copied 16 bytes at a time.  Into new sequences it also writes their tables.  Bound by memory.
constexpr int MOVE_THREADS = 256, MOVE_TOKENS = 16;

// n elements of a row by a warp, four vectors of a lane on the way
template <typename T, int VEC>
__device__ __forceinline__ void copy_row(const T* src, T* dst, int n) {
    using P = Pack<T, VEC>;
    const P* s = reinterpret_cast<const P*>(src);
    P* d = reinterpret_cast<P*>(dst);
    for (int x = threadIdx.x & 31; x < n / VEC; x += 128) {
        P v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (x + 32 * u < n / VEC) v[u] = s[x + 32 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (x + 32 * u < n / VEC) d[x + 32 * u] = v[u];
    }
}
// the tokens' V rows, a warp a token
template <typename T, int VEC>
__device__ __forceinline__ void move_v(T* vp, int64_t dst, const int64_t* from, int count, int n) {
    for (int k = threadIdx.x >> 5; k < count; k += MOVE_THREADS / 32)
        if (from[k] >= 0) copy_row<T, VEC>(vp + from[k], vp + dst + (int64_t)k * n, n);
}
// a token's heads turned by a table (cosines, then sines) by a warp.  Where the 32 lanes cover whole heads, a
// lane has the same pairs in every head and keeps their cosines and sines.
template <typename T, int VEC, bool IL>
__device__ __forceinline__ void turn_row(const T* src, T* dst, int H, int D, const mentat_rotary& r, const float* tab) {
    using P = Pack<T, VEC>;
    const int lane = threadIdx.x & 31, pairs = r.pairs, off = r.offset;
    const int turned = IL ? D / VEC : pairs / VEC, tasks = IL ? turned : turned + (D - 2 * pairs) / VEC;
    const bool whole = 32 % tasks == 0;
    constexpr int N = IL ? VEC / 2 : VEC;
    float co[N], sn[N];
    auto fetch = [&](int t) {
        const int e0 = IL ? (t * VEC - off) / 2 : t * VEC;
        const bool in = IL ? t * VEC >= off && t * VEC < off + 2 * pairs : t < turned;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            co[e] = in ? tab[e0 + e] : 1.f;
            sn[e] = in ? tab[pairs + e0 + e] : 0.f;
        }
    };
    if (whole) fetch(lane % tasks);
    const int total = H * tasks;
    for (int x0 = lane; x0 < total; x0 += 64) {
        P a[2], b[2];
        int d1[2], d2[2];
        bool pair[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int x = x0 + 32 * u;
            if (x >= total) continue;
            const int h = x / tasks, t = x - h * tasks;
            pair[u] = IL || t < turned;
            if (IL) {
                d1[u] = d2[u] = h * D + t * VEC;
            } else if (t < turned) {
                d1[u] = h * D + off + t * VEC;
                d2[u] = d1[u] + pairs;
            } else {  // passed through
                const int d = (t - turned) * VEC;
                d1[u] = d2[u] = h * D + (d >= off ? d + 2 * pairs : d);
            }
            a[u] = *reinterpret_cast<const P*>(src + d1[u]);
            if (!IL && pair[u]) b[u] = *reinterpret_cast<const P*>(src + d2[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int x = x0 + 32 * u;
            if (x >= total) continue;
            if (!whole) fetch(x % tasks);
            if (IL) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float p = Elem<T>::to_f(a[u].v[2 * e]), q = Elem<T>::to_f(a[u].v[2 * e + 1]);
                    a[u].v[2 * e] = Elem<T>::from_f(p * co[e] - q * sn[e]);
                    a[u].v[2 * e + 1] = Elem<T>::from_f(p * sn[e] + q * co[e]);
                }
            } else if (pair[u]) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float p = Elem<T>::to_f(a[u].v[e]), q = Elem<T>::to_f(b[u].v[e]);
                    a[u].v[e] = Elem<T>::from_f(p * co[e] - q * sn[e]);
                    b[u].v[e] = Elem<T>::from_f(p * sn[e] + q * co[e]);
                }
                *reinterpret_cast<P*>(dst + d2[u]) = b[u];
            }
            *reinterpret_cast<P*>(dst + d1[u]) = a[u];
        }
    }
}
template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(MOVE_THREADS, 3) k_compact_move(mentat_kv_cache c, CompactArgs a, mentat_rotary r, PagesWs w) {
    extern __shared__ float cs[];  // [MOVE_TOKENS][2 pairs]
    __shared__ int64_t s_from[MOVE_TOKENS];
    __shared__ int s_shift[MOVE_TOKENS], s_table[MOVE_TOKENS];
    griddep_wait();
    griddep_launch();
    if (*w.stop) return;
    const int tid = threadIdx.x, row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int D = c.head_dim, H = c.num_kv_heads, bs = c.block_size, lead = w.lead[row];
    const int m = a.cu[i + 1] - a.cu[i], pages = (m + bs - 1) / bs;
    const int32_t* keep = a.keep + l * a.keep_ls + a.cu[i];
    const int32_t* t = table_row(c, l, a.src[i]);
    const int32_t* fresh = w.fresh + w.first[row];
    T* kp = reinterpret_cast<T*>(c.k_pool);
    T* vp = reinterpret_cast<T*>(c.v_pool);
    if (a.dst && blockIdx.y == 0) {  // the new sequence: shared pages, fresh ones, counters
        int32_t* to = table_row(c, l, a.dst[i]);
        for (int j = tid; j < lead; j += MOVE_THREADS) {
            const int b = t[j];
            to[j] = b;
            if ((unsigned)b >= (unsigned)c.num_blocks) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            else if (atomicAdd(&c.refcounts[b], 1) <= 0) set_error(c, MENTAT_DEV_REF_FREE, b);
        }
        install(c, w, row, m, seq_index(c, l, a.dst[i]), to, tid, MOVE_THREADS);
    }
    for (int p = lead + blockIdx.y; p < pages; p += gridDim.y) {
        const int64_t to = pool_row(c, l, fresh[p - lead], 0);
        for (int j0 = p * bs; j0 < min(m, (p + 1) * bs); j0 += MOVE_TOKENS) {
            const int count = min(min(m, (p + 1) * bs) - j0, MOVE_TOKENS);
            const int64_t dst = to + (int64_t)(j0 - p * bs) * H * D;
            __syncthreads();
            if (tid < count) {
                const int from = keep[j0 + tid], b = t[from / bs], shift = r.pairs ? j0 + tid - from : 0;
                const bool ok = (unsigned)b < (unsigned)c.num_blocks;
                if (!ok) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
                s_shift[tid] = shift;
                s_from[tid] = ok ? pool_row(c, l, b, from % bs) : -1;
                // tokens that moved together share a table
                s_table[tid] = shift == 0 || (tid && j0 + tid - 1 - keep[j0 + tid - 1] == shift) ? 0 : 1;
            }
            __syncthreads();
            for (int x = tid; x < count * r.pairs; x += MOVE_THREADS) {
                const int k = x / r.pairs, e = x - k * r.pairs;
                if (s_table[k]) rotary_angle(r, e, s_shift[k], cs + k * 2 * r.pairs + e, cs + k * 2 * r.pairs + r.pairs + e);
            }
            if constexpr (VEC > 1) move_v<T, VEC>(vp, dst, s_from, count, H * D);
            __syncthreads();  // the tables
            for (int k = tid >> 5; k < count; k += MOVE_THREADS / 32) {
                if (s_from[k] < 0) continue;
                const T* src = kp + s_from[k];
                T* out = kp + dst + (int64_t)k * H * D;
                int own = k;
                while (s_shift[k] && !s_table[own]) --own;
                const float* tab = cs + own * 2 * r.pairs;
                if constexpr (VEC > 1) {
                    if (s_shift[k]) turn_row<T, VEC, IL>(src, out, H, D, r, tab);
                    else copy_row<T, VEC>(src, out, H * D);
                } else {
                    for (int x = tid & 31; x < H * D; x += 32) {
                        const int d = x % D - r.offset;
                        float v = Elem<T>::to_f(src[x]);
                        if (s_shift[k] && d >= 0 && d < 2 * r.pairs) {
                            const bool low = IL ? !(d & 1) : d < r.pairs;  // first or second of its pair
                            const int e = IL ? d / 2 : low ? d : d - r.pairs, step = IL ? 1 : r.pairs;
                            const float o = Elem<T>::to_f(src[low ? x + step : x - step]);
                            v = low ? v * tab[e] - o * tab[r.pairs + e] : o * tab[r.pairs + e] + v * tab[e];
                        }
                        out[x] = Elem<T>::from_f(v);
                    }
                    for (int x = tid & 31; x < H * D; x += 32) vp[dst + (int64_t)k * H * D + x] = vp[s_from[k] + x];
                }
            }
        }
    }
}

}  // namespace mentat

using namespace mentat;

static bool bad_pages(const mentat_kv_cache* c, int32_t n) {
    return !c || c->num_layers <= 0 || c->num_layers > 65535 || c->num_blocks <= 0 || c->block_size <= 0 ||
           c->max_seqs <= 0 || c->max_blocks_per_seq <= 0 || !c->refcounts || !c->free_ring || !c->ctrl ||
           !c->tables || !c->nblocks || !c->ntok || !c->tail || n < 0 || n > PAGES_MAX_SEQS;
}
static size_t bitmap_bytes(const mentat_kv_cache* c) { return ((size_t)c->max_seqs + 31) / 32 * 4; }
// the bitmap fits in shared memory, and a release's index in 32 bits
static bool pages_fit(const mentat_kv_cache* c, int32_t n) {
    return bitmap_bytes(c) <= 48 * 1024 && (int64_t)n * c->num_layers * c->max_blocks_per_seq < 0xffffffffll;
}
static int chunks_of(int64_t work, int64_t each, int64_t most) {
    const int64_t x = (work + each - 1) / each;
    return (int)(x < 1 ? 1 : x > most ? most : x);
}

// a kernel over one cluster of CLUSTER_CTAS
template <typename... KArgs, typename... Args>
static int launch_one_cluster(void (*kernel)(KArgs...), size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CLUSTER_CTAS);
    cfg.blockDim = dim3(CLUSTER_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CLUSTER_CTAS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...) != cudaSuccess) {
        (void)cudaGetLastError();
        return MENTAT_ERR_CUDA;
    }
    MENTAT_CHECK_LAUNCH();
    return MENTAT_OK;
}

// Releases of up to this many table entries (rows times the longest table) are one cluster's work.
constexpr int64_t FREE_CLUSTER_ENTRIES = 32768;

template <bool LEAD>
static int launch_free(const mentat_kv_cache* c, const int32_t* slots, const int32_t* cu, int32_t n, int32_t max_nb,
                       const PagesWs& w, cudaStream_t s) {
    const int rows = n * c->num_layers;
    if ((int64_t)rows * max_nb <= FREE_CLUSTER_ENTRIES)
        return launch_one_cluster(k_free_cluster<LEAD>, bitmap_bytes(c), s, *c, slots, cu, n, w);
    if (!LEAD)
        MENTAT_LAUNCH(k_pages_begin, dim3(chunks_of(c->num_blocks, 1024, 148)), dim3(256), bitmap_bytes(c), s, *c, slots, n, w);
    else
        MENTAT_LAUNCH(k_order_clear, dim3(chunks_of(c->num_blocks, 1024, 148)), dim3(256), 0, s, *c, w);
    const dim3 marks((n + MARK_SEQS - 1) / MARK_SEQS * c->num_layers, chunks_of(max_nb, 256, 64));
    const dim3 by_row((rows + PAGES_WARPS - 1) / PAGES_WARPS);
    MENTAT_LAUNCH(k_free_mark<LEAD>, marks, dim3(256), 0, s, *c, slots, n, w);
    MENTAT_LAUNCH(k_free_count<LEAD>, by_row, dim3(PAGES_THREADS), 0, s, *c, slots, rows, w);
    MENTAT_LAUNCH(k_free_scan, dim3(1), dim3(1024), 0, s, *c, rows, w);
    MENTAT_LAUNCH(k_free_push<LEAD>, by_row, dim3(PAGES_THREADS), 0, s, *c, slots, cu, rows, w);
    return MENTAT_OK;
}

namespace {
struct LaunchCompactMove {
    const mentat_kv_cache& c;
    const CompactArgs& a;
    const mentat_rotary& r;
    const PagesWs& w;
    int max_keep;
    cudaStream_t s;
    template <typename T, int VEC, bool IL>
    int operator()() {
        const dim3 grid(a.n * c.num_layers, chunks_of(max_keep, c.block_size, 65535));
        const size_t smem = (size_t)MOVE_TOKENS * 2 * r.pairs * sizeof(float);
        if (smem > 40 * 1024 && cudaFuncSetAttribute(k_compact_move<T, VEC, IL>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
            (void)cudaGetLastError();
            return MENTAT_ERR_CUDA;
        }
        MENTAT_LAUNCH(k_compact_move<T, VEC, IL>, grid, dim3(MOVE_THREADS), smem, s, c, a, r, w);
        return MENTAT_OK;
    }
};
}  // namespace

extern "C" {

int64_t mentat_pages_workspace_bytes(const mentat_kv_cache* c, int32_t n) {
    return bad_pages(c, n) ? 0 : pages_ws(c, n, nullptr, nullptr);
}

int mentat_kv_fork_batched(const mentat_kv_cache* c, const int32_t* parents, const int32_t* children, int32_t n,
                           int32_t max_nb, cudaStream_t s) {
    if (bad_pages(c, n) || max_nb < 0 || (n > 0 && (!parents || !children))) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!pages_fit(c, n)) return MENTAT_ERR_UNSUPPORTED;
    (void)max_nb;
    const dim3 grid((n + PAGES_WARPS - 1) / PAGES_WARPS, c->num_layers);
    MENTAT_LAUNCH(k_fork_batched, grid, dim3(PAGES_THREADS), bitmap_bytes(c), s, *c, parents, children, n);
    return MENTAT_OK;
}

int mentat_kv_free_batched(const mentat_kv_cache* c, const int32_t* slots, int32_t n, int32_t max_nb, void* workspace,
                           int64_t workspace_bytes, cudaStream_t s) {
    if (bad_pages(c, n) || max_nb < 0 || (n > 0 && (!slots || !workspace))) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!pages_fit(c, n)) return MENTAT_ERR_UNSUPPORTED;
    PagesWs w;
    if (workspace_bytes < pages_ws(c, n, workspace, &w)) return MENTAT_ERR_ARG;
    return launch_free<false>(c, slots, nullptr, n, max_nb, w, s);
}

int mentat_kv_compact(const mentat_kv_cache* c, const int32_t* src, const int32_t* dst, int32_t n, const int32_t* keep,
                      int64_t keep_ls, const int32_t* cu, int32_t max_keep, int32_t max_nb, const mentat_rotary* r,
                      void* workspace, int64_t workspace_bytes, cudaStream_t s) {
    if (bad_pages(c, n) || max_keep < 0 || max_nb < 0 || keep_ls < 0 || c->head_dim <= 0 || c->num_kv_heads <= 0 ||
        (n > 0 && (!src || !cu || !workspace || !c->k_pool || !c->v_pool || (max_keep > 0 && !keep))) ||
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
    const CompactArgs a{src, dst, keep, keep_ls, cu, n};
    int st = launch_one_cluster(k_compact_plan, bitmap_bytes(c), s, *c, a, chunks_of(max_keep, PLAN_CHUNK, 1 << 20), w);
    if (st == MENTAT_OK)
        st = rotary_dispatch(c->dtype, wide, turn.interleaved != 0, LaunchCompactMove{*c, a, turn, w, max_keep, s});
    return st != MENTAT_OK || dst ? st : launch_free<true>(c, src, cu, n, max_nb, w, s);
}

}  // extern "C"
