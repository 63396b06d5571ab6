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

#include "rotary.cuh"

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
// Every CTA checks the whole batch for itself, so all of them agree whether to go on.
__global__ void __launch_bounds__(256) k_fork_batched(mentat_kv_cache c, const int32_t* parents,
                                                      const int32_t* children, int n) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
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
    const int l = blockIdx.y, i = blockIdx.z, parent = parents[i], child = children[i];
    const int64_t ps = seq_index(c, l, parent), cs = seq_index(c, l, child);
    const int nb = c.nblocks[ps];
    const int32_t* src = table_row(c, l, parent);
    int32_t* dst = table_row(c, l, child);
    for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < nb; j += gridDim.x * blockDim.x) {
        const int b = src[j];
        dst[j] = b;
        if ((unsigned)b >= (unsigned)c.num_blocks) {
            set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            continue;
        }
        if (atomicAdd(&c.refcounts[b], 1) <= 0) set_error(c, MENTAT_DEV_REF_FREE, b);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        c.nblocks[cs] = nb;
        c.ntok[cs] = c.ntok[ps];
        c.tail[cs] = c.tail[ps];
    }
}

// ---------------------------------------------------------------------------
// check and reset: CTA 0 checks the batch, all of them clear `order`
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_pages_begin(mentat_kv_cache c, const int32_t* slots, const int32_t* dst,
                                                     int n, PagesWs w) {
    extern __shared__ uint32_t bits[];
    __shared__ int s_bad;
    griddep_wait();
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < c.num_blocks; b += (int64_t)gridDim.x * blockDim.x)
        w.order[b] = 0;
    if (blockIdx.x) return;
    bool ok;
    if (!dst) {
        ok = slots_distinct(c, slots, n, bits, &s_bad);
    } else {  // sources in range; destinations distinct and empty in every layer (so none is a source with tokens)
        ok = slots_distinct(c, dst, n, bits, &s_bad);
        int no = 0;
        if (ok)
            for (int64_t x = threadIdx.x; x < (int64_t)n * c.num_layers; x += blockDim.x) {
                const int i = (int)(x / c.num_layers), l = (int)(x % c.num_layers);
                if (slots[i] < 0 || slots[i] >= c.max_seqs || has_bit(bits, slots[i])) {
                    no = 1;
                    s_bad = slots[i];
                } else if (c.nblocks[seq_index(c, l, dst[i])] || c.ntok[seq_index(c, l, dst[i])]) {
                    no = 1;
                    s_bad = dst[i];
                }
            }
        ok = !__syncthreads_or(no) && ok;
    }
    if (threadIdx.x == 0) {
        if (!ok) set_error(c, MENTAT_DEV_BAD_SLOT, s_bad);
        *w.stop = has_error(c) ? 1 : 0;
    }
}

// ---------------------------------------------------------------------------
// free: rows are (sequence i, layer l), row index i * layers + l
// ---------------------------------------------------------------------------
// the order of a release: its row, then its table entry; 0 is "none"
__device__ __forceinline__ uint32_t release_index(const mentat_kv_cache& c, int row, int j) {
    return (uint32_t)row * (uint32_t)c.max_blocks_per_seq + (uint32_t)j + 1u;
}

template <bool LEAD>
__global__ void __launch_bounds__(256) k_free_mark(mentat_kv_cache c, const int32_t* slots, PagesWs w) {
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int nb = c.nblocks[seq_index(c, l, slots[i])];
    const int32_t* t = table_row(c, l, slots[i]);
    for (int j = (LEAD ? w.lead[row] : 0) + blockIdx.y * blockDim.x + threadIdx.x; j < nb; j += gridDim.y * blockDim.x) {
        const int b = t[j];
        if ((unsigned)b >= (unsigned)c.num_blocks) {
            set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            continue;
        }
        if (atomicSub(&c.refcounts[b], 1) <= 0) {
            atomicAdd(&c.refcounts[b], 1);
            set_error(c, MENTAT_DEV_RELEASE_FREE, b);
            continue;
        }
        atomicMax(&w.order[b], release_index(c, row, j));
    }
}

// whether entry j of a row frees its block
__device__ __forceinline__ bool frees(const mentat_kv_cache& c, const PagesWs& w, const int32_t* t, int row, int j) {
    const int b = t[j];
    return (unsigned)b < (unsigned)c.num_blocks && w.order[b] == release_index(c, row, j) && c.refcounts[b] == 0;
}

template <bool LEAD>
__global__ void __launch_bounds__(128) k_free_count(mentat_kv_cache c, const int32_t* slots, PagesWs w) {
    __shared__ int s_sum[4];
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int nb = c.nblocks[seq_index(c, l, slots[i])];
    const int32_t* t = table_row(c, l, slots[i]);
    int n = 0;
    for (int j = (LEAD ? w.lead[row] : 0) + threadIdx.x; j < nb; j += blockDim.x) n += frees(c, w, t, row, j);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x == 0) w.count[row] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
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
    if (*w.stop) return;
    const int total = scan_rows(w, w.base, rows, smem32);
    if (threadIdx.x == 0) c.ctrl[MENTAT_CTRL_TAIL] += total;
}

// push, and the rows' new counters (empty, or what compaction kept)
template <bool LEAD>
__global__ void __launch_bounds__(128) k_free_push(mentat_kv_cache c, const int32_t* slots, int rows, PagesWs w) {
    __shared__ int smem32[32];
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int64_t si = seq_index(c, l, slots[i]);
    const int nb = c.nblocks[si];
    const int32_t* t = table_row(c, l, slots[i]);
    // base counts from the tail before the batch, which the scan has moved past all rows
    const long long tail0 = c.ctrl[MENTAT_CTRL_TAIL] - (w.base[rows - 1] + w.count[rows - 1]);
    long long at = tail0 + w.base[row];
    for (int j0 = LEAD ? w.lead[row] : 0; j0 < nb; j0 += blockDim.x) {
        const int j = j0 + threadIdx.x;
        const bool go = j < nb && frees(c, w, t, row, j);
        int total;
        const int pos = block_exclusive_scan(go, &total, smem32);
        if (go) c.free_ring[(at + pos) % c.num_blocks] = t[j];
        at += total;
    }
    if (!LEAD && threadIdx.x == 0) c.nblocks[si] = c.ntok[si] = c.tail[si] = 0;
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

// one CTA per row: the kept positions are inside the sequence; how many pages at the
// front stay; the demand for fresh blocks
__global__ void __launch_bounds__(256) k_compact_scan(mentat_kv_cache c, CompactArgs a, PagesWs w) {
    __shared__ int s_first;
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int m = a.cu[i + 1] - a.cu[i], len = c.ntok[seq_index(c, l, a.src[i])];
    const int32_t* keep = a.keep + l * a.keep_ls + a.cu[i];
    if (threadIdx.x == 0) s_first = m;
    __syncthreads();
    int first = m;
    for (int j = threadIdx.x; j < m; j += blockDim.x) {
        const int t = keep[j];
        if (t < 0 || t >= len) set_error(c, MENTAT_DEV_BAD_TOKEN, t);
        if (t != j && j < first) first = j;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if ((threadIdx.x & 31) == 0) atomicMin(&s_first, first);
    __syncthreads();
    if (threadIdx.x == 0) {
        const int pages = (m + c.block_size - 1) / c.block_size;
        // a page kept in part is copied even if its tokens stay in place: sequences whose tail is one
        // block have tails of one length (the batched append relies on it)
        const int lead = s_first == m && m == len ? pages : s_first / c.block_size;
        if (pages > c.max_blocks_per_seq || m < 0) set_error(c, MENTAT_DEV_TABLE_OVERFLOW, a.src[i]);
        w.lead[row] = lead;
        w.count[row] = pages - lead;
    }
}

__global__ void __launch_bounds__(1024) k_compact_alloc(mentat_kv_cache c, int rows, PagesWs w) {
    __shared__ int smem32[32];
    griddep_wait();
    if (*w.stop) return;
    if (has_error(c)) {  // a bad position
        __syncthreads();
        if (threadIdx.x == 0) *w.stop = 1;
        return;
    }
    const int total = scan_rows(w, w.first, rows, smem32);
    const long long head = c.ctrl[MENTAT_CTRL_HEAD], avail = c.ctrl[MENTAT_CTRL_TAIL] - head;
    __syncthreads();
    if (total > avail) {
        if (threadIdx.x == 0) {
            set_error(c, MENTAT_DEV_OUT_OF_BLOCKS, c.num_blocks);
            *w.stop = 1;
        }
        return;
    }
    for (int k = threadIdx.x; k < total; k += blockDim.x) {
        const int b = c.free_ring[(head + k) % c.num_blocks];
        w.fresh[k] = b;
        c.refcounts[b] = 1;
    }
    if (threadIdx.x == 0) {
        c.ctrl[MENTAT_CTRL_HEAD] = head + total;
        const long long used = c.num_blocks - (avail - total);
        if (used > c.ctrl[MENTAT_CTRL_PEAK]) c.ctrl[MENTAT_CTRL_PEAK] = used;
        c.ctrl[MENTAT_CTRL_ALLOCS] += total;
    }
}

// one CTA per (row, page): the kept tokens of one fresh page
template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(256) k_compact_move(mentat_kv_cache c, CompactArgs a, mentat_rotary r, PagesWs w) {
    extern __shared__ float cs[];
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int D = c.head_dim, H = c.num_kv_heads, bs = c.block_size;
    const int m = a.cu[i + 1] - a.cu[i], pages = (m + bs - 1) / bs;
    const int32_t* keep = a.keep + l * a.keep_ls + a.cu[i];
    const int32_t* t = table_row(c, l, a.src[i]);
    T* kp = reinterpret_cast<T*>(c.k_pool);
    T* vp = reinterpret_cast<T*>(c.v_pool);
    for (int p = w.lead[row] + blockIdx.y; p < pages; p += gridDim.y) {
        const int to = w.fresh[w.first[row] + p - w.lead[row]];
        for (int j = p * bs; j < min(m, (p + 1) * bs); ++j) {
            const int from = keep[j], b = t[from / bs];
            if ((unsigned)b >= (unsigned)c.num_blocks) {
                if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
                continue;
            }
            const int64_t s = pool_row(c, l, b, from % bs), d = pool_row(c, l, to, j % bs);
            if (r.pairs && from != j) {
                __syncthreads();
                rotary_table(r, j - from, cs);
                __syncthreads();
                rotate_heads<T, VEC, IL>(kp + s, D, kp + d, D, H, D, r, cs);
            } else {
                copy_heads<T, VEC>(kp + s, D, kp + d, D, H, D);
            }
            copy_heads<T, VEC>(vp + s, D, vp + d, D, H, D);
        }
    }
}

// the rows' new tables and counters; new sequences take references on shared pages
__global__ void __launch_bounds__(256) k_compact_install(mentat_kv_cache c, CompactArgs a, PagesWs w) {
    griddep_wait();
    if (*w.stop) return;
    const int row = blockIdx.x, i = row / c.num_layers, l = row - i * c.num_layers;
    const int m = a.cu[i + 1] - a.cu[i], pages = (m + c.block_size - 1) / c.block_size, lead = w.lead[row];
    const int slot = a.dst ? a.dst[i] : a.src[i];
    int32_t* t = table_row(c, l, slot);
    const int32_t* fresh = w.fresh + w.first[row];
    if (a.dst) {
        const int32_t* s = table_row(c, l, a.src[i]);
        for (int j = threadIdx.x; j < lead; j += blockDim.x) {
            const int b = s[j];
            t[j] = b;
            if ((unsigned)b >= (unsigned)c.num_blocks) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            else if (atomicAdd(&c.refcounts[b], 1) <= 0) set_error(c, MENTAT_DEV_REF_FREE, b);
        }
    }
    for (int j = lead + threadIdx.x; j < pages; j += blockDim.x) t[j] = fresh[j - lead];
    if (threadIdx.x == 0) {
        const int64_t si = seq_index(c, l, slot);
        c.nblocks[si] = pages;
        c.ntok[si] = m;
        c.tail[si] = m - (pages - 1) * c.block_size - (m ? 0 : c.block_size);
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

template <bool LEAD>
static int launch_free(const mentat_kv_cache* c, const int32_t* slots, int32_t n, int32_t max_nb, const PagesWs& w,
                       cudaStream_t s) {
    const int rows = n * c->num_layers;
    MENTAT_LAUNCH(k_free_mark<LEAD>, dim3(rows, chunks_of(max_nb, 256, 64)), dim3(256), 0, s, *c, slots, w);
    MENTAT_LAUNCH(k_free_count<LEAD>, dim3(rows), dim3(128), 0, s, *c, slots, w);
    MENTAT_LAUNCH(k_free_scan, dim3(1), dim3(1024), 0, s, *c, rows, w);
    MENTAT_LAUNCH(k_free_push<LEAD>, dim3(rows), dim3(128), 0, s, *c, slots, rows, w);
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
        MENTAT_LAUNCH(k_compact_move<T, VEC, IL>, grid, dim3(256), 2 * r.pairs * sizeof(float), s, c, a, r, w);
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
    const dim3 grid(chunks_of(max_nb, 256, 64), c->num_layers, n);
    MENTAT_LAUNCH(k_fork_batched, grid, dim3(256), bitmap_bytes(c), s, *c, parents, children, n);
    return MENTAT_OK;
}

int mentat_kv_free_batched(const mentat_kv_cache* c, const int32_t* slots, int32_t n, int32_t max_nb, void* workspace,
                           int64_t workspace_bytes, cudaStream_t s) {
    if (bad_pages(c, n) || max_nb < 0 || (n > 0 && (!slots || !workspace))) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!pages_fit(c, n)) return MENTAT_ERR_UNSUPPORTED;
    PagesWs w;
    if (workspace_bytes < pages_ws(c, n, workspace, &w)) return MENTAT_ERR_ARG;
    MENTAT_LAUNCH(k_pages_begin, dim3(chunks_of(c->num_blocks, 1024, 148)), dim3(256), bitmap_bytes(c), s, *c, slots,
                  (const int32_t*)nullptr, n, w);
    return launch_free<false>(c, slots, n, max_nb, w, s);
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
    const int rows = n * c->num_layers, vec = 16 / dtype_bytes(c->dtype);
    mentat_rotary turn{};
    if (r) {
        turn = *r;
        turn.scale = 1.0f;
    }
    const bool wide = c->head_dim % vec == 0 && (!r || rotary_aligned(r, c->head_dim, vec)) &&
                      ((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) % 16 == 0;
    const CompactArgs a{src, dst, keep, keep_ls, cu, n};
    MENTAT_LAUNCH(k_pages_begin, dim3(chunks_of(c->num_blocks, 1024, 148)), dim3(256), bitmap_bytes(c), s, *c, src, dst,
                  n, w);
    MENTAT_LAUNCH(k_compact_scan, dim3(rows), dim3(256), 0, s, *c, a, w);
    MENTAT_LAUNCH(k_compact_alloc, dim3(1), dim3(1024), 0, s, *c, rows, w);
    if (max_keep > 0) {
        const int st = rotary_dispatch(c->dtype, wide, turn.interleaved != 0,
                                       LaunchCompactMove{*c, a, turn, w, max_keep, s});
        if (st != MENTAT_OK) return st;
    }
    if (!dst) {
        const int st = launch_free<true>(c, src, n, max_nb, w, s);
        if (st != MENTAT_OK) return st;
    }
    MENTAT_LAUNCH(k_compact_install, dim3(rows), dim3(256), 0, s, *c, a, w);
    return MENTAT_OK;
}

}  // extern "C"
