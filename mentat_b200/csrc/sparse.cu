// Sparse decode: a page index (bounds of every page's keys in 8 bits), the choice of
// pages by a score from it, and attention over the chosen pages.
//
// Index.  Per (block, KV head): lowest and highest key of every channel over the
// page's rows, in units of one power of two per (block, head), the lowest rounded
// down and the highest up, so the true keys lie between.  The unit is exact and so
// is every division by it: the index is the same whatever computes it.
//
// Score.  With q rounded to 8 bits (one power of two per query head), the largest
// product that a key between the bounds can have with it is
//   2^(eq + ek) * sum_d max(q8_d lo8_d, q8_d hi8_d)
//     = 2^(eq + ek) * (sum_d min(q8_d, 0) lo8_d + max(q8_d, 0) hi8_d),
// one dot product of 2 head_dim bytes, on the byte MMA (int32 sums, below 2 * 128 * 127^2 <
// 2^23, exact as a float).  A KV head takes the highest of its query heads' scores.
// Choosing by an exact number makes the choice reproducible.
//
// Attention.  Base-2 online softmax over the chosen pages, partials of the warps and of
// the cluster's CTAs merged in shared memory.

#include <cooperative_groups.h>

#include <type_traits>

#include "tma.cuh"

namespace cg = cooperative_groups;

namespace mentat {

// ---------------------------------------------------------------------------
// index
// ---------------------------------------------------------------------------
constexpr int EXP_MIN = -50, EXP_MAX = 50, EXP_ALL = 127;
constexpr int EXP_UNREADABLE = -128;  // in no index: the table's entry is outside the pool

// the least e with top <= 127 * 2^e, within EXP_MIN .. EXP_MAX; top finite, >= 0
__device__ __forceinline__ int unit_exponent(float top) {
    if (top == 0.f) return EXP_MIN;
    int x;
    const float m = frexpf(top, &x);  // top = m 2^x, 0.5 <= m < 1
    const int e = x - 7 + (m > 127.f / 128.f);
    return min(max(e, EXP_MIN), EXP_MAX);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// A bound in units of 1 / inv, rounded outwards.  The product is exact but for keys below 2^-99 beside one above 127,
// where it can underflow: a bound that is not zero keeps its side.
__device__ __forceinline__ int8_t bound_low(float v, float inv) {
    return (int8_t)fminf(fmaxf(floorf(v * inv), -127.f), v < 0.f ? -1.f : 127.f);
}
__device__ __forceinline__ int8_t bound_high(float v, float inv) {
    return (int8_t)fmaxf(fminf(ceilf(v * inv), 127.f), v > 0.f ? 1.f : -127.f);
}

// One CTA of head_dim threads per (block, KV head).
template <typename T>
__device__ __forceinline__ void index_page(const mentat_kv_cache& c, int layer, int b, int h, const mentat_page_index& x) {
    __shared__ float s_top[32];
    __shared__ int s_bad;
    const int D = c.head_dim, d = threadIdx.x;
    if (d == 0) s_bad = 0;
    __syncthreads();
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
    if (d < D) {
        const T* k = reinterpret_cast<const T*>(c.k_pool) + pool_row(c, layer, b, 0) + (int64_t)h * D + d;
        for (int t = 0; t < c.block_size; ++t) {
            const float v = Elem<T>::to_f(k[(int64_t)t * c.num_kv_heads * D]);
            bad |= !isfinite(v);
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
        }
    }
    float top = d < D && !bad ? fmaxf(fabsf(lo), fabsf(hi)) : 0.f;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((d & 31) == 0) s_top[d >> 5] = top;
    if (bad) s_bad = 1;
    __syncthreads();
    top = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) top = fmaxf(top, s_top[w]);
    bad = s_bad;
    const int e = unit_exponent(top);
    const float inv = pow2(-e);
    const int64_t at = ((int64_t)layer * c.num_blocks + b) * c.num_kv_heads + h;
    if (d < D) {
        int8_t* o = x.bounds + at * 2 * D + d;
        o[0] = bad ? (int8_t)0 : bound_low(lo, inv);
        o[D] = bad ? (int8_t)0 : bound_high(hi, inv);
    }
    if (d == 0) x.exps[at] = (int8_t)(bad ? EXP_ALL : e);
    __syncthreads();
}

// min and max that keep a NaN, packed where the type is 16 bits
template <typename T> struct Extreme;
template <> struct Extreme<float> {
    static constexpr int N = 1;
    using V = float;
    __device__ __forceinline__ static V lo(V a, V b) {
        V d;
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
        return d;
    }
    __device__ __forceinline__ static V hi(V a, V b) {
        V d;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
        return d;
    }
    __device__ __forceinline__ static float get(V a, int) { return a; }
};
template <> struct Extreme<__nv_bfloat16> {
    static constexpr int N = 2;
    using V = __nv_bfloat162;
    __device__ __forceinline__ static V lo(V a, V b) { return __hmin2_nan(a, b); }
    __device__ __forceinline__ static V hi(V a, V b) { return __hmax2_nan(a, b); }
    __device__ __forceinline__ static float get(V a, int i) { return __bfloat162float(i ? a.y : a.x); }
};
template <> struct Extreme<__half> {
    static constexpr int N = 2;
    using V = __half2;
    __device__ __forceinline__ static V lo(V a, V b) { return __hmin2_nan(a, b); }
    __device__ __forceinline__ static V hi(V a, V b) { return __hmax2_nan(a, b); }
    __device__ __forceinline__ static float get(V a, int i) { return __half2float(i ? a.y : a.x); }
};

// The index of all heads of one block by one CTA, 16 bytes of a row to a thread (head_dim / VEC threads to a
// head, a power of two within a warp, every thread of which takes part); the page is read once, 8 rows asked
// for at a time, of which the 32 registers that the compiler takes hold about half.  Bound by memory: 8,192 pages of 16 x
// 8 heads of 128 (285 MB) in 50 us alone with cold caches, 5.7 TB/s; among other calls 55 (15 rows at a time 58; a ring of
// bulk copies in one CTA on an SM 61).
template <typename T>
__device__ __forceinline__ void index_block(const mentat_kv_cache& c, int layer, int b, const mentat_page_index& x) {
    using E = Extreme<T>;
    constexpr int VEC = 16 / sizeof(T), W = VEC / E::N;
    using Row = Pack<typename E::V, W>;
    const int D = c.head_dim, H = c.num_kv_heads, per = D / VEC, n = H * per, bs = c.block_size;
    const Row* k = reinterpret_cast<const Row*>(reinterpret_cast<const T*>(c.k_pool) + pool_row(c, layer, b, 0));
    for (int u0 = 0; u0 < n; u0 += blockDim.x) {
        const int u = u0 + threadIdx.x, at = min(u, n - 1);
        Row lo = k[at], hi = lo;
        for (int r = 1; r < bs; r += 8) {
            Row v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k[(int64_t)min(r + e, bs - 1) * n + at];
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    lo.v[w] = E::lo(lo.v[w], v[e].v[w]);
                    hi.v[w] = E::hi(hi.v[w], v[e].v[w]);
                }
        }
        float top = 0.f;
        bool bad = false;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int e = 0; e < E::N; ++e) {
                const float l = E::get(lo.v[w], e), g = E::get(hi.v[w], e);
                bad |= !isfinite(l) || !isfinite(g);
                top = fmaxf(top, fmaxf(fabsf(l), fabsf(g)));
            }
        if (bad) top = INFINITY;
        for (int o = 1; o < per; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bad = isinf(top);
        const int e = bad ? 0 : unit_exponent(top);
        const float inv = pow2(-e);
        Pack<int8_t, VEC> ol, oh;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int i = 0; i < E::N; ++i) {
                const float l = E::get(lo.v[w], i), g = E::get(hi.v[w], i);
                ol.v[w * E::N + i] = bad ? (int8_t)0 : bound_low(l, inv);
                oh.v[w * E::N + i] = bad ? (int8_t)0 : bound_high(g, inv);
            }
        if (u < n) {
            const int h = u / per, d = (u - h * per) * VEC;
            const int64_t to = ((int64_t)layer * c.num_blocks + b) * H + h;
            int8_t* o = x.bounds + to * 2 * D + d;
            *reinterpret_cast<Pack<int8_t, VEC>*>(o) = ol;
            *reinterpret_cast<Pack<int8_t, VEC>*>(o + D) = oh;
            if (d == 0) x.exps[to] = (int8_t)(bad ? EXP_ALL : e);
        }
    }
}
// threads of a CTA that index_block can use, 0 if the head does not divide into them
static int index_block_threads(const mentat_kv_cache* c) {
    const int vec = 16 / dtype_bytes(c->dtype), per = c->head_dim / vec;
    if (c->head_dim % vec || per > 32 || (per & (per - 1)) || (uintptr_t)c->k_pool % 16) return 0;
    const int n = (c->num_kv_heads * per + 31) / 32 * 32;
    return n < 256 ? n : 256;
}

// One CTA per block (WIDE), or per block and head.
template <typename T, bool WIDE>
__global__ void k_index_blocks(mentat_kv_cache c, int layer, const int32_t* blocks, mentat_page_index x) {
    griddep_wait();
    griddep_launch();
    const int b = blocks[blockIdx.x];
    if ((unsigned)b >= (unsigned)c.num_blocks) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        return;
    }
    if constexpr (WIDE) index_block<T>(c, layer, b, x);
    else index_page<T>(c, layer, b, blockIdx.y, x);
}

template <typename T, bool WIDE>
__global__ void k_index_seqs(mentat_kv_cache c, int layer0, const int32_t* slots, int n, int first, mentat_page_index x,
                             int max_pages) {
    griddep_wait();
    griddep_launch();
    const int i = blockIdx.x / max_pages, slot = slots[i];
    if (slot < 0 || slot >= c.max_seqs) {
        if (threadIdx.x == 0 && slot != -1) set_error(c, MENTAT_DEV_BAD_SLOT, slot);
        return;
    }
    const int layer = layer0 + blockIdx.z, len = c.ntok[seq_index(c, layer, slot)];
    const int full = min(len / c.block_size, c.max_blocks_per_seq);
    int p = first + blockIdx.x % max_pages;
    if (first < 0) {
        // the page that ends with entry i's token: a sequence that occurs again behind i got later ones too
        int later = 0;
        for (int j = i + 1 + (threadIdx.x & 31); j < n; j += 32) later += slots[j] == slot;
        const int mine = len - __reduce_add_sync(0xffffffffu, later);
        if (mine <= 0 || mine % c.block_size) return;
        p = mine / c.block_size - 1;
    }
    if (p >= full) return;
    const int b = table_row(c, layer, slot)[p];
    if ((unsigned)b >= (unsigned)c.num_blocks) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        return;
    }
    if constexpr (WIDE) index_block<T>(c, layer, b, x);
    else index_page<T>(c, layer, b, blockIdx.y, x);
}

// Four pages to a CTA, each thread one piece of each of them on the way.  Bound by the stores: 8,192 pages of 8 heads
// of 128 (84 MB) take 20 us alone with cold caches; with stores that stay in L2 the index and this take 80 us, not 74.
constexpr int BOUNDS_PAGES = 4;
__global__ void __launch_bounds__(256) k_page_bounds(mentat_kv_cache c, int layer, const int32_t* blocks, int n,
                                                     mentat_page_index x, float* low, float* high, int8_t* exps) {
    griddep_wait();
    griddep_launch();
    const int D = c.head_dim, H = c.num_kv_heads, i0 = blockIdx.x * BOUNDS_PAGES;
    int64_t at[BOUNDS_PAGES];  // of the page's first head; -1: none
#pragma unroll
    for (int k = 0; k < BOUNDS_PAGES; ++k) {
        const int b = i0 + k < n ? blocks[i0 + k] : -1;
        at[k] = (unsigned)b < (unsigned)c.num_blocks ? ((int64_t)layer * c.num_blocks + b) * H : -1;
        if (i0 + k < n && at[k] < 0 && threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
    }
    auto value = [&](int v, int e) { return v * pow2(e); };
    const int64_t to = (int64_t)i0 * H;
    if (D % 4 == 0 && (((uintptr_t)low | (uintptr_t)high) & 15) == 0 && ((uintptr_t)x.bounds & 3) == 0) {
        for (int u = threadIdx.x; u < H * D / 2; u += blockDim.x) {  // 4 bytes to 16
            const int h = u / (D / 2), r = u - h * (D / 2);
            const bool top = r >= D / 4;
            const int d = (top ? r - D / 4 : r) * 4;
            char4 v[BOUNDS_PAGES];
            int e[BOUNDS_PAGES];
#pragma unroll
            for (int k = 0; k < BOUNDS_PAGES; ++k)
                if (at[k] >= 0) {
                    v[k] = *reinterpret_cast<const char4*>(x.bounds + (at[k] + h) * 2 * D + (top ? D : 0) + d);
                    e[k] = x.exps[at[k] + h];
                }
            const float inf = top ? INFINITY : -INFINITY;
#pragma unroll
            for (int k = 0; k < BOUNDS_PAGES; ++k)
                if (at[k] >= 0)
                    __stcs(reinterpret_cast<float4*>((top ? high : low) + (to + (int64_t)k * H + h) * D + d),
                           e[k] == EXP_ALL ? make_float4(inf, inf, inf, inf)
                                           : make_float4(value(v[k].x, e[k]), value(v[k].y, e[k]), value(v[k].z, e[k]),
                                                         value(v[k].w, e[k])));
        }
    } else {
        for (int u = threadIdx.x; u < BOUNDS_PAGES * H * D; u += blockDim.x) {
            const int k = u / (H * D), h = u / D % H, d = u % D;
            if (at[k] < 0) continue;
            const int e = x.exps[at[k] + h];
            const int8_t* b = x.bounds + (at[k] + h) * 2 * D + d;
            low[(to + (int64_t)k * H + h) * D + d] = e == EXP_ALL ? -INFINITY : value(b[0], e);
            high[(to + (int64_t)k * H + h) * D + d] = e == EXP_ALL ? INFINITY : value(b[D], e);
        }
    }
    for (int u = threadIdx.x; u < BOUNDS_PAGES * H; u += blockDim.x)
        if (at[u / H] >= 0) exps[to + u] = x.exps[at[u / H] + u % H];
}

// ---------------------------------------------------------------------------
// decode: one cluster per (sequence, KV head)
// ---------------------------------------------------------------------------
// The cluster's CTAs score a slice of the pages each and write the keys to all of their
// shared memories; each then makes the whole choice for itself, attends to an equal share
// of the chosen pages, and they merge their partials: one launch, and no workspace.  Bound by latency: one sequence of
// 4,000 tokens takes 10 us, 16 alone with cold caches (slots, lengths, table, bounds, the choice and the pages wait for
// one another).
// warps of a CTA: with the tensor-core path's rings two CTAs of four fit on an SM; the other path is bound by
// latency and takes eight
__host__ __device__ constexpr int sparse_warps(bool mma) { return mma ? 4 : 8; }
// groups of 16 tokens that a warp holds or has on the way: as many as leave room for two CTAs on an SM (96 KB)
constexpr int SPARSE_STAGES = 3;
constexpr int SPARSE_MAX_BUDGET = 8192, SPARSE_MAX_GROUP = 16, SPARSE_MAX_CLUSTER = 16;

struct SparseArgs {
    const int32_t* slots;
    const void* q;
    int64_t qs;
    void* out;
    int64_t os;
    int32_t* pages;
    float scale;  // times log2(e)
    int layer, G, max_len, budget, sink, recent;
    int held, share;  // most pages of a sequence, most chosen pages of a CTA's share
    // with launches before the attention: keys [n][kv heads][key_stride], chosen pages [n][kv heads][budget],
    // the queries in 8 bits (k_score_queries)
    uint32_t* keys;
    int32_t* list;
    int8_t* q8;
    float* units;
    int64_t key_stride;
    int n;
};

// shared memory, in ints (from a 1024-byte boundary): first the rings of attend_mma, whose place the
// partials o [warps][G][D] take later and which the choice has before: q bytes [GM, at least 8][2][D]
// (negative part, positive part), the keys; or, without tensor cores, the partials and the queries as
// floats [G][D]; then m, l [warps][GM], and the pages of the share and their blocks
struct SparseSmem {
    int po, q8, keys, qf, ml, pages, blocks, total;
};
__host__ __device__ inline SparseSmem sparse_smem(int G, int GM, int D, bool mma, bool listed, int pages,
                                                  int share) {
    SparseSmem s;
    share = (share + 3) / 4 * 4;
    const int warps = sparse_warps(mma), attend = mma ? warps * SPARSE_STAGES * 16 * D : 0, partials = warps * G * D;
    s.po = s.q8 = 0;
    s.keys = (GM < 8 ? 8 : GM) * 2 * D / 4;
    const int chose = listed ? 0 : s.keys + (pages + 3 + 3) / 4 * 4;
    s.qf = attend > partials ? attend : partials;
    if (chose > s.qf) s.qf = chose;
    s.ml = s.qf + (mma ? 0 : G * D);
    s.pages = s.ml + 2 * warps * GM;
    s.blocks = s.pages + share;
    s.total = s.blocks + share;
    return s;
}

__device__ __forceinline__ uint32_t ordered(float f) {  // order of floats as order of integers
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// D (16 x 8 float) += A (16 x 16) * B (16 x 8)
template <typename T>
__device__ __forceinline__ void mma_16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16<__nv_bfloat16>(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                      uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16<__half>(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A query head in 8 bits: its negative part to q8, its positive part D bytes on; a warp.
template <typename T, int D>
__device__ __forceinline__ void quantise(const T* q, bool real, int8_t* q8, float* unit) {
    const int lane = threadIdx.x & 31;
    float v[D / 32], top = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        v[j] = real ? Elem<T>::to_f(q[j * 32 + lane]) : 0.f;
        if (!isfinite(v[j])) v[j] = 0.f;
        top = fmaxf(top, fabsf(v[j]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = unit_exponent(top);
    if (lane == 0) *unit = pow2(e);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const int w = (int)fminf(fmaxf(rintf(v[j] * pow2(-e)), -127.f), 127.f);
        q8[j * 32 + lane] = (int8_t)min(w, 0);
        q8[D + j * 32 + lane] = (int8_t)max(w, 0);
    }
}

// D (16 x 8 int32) += A (16 x 32 bytes) * B (32 x 8 bytes)
__device__ __forceinline__ void mma_s8(int* d, int a0, int a1, int a2, int a3, int b0, int b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// keys[p] of the pages p0 .. p1, to every CTA of the cluster.  A warp takes 16 pages at a time as
// the rows of a product, 8 query heads (16 for GM 16) as its columns; the order of the
// channels within the product is the one that lets a lane load 16 contiguous bytes of its page.
template <int D, int GM, int WARPS>
__device__ __forceinline__ void score_pages(const mentat_kv_cache& c, const mentat_page_index& x, const SparseArgs& a,
                                            int h, const int32_t* row, int P, int p0, int p1, const int8_t* q8,
                                            const float* unit, uint32_t* keys) {
    constexpr int NT = GM > 8 ? 2 : 1, CH = 2 * D / 64;  // columns / 8, 64-byte chunks of a page's bounds
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, H = c.num_kv_heads;
    const int64_t base = (int64_t)a.layer * c.num_blocks;
    int4 b[NT][CH];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            b[nt][ch] = *reinterpret_cast<const int4*>(q8 + (nt * 8 + g) * 2 * D + ch * 64 + t * 16);
    float u[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        u[nt][0] = unit[nt * 8 + 2 * t];
        u[nt][1] = unit[nt * 8 + 2 * t + 1];
    }
    for (int p = p0 + warp * 16; p < p1; p += WARPS * 16) {
        int4 v[2][CH];
        int ek[2];
        bool ok[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int pp = p + r * 8 + g;
            const int id = pp < p1 ? row[pp] : 0;
            ok[r] = (unsigned)id < (unsigned)c.num_blocks;
            if (!ok[r] && t == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, id);
            const int64_t at = (base + (ok[r] ? id : 0)) * H + h;
            ek[r] = x.exps[at];
            const int4* src = reinterpret_cast<const int4*>(x.bounds + at * 2 * D) + t;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) v[r][ch] = src[ch * 4];
        }
        int d[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            d[nt][0] = d[nt][1] = d[nt][2] = d[nt][3] = 0;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                mma_s8(d[nt], v[0][ch].x, v[1][ch].x, v[0][ch].y, v[1][ch].y, b[nt][ch].x, b[nt][ch].y);
                mma_s8(d[nt], v[0][ch].z, v[1][ch].z, v[0][ch].w, v[1][ch].w, b[nt][ch].z, b[nt][ch].w);
            }
        }
        float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (nt * 8 + 2 * t + (i & 1) < a.G) best[i >> 1] = fmaxf(best[i >> 1], (float)d[nt][i] * u[nt][i & 1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 1));
            best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 2));
            const int pp = p + r * 8 + g;
            if (pp < p1) {
                uint32_t key = ek[r] == EXP_ALL ? 0xfffffffeu : ordered(best[r] * pow2(ek[r]));
                if (pp < a.sink || pp >= P - a.recent) key = 0xffffffffu;
                if (!ok[r]) key = 0u;
                for (int k = t; k < (int)cluster.num_blocks(); k += 4) cluster.map_shared_rank(keys, k)[pp] = key;
            }
        }
    }
}

// The k largest of keys[0 .. P) (0 < k <= P <= 16384, in shared memory, 16-byte aligned, with room up to a
// multiple of 4), ties to the lowest page, are numbered in rising order; those numbered i0 .. i1 go to
// out[0 .. i1 - i0).  A radix select of 8 bits a pass that starts below the bits which all keys have in common
// (scores of one sequence differ little in sign and exponent; the keys of the pages that are always chosen are
// left out) and ends as soon as all of a digit's keys, or a known one of at most 32, are the last chosen.  An
// ordered pass with ballots then writes the pages.
struct Chooser {
    uint32_t low, high, cut;
    int always, zeros, bin, need, count, taken, last;
    uint64_t cand[32];
    int hist[256], warp_sum[32];
};
template <int THREADS>
__device__ __forceinline__ void choose(uint32_t* keys, int P, int k, int i0, int i1, int32_t* out, Chooser& s) {
    constexpr int W = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        s.low = ~0u;
        s.high = 0u;
        s.always = s.zeros = 0;
    }
    if (tid < ((4 - P) & 3)) keys[P + tid] = 0u;
    for (int i = tid; i < 256; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    uint32_t low = ~0u, high = 0u;
    int always = 0, zeros = 0;
    for (int p = 4 * tid; p < P; p += 4 * THREADS) {
        const uint4 v = *reinterpret_cast<const uint4*>(keys + p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t key = (&v.x)[e];
            const bool a = key >= 0xfffffffeu;
            always += a;
            zeros += key == 0u;
            low = min(low, key ? key : ~0u);
            high = max(high, a ? 0u : key);
        }
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    always = __reduce_add_sync(0xffffffffu, always);
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (lane == 0) {
        atomicMin(&s.low, low);
        atomicMax(&s.high, high);
        if (always) atomicAdd(&s.always, always);
        if (zeros) atomicAdd(&s.zeros, zeros);
    }
    __syncthreads();
    // keys with the bits from `bits` up equal to prefix's are still in question; `need` of them are chosen
    int bits = 32, need = k, last = P;  // last: the last page among the chosen keys equal to the cut
    uint32_t prefix = 0u, highest = ~0u;
    if (k > s.always && s.zeros == ((4 - P) & 3)) {  // no key of 0 (a page that cannot be read) but the padding
        bits = s.low == s.high ? 0 : 32 - __clz(s.low ^ s.high);
        prefix = bits < 32 ? s.low >> bits << bits : 0u;
        need = k - s.always;
        highest = 0xfffffffdu;
        if (bits == 0 && need == P - s.always) bits = -1;  // all of them
    }
    while (bits > 0) {
        const int width = min(8, bits), shift = bits - width;
        for (int p = tid; p < P; p += THREADS) {
            const uint32_t key = keys[p];
            if (key <= highest && (bits == 32 || key >> bits == prefix >> bits))
                atomicAdd(&s.hist[(key >> shift) & ((1 << width) - 1)], 1);
        }
        __syncthreads();
        if (warp == 0) {  // lane: 8 digits, from the highest down
            int mine[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                mine[e] = s.hist[255 - 8 * lane - e];
                s.hist[255 - 8 * lane - e] = 0;
                sum += mine[e];
            }
            int above = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += y;
            }
            above -= sum;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (above < need && need <= above + mine[e]) {
                    s.bin = 255 - 8 * lane - e;
                    s.need = need - above;
                    s.count = mine[e];
                    s.taken = 0;
                }
                above += mine[e];
            }
        }
        __syncthreads();
        prefix |= (uint32_t)s.bin << shift;
        need = s.need;
        bits = shift;
        if (s.count == need) break;  // every key of the digit
        if (s.count <= 32 && bits > 0) {
            for (int p = tid; p < P; p += THREADS) {
                const uint32_t key = keys[p];
                if (key <= highest && key >> bits == prefix >> bits)
                    s.cand[atomicAdd(&s.taken, 1)] = (uint64_t)key << 32 | (uint32_t)~p;
            }
            __syncthreads();
            if (warp == 0) {
                const uint64_t mine = lane < s.count ? s.cand[lane] : 0ull;
                int above = 0;
                for (int o = 0; o < s.count; ++o) above += s.cand[o] > mine;
                if (lane < s.count && above == need - 1) {
                    s.cut = (uint32_t)(mine >> 32);
                    s.last = (int)~(uint32_t)mine;
                }
            }
            __syncthreads();
            prefix = s.cut;
            last = s.last;
            need = 0;
            break;
        }
    }
    // ordered passes: warp w takes the pages from w R
    const int R = (P + 32 * W - 1) / (32 * W) * 32, q0 = warp * R, q1 = min(P, q0 + R);
    if (bits == 0 && need > 0) {  // equal keys left: the first `need` of them (or all)
        int n = 0;
        for (int p = q0; p < q1; p += 32) n += __popc(__ballot_sync(0xffffffffu, p + lane < P && keys[p + lane] == prefix));
        if (lane == 0) s.warp_sum[warp] = n;
        if (tid == 0) s.last = P;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
        if (before < need && need <= before + n)
            for (int p = q0; p < q1; p += 32) {
                const uint32_t eq = __ballot_sync(0xffffffffu, p + lane < P && keys[p + lane] == prefix);
                if ((eq >> lane & 1) && before + __popc(eq & ((1u << lane) - 1)) == need - 1) s.last = p + lane;
                before += __popc(eq);
            }
        __syncthreads();
        last = s.last;
    }
    __syncthreads();  // warp_sum is read before it is written again
    auto chosen = [&](int p) { return p < P && (keys[p] > prefix || (keys[p] == prefix && p <= last)); };
    int n = 0;
    for (int p = q0; p < q1; p += 32) n += __popc(__ballot_sync(0xffffffffu, chosen(p + lane)));
    if (lane == 0) s.warp_sum[warp] = n;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < warp; ++w) at += s.warp_sum[w];
    for (int p = q0; p < q1; p += 32) {
        const bool go = chosen(p + lane);
        const uint32_t all = __ballot_sync(0xffffffffu, go);
        const int mine = at + __popc(all & ((1u << lane) - 1));
        if (go && mine >= i0 && mine < i1) out[mine - i0] = p + lane;
        at += __popc(all);
    }
    __syncthreads();
}

// The same over a cluster whose CTAs hold a slice of the keys each (this one's the m pages from p0), for
// more keys than one CTA can hold: a radix select whose digit counts are added over the cluster.
// The chosen pages go to list in global memory.  counts: [4][256] ints, one digit each.
template <int THREADS>
__device__ __forceinline__ void choose_cluster(const uint32_t* keys, int p0, int m, int k, int* counts, int32_t* list,
                                       int* smem32) {
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_all;
    __shared__ int2 s_own;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, cs = cluster.num_blocks();
    for (int i = tid; i < 4 * 256; i += THREADS) counts[i] = 0;
    __syncthreads();
    uint32_t prefix = 0, mask = 0;
    int need = k;
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        int* cnt = counts + 256 * pass;
        for (int w0 = tid & ~31; w0 < m; w0 += THREADS) {  // whole warps
            const int p = w0 + (tid & 31);
            const uint32_t key = p < m ? keys[p] : 0u;
            const bool in = p < m && (key & mask) == prefix;
            const uint32_t who = __ballot_sync(0xffffffffu, in);
            if (in) {
                // one addition for each digit that the warp's lanes have
                const uint32_t digit = (key >> shift) & 255, peers = __match_any_sync(who, digit);
                if ((peers & ((1u << (tid & 31)) - 1)) == 0) atomicAdd(&cnt[digit], __popc(peers));
            }
        }
        cluster.sync();
        // digits 255 - 2 tid and the one below: how many keys of the prefix there are
        int hi = 0, lo = 0;
        if (tid < 128)
            for (int r = 0; r < cs; ++r) {
                const int2 v = *reinterpret_cast<const int2*>(cluster.map_shared_rank(cnt, r) + 254 - 2 * tid);
                lo += v.x;
                hi += v.y;
            }
        int total;
        const int above = block_exclusive_scan(hi + lo, &total, smem32);
        if (above < need && need <= above + hi + lo) {
            const bool first = need <= above + hi;
            s_prefix = prefix | (uint32_t)(first ? 255 - 2 * tid : 254 - 2 * tid) << shift;
            s_need = need - above - (first ? 0 : hi);
            s_all = s_need == (first ? hi : lo);
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        mask |= 255u << shift;
        if (s_all) break;  // every key of the prefix is chosen
    }
    const int each = (m + THREADS - 1) / THREADS, q0 = min(m, tid * each), q1 = min(m, q0 + each);
    int gt = 0, eq = 0;
    for (int p = q0; p < q1; ++p) {
        gt += (keys[p] & mask) > prefix;
        eq += (keys[p] & mask) == prefix;
    }
    int gts, eqs;
    int gt0 = block_exclusive_scan(gt, &gts, smem32), eq0 = block_exclusive_scan(eq, &eqs, smem32);
    if (tid == 0) s_own = make_int2(gts, eqs);
    cluster.sync();
    for (int r = 0; r < (int)cluster.block_rank(); ++r) {
        const int2 v = *cluster.map_shared_rank(&s_own, r);
        gt0 += v.x;
        eq0 += v.y;
    }
    int at = gt0 + min(eq0, need);
    for (int p = q0; p < q1; ++p) {
        const uint32_t key = keys[p] & mask;
        if (key > prefix || (key == prefix && eq0 < need)) list[at++] = p0 + p;
        eq0 += key == prefix;
    }
    cluster.sync();  // the others' shared memory stays until everyone has read it
}

// A warp's partial of the share's pages, without tensor cores: 16 tokens at a time; for Q K^T lane =
// (half of D, token), for P V lane = D / 32 channels.  Writes m, l, o to the warp's rows.
template <typename T, int D, int GM, int WARPS>
__device__ __forceinline__ void attend_simple(const mentat_kv_cache& c, const SparseArgs& a, int h, int len,
                                              const int32_t* pages, const int32_t* blocks, int count, const float* qf,
                                              float* pm, float* pl, float* po) {
    constexpr int DL = D / 32, V = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.G, H = c.num_kv_heads, bs = c.block_size;
    float m[GM], l[GM], o[GM][DL];
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int j = 0; j < DL; ++j) o[g][j] = 0.f;
    }
    const int per = (bs + 15) / 16;  // groups of 16 rows of a page
    for (int i = warp; i < count * per; i += WARPS) {
        const int p = pages[i / per], b = blocks[i / per], t0 = (i % per) * 16;
        const int live = min(min(bs - t0, 16), len - (p * bs + t0));
        if (b < 0 || live <= 0) continue;
        const int64_t base = pool_row(c, a.layer, b, t0) + (int64_t)h * D;
        const int t = lane & 15, half = lane >> 4;
        const T* kr = reinterpret_cast<const T*>(c.k_pool) + base + (int64_t)min(t, live - 1) * H * D + half * (D / 2);
        const float* qh = qf + half * (D / 2);
        const T* vr = reinterpret_cast<const T*>(c.v_pool) + base + lane * DL;
        Pack<T, DL> vv[16];  // requested before the scores, used after them
#pragma unroll
        for (int t1 = 0; t1 < 16; ++t1)
            if (t1 < live) vv[t1] = *reinterpret_cast<const Pack<T, DL>*>(vr + (int64_t)t1 * H * D);
        float s[GM];
#pragma unroll
        for (int g = 0; g < GM; ++g) s[g] = 0.f;
        for (int d = 0; d < D / 2; d += V) {
            const Pack<T, V> kv = *reinterpret_cast<const Pack<T, V>*>(kr + d);
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                if (g >= G) break;
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(qh + g * D + d + j);
                    s[g] = fmaf(Elem<T>::to_f(kv.v[j]), x.x, s[g]);
                    s[g] = fmaf(Elem<T>::to_f(kv.v[j + 1]), x.y, s[g]);
                    s[g] = fmaf(Elem<T>::to_f(kv.v[j + 2]), x.z, s[g]);
                    s[g] = fmaf(Elem<T>::to_f(kv.v[j + 3]), x.w, s[g]);
                }
            }
        }
#pragma unroll
        for (int g = 0; g < GM; ++g) {
            if (g >= G) break;
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
            s[g] = t < live ? s[g] * a.scale : -INFINITY;
            float top = s[g];
#pragma unroll
            for (int w = 8; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float mn = fmaxf(m[g], top), ref = mn == -INFINITY ? 0.f : mn;
            const float f = exp2f(m[g] - ref);
            s[g] = exp2f(s[g] - ref);
            float sum = s[g];
#pragma unroll
            for (int w = 8; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[g] = l[g] * f + sum;
            m[g] = mn;
#pragma unroll
            for (int j = 0; j < DL; ++j) o[g][j] *= f;
        }
#pragma unroll
        for (int t1 = 0; t1 < 16; ++t1) {
            if (t1 < live) {
#pragma unroll
                for (int g = 0; g < GM; ++g) {
                    if (g >= G) break;
                    const float w = __shfl_sync(0xffffffffu, s[g], t1);
#pragma unroll
                    for (int j = 0; j < DL; ++j) o[g][j] = fmaf(w, Elem<T>::to_f(vv[t1].v[j]), o[g][j]);
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        if (g >= G) break;
        if (lane == 0) {
            pm[warp * GM + g] = m[g];
            pl[warp * GM + g] = l[g];
        }
#pragma unroll
        for (int j = 0; j < DL; ++j) po[(warp * G + g) * D + lane * DL + j] = o[g][j];
    }
}

// The same on tensor cores (16-bit types, pages of 16 rows or a multiple).  Every warp has a ring of its
// own: one lane copies the K and V tiles of 16 tokens by TMA (rows of 128 bytes, 16-byte chunk c of row r
// at chunk c ^ (r & 7)), SPARSE_STAGES - 1 tiles ahead.
//
// Lane (g, t) = (lane / 4, lane % 4).  S = Q K^T has the heads as the 16 rows (8 of them zero for GM 8)
// and 8 tokens as columns; O = P V has 8 channels as columns and takes P from the registers of S.
// Which token or channel a column stands for is free, as is the order of the channels in the first product
// (Q is loaded in the same order), so they are chosen for 16-byte reads of shared memory without bank
// conflicts: column n of S is token n / 2 + 4 (n odd), a lane's 16 bytes of K serve two products, and column
// n of O is in the chunk n / 2 + 4 (n odd) of 8 channels, whose 8 channels are 8 products.
//
// The product takes P in two parts, the element type's nearest and that one's of what is left, so a weight is off by
// at most the square of half a step (2^-16 in bf16) of itself, far below the rounding of the output; its sum is taken
// before that.  For GM 8 the second part has the rows that are zero otherwise, and costs no product.  Half has P times
// 2^15, since its steps below 2^-14 do not shrink with the value; the factor is in the sum too.  (One part: 3 % less
// time for the batch below, and an error against 64 bits 3 to 5 % above that of the output's rounding alone.)
//
// Bound by memory: 64 sequences with 128 pages each for 8 KV heads of 128 (540 MB of different rows, 1.07 GB with
// those that several sequences chose) take 88 us alone with cold caches, 6.1 TB/s of the former.  A tile of the larger tensor-core
// instruction has 128 rows, of which a KV head's group would fill at most 16.
template <typename T, int D, int GM>
__device__ __forceinline__ void attend_mma(const mentat_kv_cache& c, const SparseArgs& a, const CUtensorMap* mk,
                                           const CUtensorMap* mv, int h, int len, const int32_t* pages,
                                           const int32_t* blocks, int count, const T* q, uint8_t* ring, uint64_t* bars,
                                           float* pm, float* pl, float* po) {
    constexpr int QC = D / 32, VC = D / 64, ST = SPARSE_STAGES, HALF = 16 * 128, TILE = 2 * VC * HALF;
    constexpr int WARPS = sparse_warps(true);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, G = a.G, bs = c.block_size;
    uint2 qa[QC][2], qb[QC][2];  // rows g and g + 8
#pragma unroll
    for (int j = 0; j < QC; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = 32 * j + 8 * t + 4 * i;
            qa[j][i] = g < G ? *reinterpret_cast<const uint2*>(q + g * D + d) : make_uint2(0, 0);
            qb[j][i] = GM > 8 && g + 8 < G ? *reinterpret_cast<const uint2*>(q + (g + 8) * D + d) : make_uint2(0, 0);
        }
    float o[VC][8][4];
#pragma unroll
    for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[i][e][0] = o[i][e][1] = o[i][e][2] = o[i][e][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows g and g + 8
    constexpr float UP = std::is_same<T, __half>::value ? 32768.f : 1.f;
    const int per = bs / 16, total = count * per;
    const uint32_t bar0 = smem_u32(bars + warp * ST), ring0 = smem_u32(ring) + warp * ST * TILE;
    // tile i of the share into a stage, whose last reads are behind a __syncwarp
    auto request = [&](int i, int stage) {
        if (i < total && lane == 0) {
            const int b = blocks[i / per];
            const uint32_t bar = bar0 + 8 * stage, to = ring0 + stage * TILE;
            mbar_expect_tx(bar, b < 0 ? 0 : TILE);
            if (b >= 0) {
                const int z = b * bs + (i % per) * 16;
#pragma unroll
                for (int x = 0; x < VC; ++x) tma_load_3d(to + x * HALF, mk, bar, 64 * x, h, z);
#pragma unroll
                for (int x = 0; x < VC; ++x) tma_load_3d(to + (VC + x) * HALF, mv, bar, 64 * x, h, z);
            }
        }
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) request(warp + s * WARPS, s);
    int stage = 0, parity = 0;
    // a lane's reads: K rows t', t' + 8 (token of column g), V rows t, t + 4, t + 8, t + 12, chunk of column g
    const int kr = (g >> 1) + 4 * (g & 1), vc = kr;
    for (int i = warp; i < total; i += WARPS) {
        __syncwarp();
        request(i + (ST - 1) * WARPS, stage == 0 ? ST - 1 : stage - 1);
        if (!__all_sync(0xffffffffu, mbar_wait(bar0 + 8 * stage, parity))) {
            if (lane == 0) set_error(c, MENTAT_DEV_DECODE_TIMEOUT, 8);
            // the copies still on the way end before the shared memory is used again or given back
            for (int s = 1; s < ST; ++s) {
                stage = stage == ST - 1 ? 0 : stage + 1;
                parity ^= stage == 0;
                if (i + s * WARPS < total) (void)mbar_wait(bar0 + 8 * stage, parity);
            }
            break;
        }
        const uint8_t* kt = ring + (warp * ST + stage) * TILE;
        const uint8_t* vt = kt + VC * HALF;
        stage = stage == ST - 1 ? 0 : stage + 1;
        parity ^= stage == 0;
        const int live = min(16, len - (pages[i / per] * bs + (i % per) * 16));
        if (blocks[i / per] < 0 || live <= 0) continue;
        float s[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
            float s2[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products, half as long
#pragma unroll
            for (int j = 0; j < QC; ++j) {
                const uint4 kv = *reinterpret_cast<const uint4*>(kt + (j >> 1) * HALF + (kr + 8 * r) * 128 +
                                                                 ((((j & 1) * 4 + t) ^ kr) << 4));
                mma_16<T>(s[r], qa[j][0].x, qb[j][0].x, qa[j][0].y, qb[j][0].y, kv.x, kv.y);
                mma_16<T>(s2, qa[j][1].x, qb[j][1].x, qa[j][1].y, qb[j][1].y, kv.z, kv.w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[r][e] += s2[e];
#pragma unroll
            for (int e = 0; e < 4; ++e)  // columns 2t and 2t + 1: tokens t and t + 4
                s[r][e] = 8 * r + t + 4 * (e & 1) < live ? s[r][e] * a.scale : -INFINITY;
        }
        uint32_t pa[2][2], pb[2][2];  // [row g or g + 8][tokens t, t + 4 or t + 8, t + 12]: first and second part
#pragma unroll
        for (int x = 0; x < (GM > 8 ? 2 : 1); ++x) {
            float top = fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float mn = fmaxf(m[x], top), ref = mn == -INFINITY ? 0.f : mn;
            const float f = exp2f(m[x] - ref);
            m[x] = mn;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float u = exp2f(s[r][2 * x] - ref) * UP, v = exp2f(s[r][2 * x + 1] - ref) * UP;
                pa[x][r] = pack2(T{}, u, v);
                const Pack<T, 2> w = *reinterpret_cast<const Pack<T, 2>*>(&pa[x][r]);
                pb[x][r] = pack2(T{}, u - Elem<T>::to_f(w.v[0]), v - Elem<T>::to_f(w.v[1]));
                sum += u + v;
            }
            l[x] = l[x] * f + sum;  // over the lanes of a row at the end
#pragma unroll
            for (int j = 0; j < VC; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[j][e][2 * x] *= f;
                    o[j][e][2 * x + 1] *= f;
                    if (GM <= 8) {
                        o[j][e][2] *= f;
                        o[j][e][3] *= f;
                    }
                }
        }
        if (GM <= 8) {
            pa[1][0] = pb[0][0];
            pa[1][1] = pb[0][1];
        }
#pragma unroll
        for (int j = 0; j < VC; ++j) {
            uint4 w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[r] = *reinterpret_cast<const uint4*>(vt + j * HALF + (t + 4 * r) * 128 + ((vc ^ (t + 4 * (r & 1))) << 4));
                // rows past the last token may hold anything; their weight is 0
                if (live < 16 && t + 4 * r >= live) w[r] = make_uint4(0, 0, 0, 0);
            }
            bool finite = true;  // an infinity times what is left of its weight, which may be 0, would be NaN
            if (GM > 8) {
                uint32_t top = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e2 = 0; e2 < 4; ++e2) top = __vmaxu2(top, (&w[r].x)[e2] & 0x7fff7fffu);
                constexpr uint32_t INF = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80;
                finite = __all_sync(0xffffffffu, (top & 0xffff) < INF && top >> 16 < INF);
            }
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) {
                const uint32_t v0 = (&w[0].x)[e2], v1 = (&w[1].x)[e2], v2 = (&w[2].x)[e2], v3 = (&w[3].x)[e2];
                const uint32_t b0 = __byte_perm(v0, v1, 0x5410), b1 = __byte_perm(v2, v3, 0x5410);
                const uint32_t b2 = __byte_perm(v0, v1, 0x7632), b3 = __byte_perm(v2, v3, 0x7632);
                mma_16<T>(o[j][2 * e2], pa[0][0], pa[1][0], pa[0][1], pa[1][1], b0, b1);
                mma_16<T>(o[j][2 * e2 + 1], pa[0][0], pa[1][0], pa[0][1], pa[1][1], b2, b3);
                if (GM > 8 && finite) {
                    mma_16<T>(o[j][2 * e2], pb[0][0], pb[1][0], pb[0][1], pb[1][1], b0, b1);
                    mma_16<T>(o[j][2 * e2 + 1], pb[0][0], pb[1][0], pb[0][1], pb[1][1], b2, b3);
                }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < (GM > 8 ? 2 : 1); ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    __syncthreads();  // the partials take the rings' place
#pragma unroll
    for (int x = 0; x < (GM > 8 ? 2 : 1); ++x) {
        const int row = g + 8 * x;
        if (row >= G) continue;
        if (t == 0) {
            pm[warp * GM + row] = m[x];
            pl[warp * GM + row] = l[x];
        }
        float* w = po + (warp * G + row) * D;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {  // columns 2t and 2t + 1: chunks t and t + 4
                w[64 * j + 8 * t + e] = o[j][e][2 * x] + (GM <= 8 && isfinite(o[j][e][2]) ? o[j][e][2] : 0.f);
                w[64 * j + 32 + 8 * t + e] = o[j][e][2 * x + 1] + (GM <= 8 && isfinite(o[j][e][3]) ? o[j][e][3] : 0.f);
            }
    }
}

// LISTED: the choice was made before (k_score, k_choose); only the attention is left.
template <typename T, int D, int GM, bool MMA, bool LISTED>
__global__ void __launch_bounds__(32 * sparse_warps(MMA)) k_sparse(const __grid_constant__ CUtensorMap mk,
                                                           const __grid_constant__ CUtensorMap mv, mentat_kv_cache c,
                                                           mentat_page_index x, SparseArgs a) {
    constexpr int SPARSE_WARPS = sparse_warps(MMA), SPARSE_THREADS = 32 * SPARSE_WARPS;
    extern __shared__ int smem_raw[];
    int* smem = smem_raw + (((smem_u32(smem_raw) + 1023) & ~1023u) - smem_u32(smem_raw)) / 4;
    __shared__ uint64_t bars[SPARSE_WARPS * SPARSE_STAGES];
    __shared__ Chooser s_choose;
    __shared__ float s_unit[SPARSE_MAX_GROUP];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, cs = cluster.num_blocks(), rank = cluster.block_rank();
    const int n = blockIdx.y, h = blockIdx.x / cs, G = a.G, H = c.num_kv_heads, bs = c.block_size;
    const SparseSmem at = sparse_smem(G, GM, D, MMA, LISTED, a.held, a.share);
    float* pm = reinterpret_cast<float*>(smem + at.ml);
    float* pl = pm + SPARSE_WARPS * GM;
    float* po = reinterpret_cast<float*>(smem + at.po);
    int8_t* q8 = reinterpret_cast<int8_t*>(smem + at.q8);
    float* qf = reinterpret_cast<float*>(smem + at.qf);
    uint32_t* keys = reinterpret_cast<uint32_t*>(smem + at.keys);
    int32_t* pages = smem + at.pages;
    int32_t* blocks = smem + at.blocks;
    if (MMA && tid == 0) {
        for (int i = 0; i < SPARSE_WARPS * SPARSE_STAGES; ++i) mbar_init(smem_u32(bars + i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (!LISTED && cs > 1) cluster.barrier_arrive();  // this CTA runs: its shared memory may be written
    griddep_wait();
    griddep_launch();

    const int slot = a.slots[n];
    const T* q = reinterpret_cast<const T*>(a.q) + n * a.qs + (int64_t)h * G * D;
    T* out = reinterpret_cast<T*>(a.out) + n * a.os + (int64_t)h * G * D;
    int len = 0;
    if (slot < 0 || slot >= c.max_seqs) {
        if (tid == 0) set_error(c, MENTAT_DEV_BAD_SLOT, slot);
    } else {
        len = c.ntok[seq_index(c, a.layer, slot)];
    }
    int P = (len + bs - 1) / bs;
    if (len > a.max_len || P > c.max_blocks_per_seq) {
        if (!LISTED && tid == 0) set_error(c, MENTAT_DEV_PLAN_OVERFLOW, slot);
        P = 0;
    }
    const int32_t* row = P ? table_row(c, a.layer, slot) : nullptr;
    const int k = min(P, a.budget);
    if (!MMA)
        for (int i = tid; i < G * D; i += SPARSE_THREADS) qf[i] = Elem<T>::to_f(q[i]);

    const int i0 = (int)((int64_t)rank * k / cs), count = (int)((int64_t)(rank + 1) * k / cs) - i0;
    if (!LISTED && cs > 1) cluster.barrier_wait();
    if (!LISTED && P > k) {  // every CTA of the cluster alike
        for (int g = warp; g < (GM < 8 ? 8 : GM); g += SPARSE_WARPS)
            quantise<T, D>(q + g * D, g < G, q8 + 2 * g * D, s_unit + g);
        __syncthreads();
        const int each = (P + cs - 1) / cs, p0 = min(P, rank * each), p1 = min(P, p0 + each);
        score_pages<D, GM, SPARSE_WARPS>(c, x, a, h, row, P, p0, p1, q8, s_unit, keys);
        if (cs > 1) cluster.sync(); else __syncthreads();
        choose<SPARSE_THREADS>(keys, P, k, i0, i0 + count, pages, s_choose);
    }
    // this CTA's share of the chosen pages, and their blocks
    int32_t* told = !LISTED && a.pages ? a.pages + ((int64_t)n * H + h) * a.budget : nullptr;
    for (int i = tid; i < count; i += SPARSE_THREADS) {
        const int p = LISTED ? a.list[((int64_t)n * H + h) * a.budget + i0 + i] : P > k ? pages[i] : i0 + i, b = row[p];
        const bool ok = (unsigned)b < (unsigned)c.num_blocks;
        if (!ok) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        pages[i] = p;
        blocks[i] = ok ? b : -1;
        if (told) told[i0 + i] = p;
    }
    if (told && rank == 0)
        for (int i = k + tid; i < a.budget; i += SPARSE_THREADS) told[i] = -1;
    if (MMA && !LISTED) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // keys, then TMA, in one place
    __syncthreads();
    if constexpr (MMA)
        attend_mma<T, D, GM>(c, a, &mk, &mv, h, len, pages, blocks, count, q, reinterpret_cast<uint8_t*>(smem), bars, pm,
                             pl, po);
    else
        attend_simple<T, D, GM, SPARSE_WARPS>(c, a, h, len, pages, blocks, count, qf, pm, pl, po);
    __syncthreads();
    // the warps' partials into the first one's place
    for (int i = tid; i < G * D; i += SPARSE_THREADS) {
        const int g = i / D;
        float mx = pm[g];
#pragma unroll
        for (int w = 1; w < SPARSE_WARPS; ++w) mx = fmaxf(mx, pm[w * GM + g]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float os = 0.f;
#pragma unroll
        for (int w = 0; w < SPARSE_WARPS; ++w) os += po[w * G * D + i] * exp2f(pm[w * GM + g] - ref);
        po[i] = os;
    }
    __syncthreads();
    if (tid < G) {
        float mx = pm[tid], ls = 0.f;
        for (int w = 1; w < SPARSE_WARPS; ++w) mx = fmaxf(mx, pm[w * GM + tid]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        for (int w = 0; w < SPARSE_WARPS; ++w) ls += pl[w * GM + tid] * exp2f(pm[w * GM + tid] - ref);
        pm[tid] = mx;
        pl[tid] = ls;
    }
    // and the CTAs' into the output, a part of it each
    if (cs > 1) cluster.sync(); else __syncthreads();
    const int part = (G * D + cs - 1) / cs, o0 = min(G * D, rank * part), o1 = min(G * D, o0 + part);
    for (int i = o0 + tid; i < o1; i += SPARSE_THREADS) {
        const int g = i / D;
        float mx = -INFINITY;
        for (int r = 0; r < cs; ++r) mx = fmaxf(mx, cluster.map_shared_rank(pm, r)[g]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float ls = 0.f, os = 0.f;
        for (int r = 0; r < cs; ++r) {
            const float f = exp2f(cluster.map_shared_rank(pm, r)[g] - ref);
            ls += cluster.map_shared_rank(pl, r)[g] * f;
            os += cluster.map_shared_rank(po, r)[i] * f;
        }
        out[i] = Elem<T>::from_f(P ? os / ls : 0.f);  // an empty sequence gives zeros
    }
    if (cs > 1) cluster.sync();  // the others' shared memory stays until everyone has read it
}

// ---------------------------------------------------------------------------
// large batches: scores, choice and attention in launches of their own
// ---------------------------------------------------------------------------
// Adjacent sequences of a tree share most of their pages, so a CTA scores its pages for several
// of them at once: the query heads of up to 16 sequences are the columns of the product (GP columns each,
// the group rounded up to a power of two; the columns past the group have no part; at most 64 columns), and
// where all of them have the same 16 blocks the bounds are read once.  Two warps take 16 pages, half of the
// columns each.  Pages that are not shared are put aside, and then shared out by sequence among all warps of the
// CTA.  A warp has the next pages' bounds and the blocks of those after them on the way while it works.
// Bound by latency and issue: 64 sequences of 2,050 to 2,300 pages, 2,048 in common, 8 KV heads of 4 query heads: 19 us,
// 21 alone with cold caches (the bounds are 4 MB, the byte products 3 us); 24 where each warp pair scored its own unshared tiles.
constexpr int SCORE_THREADS = 256, SCORE_WARPS = SCORE_THREADS / 32;
constexpr int SCORE_TILES = SCORE_WARPS / 2;  // tiles of 16 pages at a time
constexpr int SCORE_ASIDE = 1024;             // tiles between two looks at those put aside

// The query heads in 8 bits, [n][Hq][2 D], negative part and positive part, and their units.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_score_queries(const T* q, int64_t qs, int heads, int Hq, int8_t* q8, float* units) {
    griddep_wait();
    griddep_launch();
    const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i < heads)
        quantise<T, D>(q + (int64_t)(i / Hq) * qs + (int64_t)(i % Hq) * D, true, q8 + (int64_t)i * 2 * D, units + i);
}

// d = the bounds of 16 pages times N tiles of 8 columns; cols: the first of lane (g, t)'s bytes
template <int D, int N>
__device__ __forceinline__ void score_product(const int4 (&v)[2][2 * D / 64], const uint8_t* cols, int (&d)[N][4]) {
    constexpr int QS = 2 * D + 16;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0;
#pragma unroll
        for (int ch = 0; ch < 2 * D / 64; ++ch) {
            const int4 b = *reinterpret_cast<const int4*>(cols + k * 8 * QS + ch * 64);
            mma_s8(d[k], v[0][ch].x, v[1][ch].x, v[0][ch].y, v[1][ch].y, b.x, b.y);
            mma_s8(d[k], v[0][ch].z, v[1][ch].z, v[0][ch].w, v[1][ch].w, b.z, b.w);
        }
    }
}

template <int GP>
struct ScoreShape {  // sequences and columns of a CTA
    static constexpr int ROWS = GP > 4 ? 64 / GP : 16, COLS = ROWS * GP;
};

template <int D, int GP>
__global__ void __launch_bounds__(SCORE_THREADS, 2) k_score(mentat_kv_cache c, mentat_page_index x, SparseArgs a,
                                                         const uint4* q8, const float* units) {
    constexpr int ROWS = ScoreShape<GP>::ROWS, COLS = ScoreShape<GP>::COLS, IDS = ROWS / 2;
    constexpr int CH = 2 * D / 64, QS = 2 * D + 16;  // a column's bytes, padded against bank conflicts
    constexpr int HALF = COLS / 16;                  // column tiles of a warp
    extern __shared__ __align__(16) uint8_t smem_q[];  // [COLS][QS]
    __shared__ __align__(8) float s_unit[COLS];
    __shared__ int s_pages[ROWS];
    __shared__ const int32_t* s_row[ROWS];
    __shared__ int s_aside[SCORE_ASIDE], s_count;
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.G, H = c.num_kv_heads, Hq = G * H, h = blockIdx.y, bs = c.block_size;
    const int n0 = blockIdx.z * ROWS, rows = min(ROWS, a.n - n0);
    int P = 0;
    if (tid < rows) {
        const int slot = a.slots[n0 + tid];
        int len = 0;
        if (slot < 0 || slot >= c.max_seqs) {
            if (blockIdx.x == 0) set_error(c, MENTAT_DEV_BAD_SLOT, slot);
        } else {
            len = c.ntok[seq_index(c, a.layer, slot)];
        }
        P = (len + bs - 1) / bs;
        if (len > a.max_len || P > c.max_blocks_per_seq) {
            if (blockIdx.x == 0) set_error(c, MENTAT_DEV_PLAN_OVERFLOW, slot);
            P = 0;
        }
        s_row[tid] = P ? table_row(c, a.layer, slot) : nullptr;
    }
    if (tid < ROWS) s_pages[tid] = P;  // 0 for the sequences past the batch
    // neighbouring tiles go to different CTAs: the ones that are not shared lie together
    const int tile0 = (warp >> 1) * gridDim.x + blockIdx.x, step = gridDim.x * SCORE_TILES, half = warp & 1;
    if (!__syncthreads_or(P > (int)blockIdx.x * 16 && P > a.budget)) return;  // nothing to choose
    for (int w = tid; w < COLS * (D / 8); w += SCORE_THREADS) {
        const int col = w / (D / 8), ch = w % (D / 8), i = col / GP, e = col % GP;
        const int src = i < rows && e < G ? 16 : 0;
        const uint4* from = q8 + ((int64_t)(n0 + min(i, rows - 1)) * Hq + h * G + min(e, G - 1)) * (D / 8) + ch;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_q + col * QS + ch * 16)), "l"(from),
                     "r"(src)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (tid < COLS) {  // a column without a head: NaN, which no maximum takes
        const int i = tid / GP, e = tid % GP;
        s_unit[tid] = i < rows && e < G ? units[(int64_t)(n0 + i) * Hq + h * G + e] : __int_as_float(0x7fffffff);
    }
    int most = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) most = max(most, s_pages[i]);
    const int tiles = (most + 15) / 16;
    const int64_t base = (int64_t)a.layer * c.num_blocks;

    // a lane's blocks of tile tl: page lane % 16 of every second sequence; NONE where a sequence has no such page
    constexpr int NONE = -2147483647 - 1;
    auto fetch = [&](int tl, int (&id)[IDS]) {
        const int pp = tl * 16 + (lane & 15);
#pragma unroll
        for (int e = 0; e < IDS; ++e) {
            const int i = 2 * e + (lane >> 4);
            id[e] = pp < s_pages[i] ? s_row[i][pp] : NONE;
        }
    };
    // whether every sequence that has the tile's pages has the same (readable) blocks there; `first`: the blocks
    auto common = [&](const int (&id)[IDS], int& first) {
        first = -1;
        bool same = true;
#pragma unroll
        for (int e = 0; e < IDS; ++e) {
            const bool good = (unsigned)id[e] < (unsigned)c.num_blocks;
            if (good && first < 0) first = id[e];
            same = same && (id[e] == NONE || (good && id[e] == first));
        }
        const int other = __shfl_xor_sync(0xffffffffu, first, 16);
        same = same && (first < 0 || other < 0 || first == other);
        first = first < 0 ? other : first;
        return (bool)__all_sync(0xffffffffu, same);
    };
    // the bounds of pages g and 8 + g of a tile, in blocks b0 and b1 (-1: any)
    auto load = [&](int b0, int b1, int4 (&v)[2][CH], int (&ek)[2]) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t at = (base + max(r ? b1 : b0, 0)) * H + h;
            ek[r] = __ldg(x.exps + at);
            const int4* src = reinterpret_cast<const int4*>(x.bounds + at * 2 * D) + t;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) v[r][ch] = __ldg(src + ch * 4);
        }
    };
    // of a sequence's columns in one column tile, the highest score for page g (r 0) or g + 8; u: the lane's units
    auto highest = [&](const int* d, float2 u, int r) {
        float best = fmaxf((float)d[2 * r] * u.x, (float)d[2 * r + 1] * u.y);
        if (GP >= 4) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        if (GP >= 8) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        return best;
    };
    uint32_t* const out = a.keys + ((int64_t)n0 * H + h) * a.key_stride;
    const int64_t out_step = (int64_t)H * a.key_stride;
    auto put = [&](int i, int pp, float best, int ek) {
        const int P = s_pages[i];
        if (pp >= P) return;
        uint32_t key = ek == EXP_ALL ? 0xfffffffeu : ordered(best * pow2(ek));
        if (pp < a.sink || pp >= P - a.recent) key = 0xffffffffu;
        if (ek == EXP_UNREADABLE) key = 0u;  // behind all others
        out[i * out_step + pp] = key;
    };
    auto unit_of = [&](int nt) { return *reinterpret_cast<const float2*>(s_unit + nt * 8 + 2 * t); };
    const uint8_t* cols = smem_q + g * QS + t * 16;

    // the next piece of work's bounds, and the blocks of the one after it, are on the way
    int4 v[2][CH], nv[2][CH];
    int ek[2], nek[2];
    auto advance = [&] {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            ek[r] = nek[r];
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) v[r][ch] = nv[r][ch];
        }
    };
    for (int t0 = 0; t0 < tiles; t0 += step * (SCORE_ASIDE / SCORE_TILES)) {
        const int t1 = min(tiles, t0 + step * (SCORE_ASIDE / SCORE_TILES));
        if (t0 > 0) __syncthreads();
        if (tid == 0) s_count = 0;
        int id[IDS], first, tl = t0 + tile0;
        bool shared = false;
        auto look = [&] {
            shared = common(id, first);
            if (shared) load(__shfl_sync(0xffffffffu, first, g), __shfl_sync(0xffffffffu, first, 8 + g), nv, nek);
        };
        if (tl < t1) {
            fetch(tl, id);
            look();
            if (tl + step < t1) fetch(tl + step, id);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        for (; tl < t1; tl += step) {
            const bool now = shared;
            advance();
            if (tl + step < t1) {
                look();
                if (tl + 2 * step < t1) fetch(tl + 2 * step, id);
            }
            if (!now) {
                if (half == 0 && lane == 0) s_aside[atomicAdd(&s_count, 1)] = tl;
                continue;
            }
            int d[HALF][4];
            const int nt0 = half * HALF;
            score_product<D, HALF>(v, cols + nt0 * 8 * QS, d);
#pragma unroll
            for (int k = 0; k < HALF; ++k) {
                const int nt = nt0 + k;
                const float2 u = unit_of(nt);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int pp = tl * 16 + r * 8 + g;
                    if (GP == 1) {  // each column is a sequence
                        put(nt * 8 + 2 * t, pp, (float)d[k][2 * r] * u.x, ek[r]);
                        put(nt * 8 + 2 * t + 1, pp, (float)d[k][2 * r + 1] * u.y, ek[r]);
                    } else if (GP <= 8) {
                        const float best = highest(d[k], u, r);
                        if (t % (GP > 2 ? GP / 2 : 1) == 0) put((nt * 8 + 2 * t) / GP, pp, best, ek[r]);
                    } else if (k % 2 == 0) {
                        const float best = fmaxf(highest(d[k], u, r), highest(d[(k + 1) % HALF], unit_of(nt + 1), r));
                        if (t == 0) put(nt / 2, pp, best, ek[r]);
                    }
                }
            }
        }
        __syncthreads();
        // (tile, sequence) by warp
        const int units = s_count * ROWS;
        int b[2];
        auto blocks_of = [&](int u) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int i = u % ROWS, pp = u < units ? s_aside[u / ROWS] * 16 + r * 8 + g : 0;
                b[r] = u < units && pp < s_pages[i] ? s_row[i][pp] : NONE;
            }
        };
        auto load_blocks = [&] {
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (b[r] != NONE && (unsigned)b[r] >= (unsigned)c.num_blocks) {
                    if (t == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b[r]);
                    b[r] = -1;
                }
            load(b[0], b[1], nv, nek);
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (b[r] == -1) nek[r] = EXP_UNREADABLE;
        };
        if (warp < units) {
            blocks_of(warp);
            load_blocks();
            blocks_of(warp + SCORE_WARPS);
        }
        constexpr int N1 = GP > 8 ? 2 : 1;
        for (int u = warp; u < units; u += SCORE_WARPS) {
            advance();
            if (u + SCORE_WARPS < units) {
                load_blocks();
                blocks_of(u + 2 * SCORE_WARPS);
            }
            const int i = u % ROWS, nt = i * GP / 8, col = i * GP % 8;  // its first column in its tile
            int d[N1][4];
            score_product<D, N1>(v, cols + nt * 8 * QS, d);
            const float2 un = unit_of(nt);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int pp = s_aside[u / ROWS] * 16 + r * 8 + g;
                if (GP == 1) {
                    if (t == col / 2) put(i, pp, (float)d[0][2 * r + (col & 1)] * (col & 1 ? un.y : un.x), ek[r]);
                } else {
                    float best = highest(d[0], un, r);
                    if (GP > 8) best = fmaxf(best, highest(d[N1 - 1], unit_of(nt + N1 - 1), r));
                    if (t == col / 2) put(i, pp, best, ek[r]);
                }
            }
        }
    }
}

// The chosen pages from the keys (12 us for 512 of 2,200 pages; made by the attention's CTAs instead, the same batch
// took 126 us in all where this took 121): one CTA per (sequence, KV head), or a cluster where a sequence may have
// more than HELD_PAGES pages.
constexpr int CHOOSE_THREADS = 256, HELD_PAGES = 16384;
template <bool CL>
__global__ void __launch_bounds__(CHOOSE_THREADS) k_choose(mentat_kv_cache c, SparseArgs a) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ int smem32[CL ? 32 : 1], counts[CL ? 4 * 256 : 1];
    __shared__ Chooser s_choose;
    griddep_wait();
    griddep_launch();
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = CL ? cluster.num_blocks() : 1, rank = CL ? cluster.block_rank() : 0;
    const int tid = threadIdx.x, n = blockIdx.y, h = blockIdx.x / cs, H = c.num_kv_heads, bs = c.block_size;
    const int slot = a.slots[n];
    int len = slot >= 0 && slot < c.max_seqs ? c.ntok[seq_index(c, a.layer, slot)] : 0;
    if (len > a.max_len || (len + bs - 1) / bs > c.max_blocks_per_seq) len = 0;
    const int P = (len + bs - 1) / bs, k = min(P, a.budget);
    int32_t* list = a.list + ((int64_t)n * H + h) * a.budget;
    if (rank == 0) {
        for (int i = k + tid; i < a.budget; i += CHOOSE_THREADS) list[i] = -1;
        if (P <= k)
            for (int i = tid; i < k; i += CHOOSE_THREADS) list[i] = i;
    }
    if (P <= k) return;  // every CTA of the cluster alike
    const int each = (P + cs - 1) / cs, p0 = min(P, rank * each), p1 = min(P, p0 + each);
    const uint32_t* from = a.keys + ((int64_t)n * H + h) * a.key_stride;
    for (int p = p0 + tid; p < p1; p += CHOOSE_THREADS) keys[p - p0] = from[p];
    __syncthreads();
    if constexpr (CL)
        choose_cluster<CHOOSE_THREADS>(keys, p0, p1 - p0, k, counts, list, smem32);
    else
        choose<CHOOSE_THREADS>(keys, P, k, 0, k, list, s_choose);
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------
// How many CTAs share one (sequence, KV head): the largest power of two up to 8 that still runs all CTAs at
// once, two on an SM.  Budget 64, 8 KV heads of 128 in bf16, sequences of up to 1,000 pages, with 1 / 2 / 4 / 8: one
// 31.8 / 21.6 / 15.4 / 12.8 us, 8 of them 36.8 / 25.7 / 19.5 / 31.0, 16 of them 41.8 / 33.1 / 40.1 / 62.6.  Of
// 2 heads of 64 in fp32, 500 pages, 32 of them 48.6 / 29.3 / 25.0 / 33.6.
static int sparse_cluster(int heads) {
    int cs = 1;
    while (cs < 8 && (int64_t)heads * cs * 2 <= 2 * 148) cs *= 2;
    return cs;
}
static bool sparse_mma(const mentat_kv_cache* c) { return c->dtype != MENTAT_F32 && c->block_size % 16 == 0; }

// Whether the scores and the choice get launches of their own: from 600 pages for each CTA to score (and past
// what k_sparse can hold).  In one launch and in several, as above: 16 sequences of up to 1,000 pages (500 a CTA)
// 33.2 and 35.7 us, 24 of them (1,000) 56.6 and 46.7; behind a prefix of 32,768 tokens in common, 2,170 pages,
// 8 of them (540) 28.9 and 29.8, 16 of them (1,090) 43 and 36, 64 of them 160 and 79.
static bool sparse_listed(const mentat_kv_cache* c, int n, int max_len, int budget) {
    const int64_t pages = ((int64_t)max_len + c->block_size - 1) / c->block_size;
    if (pages <= budget) return false;
    return pages > HELD_PAGES || pages > 600 * sparse_cluster(n * c->num_kv_heads);
}

template <typename T, int D, int GM, bool MMA, bool LISTED>
static int launch_sparse(const mentat_kv_cache* c, const mentat_page_index* x, SparseArgs a, cudaStream_t s) {
    const int pages = (a.max_len + c->block_size - 1) / c->block_size, cs = sparse_cluster(a.n * c->num_kv_heads);
    a.held = pages;
    a.share = (min(pages, a.budget) + cs - 1) / cs;
    const size_t smem = 4 * (size_t)sparse_smem(a.G, GM, D, MMA, LISTED, a.held, a.share).total + 1024;
    CUtensorMap mk{}, mv{};
    if (MMA && !pool_maps(c, a.layer, &mk, &mv)) return MENTAT_ERR_CUDA;
    return launch_cluster<k_sparse<T, D, GM, MMA, LISTED>>(cs, dim3(c->num_kv_heads * cs, a.n), 32 * sparse_warps(MMA), smem,
                                                           s, mk, mv, *c, *x, a);
}

// 16-bit types with pages of 16 rows or a multiple run on tensor cores
template <typename T, int D, int GM, bool LISTED>
static int launch_sparse_kind(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a,
                              cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (sparse_mma(c) && a.qs % 4 == 0 && (uintptr_t)a.q % 8 == 0)
            return launch_sparse<T, D, (GM > 8 ? 16 : 8), true, LISTED>(c, x, a, s);
    return launch_sparse<T, D, GM, false, LISTED>(c, x, a, s);
}

template <typename T, int D, bool LISTED>
static int launch_sparse_group(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a,
                               cudaStream_t s) {
    if (a.G <= 2) return launch_sparse_kind<T, D, 2, LISTED>(c, x, a, s);
    if (a.G <= 4) return launch_sparse_kind<T, D, 4, LISTED>(c, x, a, s);
    if (a.G <= 8) return launch_sparse_kind<T, D, 8, LISTED>(c, x, a, s);
    return launch_sparse_kind<T, D, 16, LISTED>(c, x, a, s);
}

template <int D, int GP>
static int launch_score(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a, cudaStream_t s) {
    constexpr int ROWS = ScoreShape<GP>::ROWS;
    const int pages = (a.max_len + c->block_size - 1) / c->block_size, per = SCORE_TILES * 16;
    const int groups = c->num_kv_heads * ((a.n + ROWS - 1) / ROWS), chunks = (pages + per - 1) / per;
    const int wanted = groups < 2 * 148 ? 2 * 148 / groups : 1;  // all CTAs at once, two on an SM
    const dim3 grid(wanted < chunks ? wanted : chunks, c->num_kv_heads, (a.n + ROWS - 1) / ROWS);
    MENTAT_LAUNCH((k_score<D, GP>), grid, dim3(SCORE_THREADS), ScoreShape<GP>::COLS * (2 * D + 16), s, *c, *x, a,
                  reinterpret_cast<const uint4*>(a.q8), a.units);
    return MENTAT_OK;
}

template <typename T, int D>
static int launch_sparse_dim(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a,
                             cudaStream_t s) {
    if (!a.keys) return launch_sparse_group<T, D, false>(c, x, a, s);
    const int heads = a.n * a.G * c->num_kv_heads;
    MENTAT_LAUNCH(k_score_queries<T, D>, dim3((heads + 3) / 4), dim3(128), 0, s, (const T*)a.q, a.qs, heads,
                  a.G * c->num_kv_heads, a.q8, a.units);
    int sc = MENTAT_OK;
    if (a.G == 1) sc = launch_score<D, 1>(c, x, a, s);
    else if (a.G == 2) sc = launch_score<D, 2>(c, x, a, s);
    else if (a.G <= 4) sc = launch_score<D, 4>(c, x, a, s);
    else if (a.G <= 8) sc = launch_score<D, 8>(c, x, a, s);
    else sc = launch_score<D, 16>(c, x, a, s);
    if (sc != MENTAT_OK) return sc;
    const int pages = (a.max_len + c->block_size - 1) / c->block_size;
    int cs = 1;
    while (cs < SPARSE_MAX_CLUSTER && (pages + cs - 1) / cs > HELD_PAGES) cs *= 2;
    const size_t smem = 4 * (size_t)((pages + cs - 1) / cs + 3);
    const dim3 grid(c->num_kv_heads * cs, a.n);
    const int st = cs > 1 ? launch_cluster<k_choose<true>>(cs, grid, CHOOSE_THREADS, smem, s, *c, a)
                          : launch_cluster<k_choose<false>>(1, grid, CHOOSE_THREADS, smem, s, *c, a);
    if (st != MENTAT_OK) return st;
    return launch_sparse_group<T, D, true>(c, x, a, s);
}

}  // namespace mentat

using namespace mentat;

static bool bad_index(const mentat_kv_cache* c, const mentat_page_index* x) {
    return !c || !x || !x->bounds || !x->exps || ((uintptr_t)x->bounds & 15) || c->num_layers <= 0 ||
           c->num_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535 ||
           c->head_dim <= 0 || c->head_dim > 1024 || !c->k_pool || !c->ctrl;
}
#define MENTAT_BY_DTYPE(...)                                                                        \
    switch (c->dtype) {                                                                             \
        case MENTAT_F32: { using T = float; __VA_ARGS__; break; }                                    \
        case MENTAT_BF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }                           \
        case MENTAT_F16: { using T = __half; __VA_ARGS__; break; }                                   \
        default: return MENTAT_ERR_UNSUPPORTED;                                                     \
    }

extern "C" {

int mentat_page_index_blocks(const mentat_kv_cache* c, int32_t layer, const int32_t* blocks, int32_t n,
                             const mentat_page_index* x, cudaStream_t s) {
    if (bad_index(c, x) || layer < 0 || layer >= c->num_layers || n < 0 || (n > 0 && !blocks)) return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (const int threads = index_block_threads(c)) {
        MENTAT_BY_DTYPE(MENTAT_LAUNCH((k_index_blocks<T, true>), dim3(n), dim3(threads), 0, s, *c, layer, blocks, *x))
        return MENTAT_OK;
    }
    const dim3 grid(n, c->num_kv_heads), block((c->head_dim + 31) / 32 * 32);
    MENTAT_BY_DTYPE(MENTAT_LAUNCH((k_index_blocks<T, false>), grid, block, 0, s, *c, layer, blocks, *x))
    return MENTAT_OK;
}

int mentat_page_index_seqs(const mentat_kv_cache* c, int32_t layer, const int32_t* slots, int32_t n, int32_t first,
                           int32_t max_pages, const mentat_page_index* x, cudaStream_t s) {
    if (bad_index(c, x) || layer < -1 || layer >= c->num_layers || n < 0 || first < -1 || max_pages < 0 ||
        !c->tables || !c->ntok || c->num_layers > 65535 || (n > 0 && !slots) || (int64_t)n * max_pages > 0x7fffffff ||
        (int64_t)first + max_pages > 0x7fffffff)  // a page's number is an int
        return MENTAT_ERR_ARG;
    if (first < 0) max_pages = 1;
    if (n == 0 || max_pages == 0) return MENTAT_OK;
    const int l0 = layer < 0 ? 0 : layer, layers = layer < 0 ? c->num_layers : 1;
    if (const int threads = index_block_threads(c)) {
        MENTAT_BY_DTYPE(MENTAT_LAUNCH((k_index_seqs<T, true>), dim3(n * max_pages, 1, layers), dim3(threads), 0, s, *c, l0,
                                      slots, n, first, *x, max_pages))
        return MENTAT_OK;
    }
    const dim3 grid(n * max_pages, c->num_kv_heads, layers), block((c->head_dim + 31) / 32 * 32);
    MENTAT_BY_DTYPE(MENTAT_LAUNCH((k_index_seqs<T, false>), grid, block, 0, s, *c, l0, slots, n, first, *x, max_pages))
    return MENTAT_OK;
}

int mentat_page_bounds(const mentat_kv_cache* c, int32_t layer, const int32_t* blocks, int32_t n,
                       const mentat_page_index* x, float* low, float* high, int8_t* exps, cudaStream_t s) {
    if (bad_index(c, x) || layer < 0 || layer >= c->num_layers || n < 0 || (n > 0 && (!blocks || !low || !high || !exps)))
        return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    MENTAT_LAUNCH(k_page_bounds, dim3((n + BOUNDS_PAGES - 1) / BOUNDS_PAGES), dim3(256), 0, s, *c, layer, blocks, n, *x, low,
                  high, exps);
    return MENTAT_OK;
}

int64_t mentat_sparse_workspace_bytes(const mentat_kv_cache* c, int32_t n, int32_t max_len, int32_t budget) {
    if (!c || c->block_size <= 0 || c->num_kv_heads <= 0 || n <= 0 || max_len < 0 || budget <= 0 ||
        !sparse_listed(c, n, max_len, budget))
        return 0;
    const int64_t pages = ((int64_t)max_len + c->block_size - 1) / c->block_size;
    // keys, queries (at most 16 heads of 2 head_dim bytes for each KV head) and units, chosen pages
    return 4 * (int64_t)n * c->num_kv_heads * ((pages + 3) / 4 * 4 + SPARSE_MAX_GROUP * ((int64_t)c->head_dim / 2 + 1) + budget);
}

int mentat_sparse_decode(const mentat_kv_cache* c, int32_t layer, const mentat_page_index* x, const int32_t* slots,
                         int32_t n, const void* q, int64_t q_stride, int32_t Hq, void* out, int64_t out_stride,
                         float scale, int32_t max_len, int32_t budget, int32_t sink, int32_t recent, int32_t* pages,
                         void* workspace, int64_t workspace_bytes, cudaStream_t s) {
    if (bad_index(c, x) || layer < 0 || layer >= c->num_layers || n < 0 || n > 65535 || Hq <= 0 ||
        Hq % c->num_kv_heads || max_len < 0 || !(scale > 0.f) || sink < 0 || recent < 1 || budget < 1 ||
        (int64_t)sink + recent > budget || !c->v_pool || !c->tables || !c->ntok ||
        (n > 0 && (!slots || !q || !out)) || (((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) & 15))
        return MENTAT_ERR_ARG;
    const int G = Hq / c->num_kv_heads;
    if (G > SPARSE_MAX_GROUP || budget > SPARSE_MAX_BUDGET) return MENTAT_ERR_UNSUPPORTED;
    if (((int64_t)max_len + c->block_size - 1) / c->block_size > (int64_t)HELD_PAGES * SPARSE_MAX_CLUSTER)
        return MENTAT_ERR_UNSUPPORTED;
    if (n == 0) return MENTAT_OK;
    const int64_t need = mentat_sparse_workspace_bytes(c, n, max_len, budget);
    if (workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15)))) return MENTAT_ERR_ARG;
    SparseArgs a{slots, q, q_stride, out, out_stride, pages, scale * 1.4426950408889634f, layer, G, max_len, budget,
                 sink, recent, 0, 0, nullptr, nullptr, nullptr, nullptr, 0, n};
    if (need) {
        a.key_stride = (((int64_t)max_len + c->block_size - 1) / c->block_size + 3) / 4 * 4;
        a.keys = reinterpret_cast<uint32_t*>(workspace);
        uint32_t* next = a.keys + (int64_t)n * c->num_kv_heads * a.key_stride;
        a.q8 = reinterpret_cast<int8_t*>(next);
        next += (int64_t)n * Hq * c->head_dim / 2;
        a.units = reinterpret_cast<float*>(next);
        a.list = pages ? pages : reinterpret_cast<int32_t*>(next + (int64_t)n * Hq);
    }
    int st = MENTAT_OK;
    if (c->head_dim == 128) {
        MENTAT_BY_DTYPE(st = launch_sparse_dim<T, 128>(c, x, a, s))
    } else if (c->head_dim == 64) {
        MENTAT_BY_DTYPE(st = launch_sparse_dim<T, 64>(c, x, a, s))
    } else {
        st = MENTAT_ERR_UNSUPPORTED;
    }
    return st;
}

}  // extern "C"
