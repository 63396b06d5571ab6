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
// two dot products of bytes (dp4a, int32; at most 2 * 128 * 127^2 < 2^23, exact as a
// float).  A KV head takes the highest of its query heads' scores.  Choosing by an
// exact number makes the choice reproducible.
//
// Attention.  Base-2 online softmax over the chosen pages, partials of a CTA's warps
// merged in shared memory.

#include "common.cuh"

namespace mentat {

// ---------------------------------------------------------------------------
// index
// ---------------------------------------------------------------------------
constexpr int EXP_MIN = -50, EXP_MAX = 50, EXP_ALL = 127;

// the least e with top <= 127 * 2^e, within EXP_MIN .. EXP_MAX; top finite, >= 0
__device__ __forceinline__ int unit_exponent(float top) {
    if (top == 0.f) return EXP_MIN;
    int x;
    const float m = frexpf(top, &x);  // top = m 2^x, 0.5 <= m < 1
    const int e = x - 7 + (m > 127.f / 128.f);
    return min(max(e, EXP_MIN), EXP_MAX);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

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
        o[0] = bad ? 0 : (int8_t)fminf(fmaxf(floorf(lo * inv), -127.f), 127.f);
        o[D] = bad ? 0 : (int8_t)fminf(fmaxf(ceilf(hi * inv), -127.f), 127.f);
    }
    if (d == 0) x.exps[at] = (int8_t)(bad ? EXP_ALL : e);
    __syncthreads();
}

template <typename T>
__global__ void k_index_blocks(mentat_kv_cache c, int layer, const int32_t* blocks, mentat_page_index x) {
    griddep_wait();
    const int b = blocks[blockIdx.x];
    if ((unsigned)b >= (unsigned)c.num_blocks) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        return;
    }
    index_page<T>(c, layer, b, blockIdx.y, x);
}

template <typename T>
__global__ void k_index_seqs(mentat_kv_cache c, int layer0, const int32_t* slots, int first, mentat_page_index x,
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
        if (len == 0 || len % c.block_size) return;
        p = full - 1;
    }
    if (p >= full) return;
    const int b = table_row(c, layer, slot)[p];
    if ((unsigned)b >= (unsigned)c.num_blocks) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        return;
    }
    index_page<T>(c, layer, b, blockIdx.y, x);
}

__global__ void k_page_bounds(mentat_kv_cache c, int layer, const int32_t* blocks, mentat_page_index x, float* low,
                              float* high, int8_t* exps) {
    griddep_wait();
    const int b = blocks[blockIdx.x], h = blockIdx.y, D = c.head_dim;
    if ((unsigned)b >= (unsigned)c.num_blocks) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
        return;
    }
    const int64_t at = ((int64_t)layer * c.num_blocks + b) * c.num_kv_heads + h;
    const int64_t to = (int64_t)blockIdx.x * c.num_kv_heads + h;
    const int e = x.exps[at];
    const float unit = e == EXP_ALL ? INFINITY : pow2(e);
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        low[to * D + d] = e == EXP_ALL ? -unit : x.bounds[at * 2 * D + d] * unit;
        high[to * D + d] = e == EXP_ALL ? unit : x.bounds[at * 2 * D + D + d] * unit;
    }
    if (threadIdx.x == 0) exps[to] = (int8_t)e;
}

// ---------------------------------------------------------------------------
// decode: one CTA per (sequence, KV head)
// ---------------------------------------------------------------------------
constexpr int SPARSE_THREADS = 256, SPARSE_WARPS = SPARSE_THREADS / 32;
constexpr int SPARSE_MAX_BUDGET = 8192, SPARSE_MAX_GROUP = 16;

struct SparseArgs {
    const int32_t* slots;
    const void* q;
    int64_t qs;
    void* out;
    int64_t os;
    int32_t* pages;
    float scale;  // times log2(e)
    int layer, G, max_len, cap, budget, sink, recent;
};

// shared memory: keys [cap], chosen pages [budget], q float [G][D], q bytes
// [G][2][D] (negative part, positive part), partials m, l [warps][G], o [warps][G][D]
static size_t sparse_smem(int cap, int budget, int G, int D) {
    return 4 * ((size_t)cap + budget + G * D + SPARSE_WARPS * 2 * G + (size_t)SPARSE_WARPS * G * D) + 2 * G * D + 64;
}

__device__ __forceinline__ uint32_t ordered(float f) {  // order of floats as order of integers
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The k largest of keys[0 .. P) (k <= P), ties to the lowest index, into chosen in rising order.
__device__ __forceinline__ void choose(const uint32_t* keys, int P, int k, int32_t* chosen, int* hist, int* smem32) {
    const int tid = threadIdx.x;
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    if (tid == 0) {
        s_prefix = 0;
        s_need = k;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int p = tid; p < P; p += SPARSE_THREADS)
            if ((keys[p] & mask) == prefix) atomicAdd(&hist[(keys[p] >> shift) & 255], 1);
        __syncthreads();
        // digit 255 - tid: how many keys of this prefix have a higher digit
        int total;
        const int mine = hist[255 - tid], need = s_need;
        const int above = block_exclusive_scan(mine, &total, smem32);
        if (above < need && need <= above + mine) {
            s_prefix = prefix | (uint32_t)(255 - tid) << shift;
            s_need = need - above;
        }
        __syncthreads();
    }
    const uint32_t cut = s_prefix;  // the k-th largest key; s_need of its equals are chosen
    const int need = s_need, each = (P + SPARSE_THREADS - 1) / SPARSE_THREADS;
    const int p0 = min(P, tid * each), p1 = min(P, p0 + each);
    int gt = 0, eq = 0;
    for (int p = p0; p < p1; ++p) {
        gt += keys[p] > cut;
        eq += keys[p] == cut;
    }
    int total;
    const int gt0 = block_exclusive_scan(gt, &total, smem32);
    int eq0 = block_exclusive_scan(eq, &total, smem32);
    int at = gt0 + min(eq0, need);
    for (int p = p0; p < p1; ++p) {
        const bool e = keys[p] == cut;
        if (keys[p] > cut || (e && eq0 < need)) chosen[at++] = p;
        eq0 += e;
    }
    __syncthreads();
}

template <typename T, int D, int GM>
__global__ void __launch_bounds__(SPARSE_THREADS) k_sparse(mentat_kv_cache c, mentat_page_index x, SparseArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int hist[256], smem32[32];
    __shared__ int s_eq[SPARSE_MAX_GROUP];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = blockIdx.y, h = blockIdx.x, G = a.G, H = c.num_kv_heads, bs = c.block_size;
    float* qf = reinterpret_cast<float*>(smem);
    int8_t* q8 = reinterpret_cast<int8_t*>(qf + G * D);
    float* po = reinterpret_cast<float*>(q8 + 2 * G * D);  // [warps][G][D]
    float* pm = po + SPARSE_WARPS * G * D;
    float* pl = pm + SPARSE_WARPS * G;
    uint32_t* keys = reinterpret_cast<uint32_t*>(pl + SPARSE_WARPS * G);
    int32_t* chosen = reinterpret_cast<int32_t*>(keys + a.cap);
    griddep_wait();
    griddep_launch();

    const int slot = a.slots[n];
    const T* q = reinterpret_cast<const T*>(a.q) + n * a.qs + (int64_t)h * G * D;
    T* out = reinterpret_cast<T*>(a.out) + n * a.os + (int64_t)h * G * D;
    int32_t* list = a.pages ? a.pages + ((int64_t)n * H + h) * a.budget : nullptr;
    int len = 0;
    if (slot < 0 || slot >= c.max_seqs) {
        if (tid == 0) set_error(c, MENTAT_DEV_BAD_SLOT, slot);
    } else {
        len = c.ntok[seq_index(c, a.layer, slot)];
    }
    int P = (len + bs - 1) / bs;
    if (len > a.max_len || P > c.max_blocks_per_seq) {
        if (tid == 0) set_error(c, MENTAT_DEV_PLAN_OVERFLOW, slot);
        P = 0;
    }
    const int32_t* row = P ? table_row(c, a.layer, slot) : nullptr;
    const int k = min(P, a.budget);
    for (int i = tid; i < G * D; i += SPARSE_THREADS) qf[i] = Elem<T>::to_f(q[i]);
    __syncthreads();

    if (P > k) {
        for (int g = warp; g < G; g += SPARSE_WARPS) {
            float top = 0.f;
            for (int d = lane; d < D; d += 32) top = fmaxf(top, isfinite(qf[g * D + d]) ? fabsf(qf[g * D + d]) : 0.f);
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = unit_exponent(top);
            if (lane == 0) s_eq[g] = e;
            for (int d = lane; d < D; d += 32) {
                const float v = isfinite(qf[g * D + d]) ? rintf(qf[g * D + d] * pow2(-e)) : 0.f;
                const int w = (int)fminf(fmaxf(v, -127.f), 127.f);
                q8[(2 * g) * D + d] = (int8_t)min(w, 0);
                q8[(2 * g + 1) * D + d] = (int8_t)max(w, 0);
            }
        }
        __syncthreads();
        // scores: one thread per page
        for (int p = tid; p < P; p += SPARSE_THREADS) {
            uint32_t key = 0xffffffffu;
            if (p >= a.sink && p < P - a.recent) {
                const int b = row[p];
                if ((unsigned)b >= (unsigned)c.num_blocks) {
                    set_error(c, MENTAT_DEV_BAD_BLOCK, b);
                    key = 0;
                } else {
                    const int64_t at = ((int64_t)a.layer * c.num_blocks + b) * H + h;
                    const int ek = x.exps[at];
                    const int4* bounds = reinterpret_cast<const int4*>(x.bounds + at * 2 * D);
                    int dot[GM];
#pragma unroll
                    for (int g = 0; g < GM; ++g) dot[g] = 0;
                    for (int d = 0; d < 2 * D / 16; ++d) {  // lo against the negative part, then hi against the positive
                        const int4 v = bounds[d];
#pragma unroll
                        for (int g = 0; g < GM; ++g) {
                            if (g >= G) break;
                            const int4 w = *reinterpret_cast<const int4*>(q8 + 2 * g * D + d * 16);
                            dot[g] = __dp4a(v.x, w.x, __dp4a(v.y, w.y, __dp4a(v.z, w.z, __dp4a(v.w, w.w, dot[g]))));
                        }
                    }
                    float best = -INFINITY;
#pragma unroll
                    for (int g = 0; g < GM; ++g)
                        if (g < G) best = fmaxf(best, (float)dot[g] * pow2(s_eq[g]));
                    key = ek == EXP_ALL ? 0xfffffffeu : ordered(best * pow2(ek));
                }
            }
            keys[p] = key;
        }
        __syncthreads();
        choose(keys, P, k, chosen, hist, smem32);
    } else {
        for (int p = tid; p < k; p += SPARSE_THREADS) chosen[p] = p;
        __syncthreads();
    }
    if (list)
        for (int i = tid; i < a.budget; i += SPARSE_THREADS) list[i] = i < k ? chosen[i] : -1;

    // attention: a warp takes 16 tokens at a time; for Q K^T lane = (half of D, token), for P V lane = D / 32 channels
    constexpr int DL = D / 32;
    float m[GM], l[GM], o[GM][DL];
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int j = 0; j < DL; ++j) o[g][j] = 0.f;
    }
    const int per = (bs + 15) / 16;  // groups of 16 rows of a page
    for (int i = warp; i < k * per; i += SPARSE_WARPS) {
        const int p = chosen[i / per], t0 = (i % per) * 16;
        const int b = row[p];
        if ((unsigned)b >= (unsigned)c.num_blocks) {
            if (lane == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, b);
            continue;
        }
        const int live = min(min(bs - t0, 16), len - (p * bs + t0));
        if (live <= 0) continue;
        const int64_t base = pool_row(c, a.layer, b, t0) + (int64_t)h * D;
        const int t = lane & 15, half = lane >> 4;
        const T* kr = reinterpret_cast<const T*>(c.k_pool) + base + (int64_t)min(t, live - 1) * H * D + half * (D / 2);
        const float* qh = qf + half * (D / 2);
        float s[GM];
#pragma unroll
        for (int g = 0; g < GM; ++g) s[g] = 0.f;
        constexpr int V = 16 / sizeof(T);
        for (int d = 0; d < D / 2; d += V) {
            alignas(16) T kv[V];
            *reinterpret_cast<uint4*>(kv) = *reinterpret_cast<const uint4*>(kr + d);
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                if (g >= G) break;
#pragma unroll
                for (int j = 0; j < V; ++j) s[g] = fmaf(Elem<T>::to_f(kv[j]), qh[g * D + d + j], s[g]);
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
        const T* vr = reinterpret_cast<const T*>(c.v_pool) + base + lane * DL;
        for (int t1 = 0; t1 < live; ++t1) {
            alignas(16) T vv[DL];
            *reinterpret_cast<Pack<T, DL>*>(vv) = *reinterpret_cast<const Pack<T, DL>*>(vr + (int64_t)t1 * H * D);
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                if (g >= G) break;
                const float w = __shfl_sync(0xffffffffu, s[g], t1);
#pragma unroll
                for (int j = 0; j < DL; ++j) o[g][j] = fmaf(w, Elem<T>::to_f(vv[j]), o[g][j]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        if (g >= G) break;
        if (lane == 0) {
            pm[warp * G + g] = m[g];
            pl[warp * G + g] = l[g];
        }
#pragma unroll
        for (int j = 0; j < DL; ++j) po[(warp * G + g) * D + lane * DL + j] = o[g][j];
    }
    __syncthreads();
    for (int i = tid; i < G * D; i += SPARSE_THREADS) {
        const int g = i / D;
        float mx = -INFINITY;
        for (int w = 0; w < SPARSE_WARPS; ++w) mx = fmaxf(mx, pm[w * G + g]);
        // a NaN score makes m NaN-free but l NaN; an empty sequence has no weight at all and gives zeros
        const float ref = mx == -INFINITY ? 0.f : mx;
        float ls = 0.f, os = 0.f;
        for (int w = 0; w < SPARSE_WARPS; ++w) {
            const float f = exp2f(pm[w * G + g] - ref);
            ls += pl[w * G + g] * f;
            os += po[(w * G) * D + i] * f;
        }
        out[i] = Elem<T>::from_f(P ? os / ls : 0.f);
    }
}

template <typename T, int D, int GM>
static int launch_sparse(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a, int n, cudaStream_t s) {
    const size_t smem = sparse_smem(a.cap, a.budget, a.G, D);
    if (smem > 200 * 1024) return MENTAT_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(k_sparse<T, D, GM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) !=
            cudaSuccess ||
        launch(pdl_enabled(), k_sparse<T, D, GM>, dim3(c->num_kv_heads, n), dim3(SPARSE_THREADS), smem, s, *c, *x, a) !=
            cudaSuccess) {
        (void)cudaGetLastError();
        return MENTAT_ERR_CUDA;
    }
    MENTAT_CHECK_LAUNCH();
    return MENTAT_OK;
}

template <typename T, int D>
static int launch_sparse_group(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a, int n,
                               cudaStream_t s) {
    if (a.G <= 2) return launch_sparse<T, D, 2>(c, x, a, n, s);
    if (a.G <= 4) return launch_sparse<T, D, 4>(c, x, a, n, s);
    if (a.G <= 8) return launch_sparse<T, D, 8>(c, x, a, n, s);
    return launch_sparse<T, D, 16>(c, x, a, n, s);
}

template <typename T>
static int launch_sparse_dim(const mentat_kv_cache* c, const mentat_page_index* x, const SparseArgs& a, int n,
                             cudaStream_t s) {
    if (c->head_dim == 128) return launch_sparse_group<T, 128>(c, x, a, n, s);
    if (c->head_dim == 64) return launch_sparse_group<T, 64>(c, x, a, n, s);
    return MENTAT_ERR_UNSUPPORTED;
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
    const dim3 grid(n, c->num_kv_heads), block((c->head_dim + 31) / 32 * 32);
    MENTAT_BY_DTYPE(MENTAT_LAUNCH(k_index_blocks<T>, grid, block, 0, s, *c, layer, blocks, *x))
    return MENTAT_OK;
}

int mentat_page_index_seqs(const mentat_kv_cache* c, int32_t layer, const int32_t* slots, int32_t n, int32_t first,
                           int32_t max_pages, const mentat_page_index* x, cudaStream_t s) {
    if (bad_index(c, x) || layer < -1 || layer >= c->num_layers || n < 0 || first < -1 || max_pages < 0 ||
        !c->tables || !c->ntok || c->num_layers > 65535 || (n > 0 && !slots) || (int64_t)n * max_pages > 0x7fffffff)
        return MENTAT_ERR_ARG;
    if (first < 0) max_pages = 1;
    if (n == 0 || max_pages == 0) return MENTAT_OK;
    const dim3 grid(n * max_pages, c->num_kv_heads, layer < 0 ? c->num_layers : 1), block((c->head_dim + 31) / 32 * 32);
    const int l0 = layer < 0 ? 0 : layer;
    MENTAT_BY_DTYPE(MENTAT_LAUNCH(k_index_seqs<T>, grid, block, 0, s, *c, l0, slots, first, *x, max_pages))
    return MENTAT_OK;
}

int mentat_page_bounds(const mentat_kv_cache* c, int32_t layer, const int32_t* blocks, int32_t n,
                       const mentat_page_index* x, float* low, float* high, int8_t* exps, cudaStream_t s) {
    if (bad_index(c, x) || layer < 0 || layer >= c->num_layers || n < 0 || (n > 0 && (!blocks || !low || !high || !exps)))
        return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    MENTAT_LAUNCH(k_page_bounds, dim3(n, c->num_kv_heads), dim3(128), 0, s, *c, layer, blocks, *x, low, high, exps);
    return MENTAT_OK;
}

int mentat_sparse_decode(const mentat_kv_cache* c, int32_t layer, const mentat_page_index* x, const int32_t* slots,
                         int32_t n, const void* q, int64_t q_stride, int32_t Hq, void* out, int64_t out_stride,
                         float scale, int32_t max_len, int32_t budget, int32_t sink, int32_t recent, int32_t* pages,
                         cudaStream_t s) {
    if (bad_index(c, x) || layer < 0 || layer >= c->num_layers || n < 0 || n > 65535 || Hq <= 0 ||
        Hq % c->num_kv_heads || max_len < 0 || !(scale > 0.f) || sink < 0 || recent < 1 || budget < 1 ||
        (int64_t)sink + recent > budget || !c->v_pool || !c->tables || !c->ntok ||
        (n > 0 && (!slots || !q || !out)) || (((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) & 15))
        return MENTAT_ERR_ARG;
    const int G = Hq / c->num_kv_heads;
    if (G > SPARSE_MAX_GROUP || budget > SPARSE_MAX_BUDGET) return MENTAT_ERR_UNSUPPORTED;
    if (n == 0) return MENTAT_OK;
    const int cap = (int)(((int64_t)max_len + c->block_size - 1) / c->block_size);
    const SparseArgs a{slots, q, q_stride, out, out_stride, pages, scale * 1.4426950408889634f, layer, G,
                       max_len, cap, budget, sink, recent};
    int st = MENTAT_OK;
    MENTAT_BY_DTYPE(st = launch_sparse_dim<T>(c, x, a, n, s))
    return st;
}

}  // extern "C"
