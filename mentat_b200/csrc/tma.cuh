// mbarriers with bounded waits, TMA loads, and the tensor maps of a layer's pools.
#pragma once

#include <cuda.h>

#include <mutex>

#include "common.cuh"

namespace mentat {

constexpr long long TC_WAIT_CYCLES = 4000000000ll;  // ~2 s at 1.9 GHz

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// bounded wait: false once `limit` clock cycles have passed
__device__ __forceinline__ bool mbar_wait_for(uint32_t bar, uint32_t parity, long long limit) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (clock64() - t0 > limit) return false;
    }
    return true;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    return mbar_wait_for(bar, parity, TC_WAIT_CYCLES);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// bulk copy of `bytes` from this CTA's shared memory to global memory (no tensor map,
// no multicast); both addresses 16-byte aligned, bytes a multiple of 16
__device__ __forceinline__ void bulk_store(void* gdst, uint32_t ssrc, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gdst), "r"(ssrc), "r"(bytes)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// the bulk copies of this thread have read their shared-memory sources
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// the bulk copies of this thread have completed
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// bulk copy of `bytes` from global memory to this CTA's shared memory, counted by an mbarrier (same limits)
__device__ __forceinline__ void bulk_load(uint32_t sdst, const void* gsrc, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(sdst),
                 "l"(gsrc), "r"(bytes), "r"(bar)
                 : "memory");
}
// ---------------------------------------------------------------------------
// host: tensor maps of a layer's K and V pools (cached per pool and layer)
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

struct PoolMaps {
    const void* k_pool;
    const void* v_pool;
    int layer, num_blocks, block_size, kv_heads, head_dim, dtype, device;
    CUtensorMap mk, mv;
};

static bool make_pool_map(CUtensorMap* m, const mentat_kv_cache* c, const void* pool, int layer) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const int esz = dtype_bytes(c->dtype);
    const int64_t layer_bytes = (int64_t)c->num_blocks * c->block_size * c->num_kv_heads * c->head_dim * esz;
    void* base = (char*)pool + layer * layer_bytes;
    cuuint64_t dims[3] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->num_kv_heads,
                          (cuuint64_t)c->num_blocks * c->block_size};
    cuuint64_t strides[2] = {(cuuint64_t)c->head_dim * esz, (cuuint64_t)c->num_kv_heads * c->head_dim * esz};
    cuuint32_t box[3] = {64, 1, 16};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType dt =
        c->dtype == MENTAT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return fn(m, dt, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The maps of a layer's pools, encoded once for each pool, layer and layout (what they hold depends
// on nothing else); false if they cannot be encoded.  Callable from several threads.
static bool pool_maps(const mentat_kv_cache* c, int layer, CUtensorMap* mk, CUtensorMap* mv) {
    constexpr int CAP = 256;
    static std::mutex lock;
    static PoolMaps cache[CAP];
    static int used = 0, next = 0;
    const std::lock_guard<std::mutex> held(lock);
    int dev = 0;
    cudaGetDevice(&dev);
    int at = 0;
    while (at < used && !(cache[at].k_pool == c->k_pool && cache[at].v_pool == c->v_pool && cache[at].layer == layer &&
                          cache[at].num_blocks == c->num_blocks && cache[at].block_size == c->block_size &&
                          cache[at].kv_heads == c->num_kv_heads && cache[at].head_dim == c->head_dim &&
                          cache[at].dtype == c->dtype && cache[at].device == dev))
        ++at;
    if (at == used) {
        PoolMaps e;
        e.k_pool = c->k_pool;
        e.v_pool = c->v_pool;
        e.layer = layer;
        e.num_blocks = c->num_blocks;
        e.block_size = c->block_size;
        e.kv_heads = c->num_kv_heads;
        e.head_dim = c->head_dim;
        e.dtype = c->dtype;
        e.device = dev;
        if (!make_pool_map(&e.mk, c, c->k_pool, layer) || !make_pool_map(&e.mv, c, c->v_pool, layer)) return false;
        at = used < CAP ? used++ : (next++ % CAP);
        cache[at] = e;
    }
    *mk = cache[at].mk;
    *mv = cache[at].mv;
    return true;
}

}  // namespace mentat
