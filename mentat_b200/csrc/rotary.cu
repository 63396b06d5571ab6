// Rotary positions of q and k, to tensors or into rows of the paged cache.
//
// One CTA per token: the cosines and sines of its pairs are computed once into
// shared memory and serve every head of q and k.  The bound is memory: each row is
// read and written once.  8,192 tokens with 64 + 8 + 8 heads of 128 (336 MB): 58 us,
// 5.75 TB/s, with 128 threads; 65 us with 256 and 110 us with 512, whose CTAs leave
// more of a token's few microseconds (position, angles, barrier) uncovered.

#include "rotary.cuh"

namespace mentat {

struct RotaryArgs {
    mentat_rotary r;
    mentat_rows q, qo, k, ko, v;
    const int64_t* positions;
    const int64_t* rows;  // cache rows of k and v, or NULL: k goes to ko
    int D;
};

template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(ROTARY_THREADS) k_rotary(RotaryArgs a, mentat_kv_cache c, int layer) {
    extern __shared__ float cs[];
    griddep_wait();
    griddep_launch();
    const int64_t i = blockIdx.x;
    rotary_table(a.r, a.positions[i], cs);
    __syncthreads();
    if (a.q.heads)
        rotate_heads<T, VEC, IL>((const T*)a.q.ptr + i * a.q.token_stride, a.q.head_stride,
                                 (T*)a.qo.ptr + i * a.qo.token_stride, a.qo.head_stride, a.q.heads, a.D, a.r, cs);
    if (!a.k.heads) return;
    const T* k = (const T*)a.k.ptr + i * a.k.token_stride;
    if (!a.rows) {
        rotate_heads<T, VEC, IL>(k, a.k.head_stride, (T*)a.ko.ptr + i * a.ko.token_stride, a.ko.head_stride,
                                 a.k.heads, a.D, a.r, cs);
        return;
    }
    const int64_t row = a.rows[i];
    if (row == -1) return;
    if (row < 0 || row >= (int64_t)c.num_blocks * c.block_size) {
        if (threadIdx.x == 0) set_error(c, MENTAT_DEV_BAD_BLOCK, row < 0 ? row : row / c.block_size);
        return;
    }
    const int64_t at = pool_row(c, layer, 0, 0) + row * (int64_t)a.k.heads * a.D;
    rotate_heads<T, VEC, IL>(k, a.k.head_stride, (T*)c.k_pool + at, a.D, a.k.heads, a.D, a.r, cs);
    copy_heads<T, VEC>((const T*)a.v.ptr + i * a.v.token_stride, a.v.head_stride, (T*)c.v_pool + at, a.D, a.v.heads,
                       a.D);
}

struct LaunchRotary {
    const RotaryArgs& a;
    const mentat_kv_cache& c;
    int layer, n;
    cudaStream_t s;
    template <typename T, int VEC, bool IL>
    int operator()() {
        const int heads = a.q.heads + (a.rows ? 2 : 1) * a.k.heads;
        int threads = (heads * a.D / VEC + 31) / 32 * 32;
        threads = threads < 64 ? 64 : threads > ROTARY_THREADS ? ROTARY_THREADS : threads;
        MENTAT_LAUNCH(k_rotary<T, VEC, IL>, dim3(n), dim3(threads), 2 * a.r.pairs * sizeof(float), s, a, c, layer);
        return MENTAT_OK;
    }
};

}  // namespace mentat

using namespace mentat;

extern "C" {

int mentat_rotary_apply(int32_t dtype, int32_t D, int32_t n, const mentat_rows* q, const mentat_rows* qo,
                        const mentat_rows* k, const mentat_rows* ko, const int64_t* positions, const mentat_rotary* r,
                        cudaStream_t s) {
    if (n < 0 || !rotary_ok(r, D) || !rows_ok(q, true) || !rows_ok(k, true) || !rows_ok(qo, true) ||
        !rows_ok(ko, true) || qo->heads != q->heads || ko->heads != k->heads)
        return MENTAT_ERR_ARG;
    if (n == 0 || (!q->heads && !k->heads)) return MENTAT_OK;
    if (!positions) return MENTAT_ERR_ARG;
    RotaryArgs a{*r, *q, *qo, *k, *ko, {}, positions, nullptr, D};
    const int esz = dtype_bytes(dtype), vec = 16 / esz;
    const bool wide = rotary_aligned(r, D, vec) && rows_aligned(q, vec, esz) && rows_aligned(qo, vec, esz) &&
                      rows_aligned(k, vec, esz) && rows_aligned(ko, vec, esz);
    const mentat_kv_cache none{};
    return rotary_dispatch(dtype, wide, r->interleaved != 0, LaunchRotary{a, none, 0, n, s});
}

int mentat_rotary_append(const mentat_kv_cache* c, int32_t layer, int32_t n, const int64_t* rows, const mentat_rows* q,
                         const mentat_rows* qo, const mentat_rows* k, const mentat_rows* v, const int64_t* positions,
                         const mentat_rotary* r, cudaStream_t s) {
    if (!c || layer < 0 || layer >= c->num_layers || n < 0 || !c->k_pool || !c->v_pool || !c->ctrl) return MENTAT_ERR_ARG;
    const int D = c->head_dim;
    if (!rotary_ok(r, D) || !rows_ok(q, true) || !rows_ok(qo, true) || !rows_ok(k, false) ||
        !rows_ok(v, false) || qo->heads != q->heads || k->heads != c->num_kv_heads || v->heads != c->num_kv_heads)
        return MENTAT_ERR_ARG;
    if (n == 0) return MENTAT_OK;
    if (!positions || !rows) return MENTAT_ERR_ARG;
    RotaryArgs a{*r, *q, *qo, *k, {}, *v, positions, rows, D};
    const int esz = dtype_bytes(c->dtype), vec = 16 / esz;
    const bool wide = rotary_aligned(r, D, vec) && rows_aligned(q, vec, esz) && rows_aligned(qo, vec, esz) &&
                      rows_aligned(k, vec, esz) && rows_aligned(v, vec, esz) &&
                      ((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) % 16 == 0;
    return rotary_dispatch(c->dtype, wide, r->interleaved != 0, LaunchRotary{a, *c, layer, n, s});
}

}  // extern "C"
