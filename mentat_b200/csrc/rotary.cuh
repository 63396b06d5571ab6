// Rotary positions: device helpers shared by the stateless entry points
// (rotary.cu) and the appends (kv_cache.cu).
//
// Pair i of a token at position p is turned by p * inv_freq[i]: (x1, x2) ->
// scale * (x1 cos - x2 sin, x1 sin + x2 cos).  The angle is taken in turns,
// p * (inv_freq / 2 pi), as a sum of two doubles: one double would know 2^60 turns to 2^7 of
// a turn, and 2^17 (p = 2^20 at one radian per position) to 2^-35.  The factor
// 1 / 2 pi and its product with inv_freq have an error of 2^-104 of themselves, the products
// with p leave their rounding in a fused multiply-add, and whole turns are dropped
// before the parts are added.  So the fraction of a turn is off by less than 2^-42 for every int64
// position and every inv_freq up to one radian.  It goes to the float sincospif as the nearest float;
// what that leaves (up to 2^-26 of a turn) is added to first order, the second being below 2^-47.
// Products and sums are float, one rounding to the element type at the end.
#pragma once

#include "common.cuh"

namespace mentat {

constexpr int ROTARY_THREADS = 128;   // most threads that share a token
constexpr int ROTARY_MAX_DIM = 1024;  // largest head_dim of the rotary entry points

// p * (fh + fl) without whole turns; p exact
__device__ __forceinline__ double rotary_turns(double p, double fh, double fl) {
    const double a = __dmul_rn(p, fh);  // rounded: not to be fused with the difference
    return (a - rint(a)) + fma(p, fl, fma(p, fh, -a));
}
__device__ __forceinline__ void rotary_angle(const mentat_rotary& r, int i, int64_t pos, float* c, float* s) {
    constexpr double H = 0.15915494309189535, L = -9.839338337591243e-18;  // 1 / 2 pi
    const double f = r.inv_freq[i], fh = __dmul_rn(f, H), fl = fma(f, L, fma(f, H, -fh));
    double t = rotary_turns((double)(uint32_t)pos, fh, fl);
    const int high = (int)(pos >> 32);
    if (high) t += rotary_turns((double)high * 4294967296.0, fh, fl);
    t -= rint(t);
    const float th = (float)t, d = 6.2831853f * (float)(t - (double)th);
    float sn, cs;
    sincospif(2.0f * th, &sn, &cs);
    *c = (cs - sn * d) * r.scale;
    const float turned = (sn + cs * d) * r.scale;
    *s = r.inverse ? -turned : turned;
}

// cos and sin of every pair of one token, to cs[0 .. pairs) and cs[pairs ..); the caller synchronises
__device__ __forceinline__ void rotary_table(const mentat_rotary& r, int64_t pos, float* cs) {
    for (int i = threadIdx.x; i < r.pairs; i += blockDim.x) rotary_angle(r, i, pos, cs + i, cs + r.pairs + i);
}

// The heads of one token, turned by the table, a CTA's threads over (head, task).
// VEC elements per access; VEC > 1 needs strides, offset, pairs (2 pairs if
// interleaved) and addresses that are multiples of VEC elements.  A task loads all it
// turns before it stores, and tasks are disjoint, so src may be dst.
template <typename T, int VEC, bool IL>
__device__ __forceinline__ void rotate_heads(const T* src, int64_t src_hs, T* dst, int64_t dst_hs, int heads, int D,
                                             const mentat_rotary& r, const float* cs) {
    using P = Pack<T, VEC>;
    const int pairs = r.pairs, off = r.offset;
    const float* sn = cs + pairs;
    if (IL && VEC > 1) {
        const int tasks = D / VEC;
        for (int x = threadIdx.x; x < heads * tasks; x += blockDim.x) {
            const int h = x / tasks, d = (x - h * tasks) * VEC;
            P a = *reinterpret_cast<const P*>(src + h * src_hs + d);
            if (d >= off && d < off + 2 * pairs) {
                const int i = (d - off) / 2;
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const float u = Elem<T>::to_f(a.v[2 * j]), w = Elem<T>::to_f(a.v[2 * j + 1]);
                    a.v[2 * j] = Elem<T>::from_f(u * cs[i + j] - w * sn[i + j]);
                    a.v[2 * j + 1] = Elem<T>::from_f(u * sn[i + j] + w * cs[i + j]);
                }
            }
            *reinterpret_cast<P*>(dst + h * dst_hs + d) = a;
        }
        return;
    }
    const int turned = pairs / VEC, tasks = turned + (D - 2 * pairs) / VEC;
    for (int x = threadIdx.x; x < heads * tasks; x += blockDim.x) {
        const int h = x / tasks, t = x - h * tasks;
        const T* s = src + h * src_hs;
        T* o = dst + h * dst_hs;
        if (t < turned) {
            const int i = t * VEC, d1 = off + (IL ? 2 * i : i), d2 = d1 + (IL ? 1 : pairs);
            P a = *reinterpret_cast<const P*>(s + d1), b = *reinterpret_cast<const P*>(s + d2);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float u = Elem<T>::to_f(a.v[j]), w = Elem<T>::to_f(b.v[j]);
                a.v[j] = Elem<T>::from_f(u * cs[i + j] - w * sn[i + j]);
                b.v[j] = Elem<T>::from_f(u * sn[i + j] + w * cs[i + j]);
            }
            *reinterpret_cast<P*>(o + d1) = a;
            *reinterpret_cast<P*>(o + d2) = b;
        } else {
            int d = (t - turned) * VEC;
            if (d >= off) d += 2 * pairs;
            *reinterpret_cast<P*>(o + d) = *reinterpret_cast<const P*>(s + d);
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void copy_heads(const T* src, int64_t src_hs, T* dst, int64_t dst_hs, int heads, int D) {
    using P = Pack<T, VEC>;
    const int tasks = D / VEC;
    for (int x = threadIdx.x; x < heads * tasks; x += blockDim.x) {
        const int h = x / tasks, d = (x - h * tasks) * VEC;
        *reinterpret_cast<P*>(dst + h * dst_hs + d) = *reinterpret_cast<const P*>(src + h * src_hs + d);
    }
}

// ---- host side ------------------------------------------------------------
static inline bool rows_ok(const mentat_rows* x, bool may_be_empty) {
    return x && (x->heads > 0 ? x->ptr != nullptr : x->heads == 0 && may_be_empty);
}
static inline bool rotary_ok(const mentat_rotary* r, int head_dim) {
    return r && r->inv_freq && r->pairs > 0 && r->offset >= 0 && head_dim > 0 && head_dim <= ROTARY_MAX_DIM &&
           r->pairs <= head_dim / 2 && r->offset <= head_dim - 2 * r->pairs;
}
// whether rows can be read and written `vec` elements at a time
static inline bool rows_aligned(const mentat_rows* x, int vec, int esz) {
    if (x->heads == 0) return true;
    return (reinterpret_cast<uintptr_t>(x->ptr) % (vec * esz)) == 0 && x->token_stride % vec == 0 &&
           (x->heads == 1 || x->head_stride % vec == 0);
}
static inline bool rotary_aligned(const mentat_rotary* r, int head_dim, int vec) {
    return head_dim % vec == 0 && r->offset % vec == 0 && (r->interleaved ? 2 * r->pairs : r->pairs) % vec == 0;
}

// Calls f.template operator()<T, VEC, IL>() for a dtype; VEC is one 16-byte access
// where alignment lets it, else single elements.
template <typename F>
static int rotary_dispatch(int dtype, bool vec, bool il, F&& f) {
    switch (dtype) {
#define MENTAT_ROTARY_CASE(code, T, V)                                                     \
    case code:                                                                             \
        if (vec) return il ? f.template operator()<T, V, true>() : f.template operator()<T, V, false>(); \
        return il ? f.template operator()<T, 1, true>() : f.template operator()<T, 1, false>();
        MENTAT_ROTARY_CASE(MENTAT_F32, float, 4)
        MENTAT_ROTARY_CASE(MENTAT_BF16, __nv_bfloat16, 8)
        MENTAT_ROTARY_CASE(MENTAT_F16, __half, 8)
#undef MENTAT_ROTARY_CASE
        default: return MENTAT_ERR_UNSUPPORTED;
    }
}

}  // namespace mentat
