// b2q_decode.cuh — what the decode kernels share: element types, the paged
// cache as a kernel sees it, and the check of a caller's cache description.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "b2q_internal.h"
#include "b2q_ptx.cuh"

namespace b2q {

inline bool ptr_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int log2_of(int p) { return p <= 1 ? 0 : 1 + log2_of(p >> 1); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ void report(uint32_t* err, uint32_t code) { atomicCAS(err, 0u, code); }

// The paged cache in a kernel.  Offsets are 64-bit: a cache passes 2^32
// elements long before it passes the GPU's memory.
template <class T>
struct CacheView {
    T* k;
    T* v;
    int64_t page_stride, head_stride, token_stride;
    int n_pages, page_shift, page_mask;
};

// B2Q_OK and the strides filled in, or the error of a bad description.
inline b2q_status check_cache(const b2q_kv_cache* in, b2q_kv_cache* c) {
    if (!in || !in->k || !in->v) return set_error(B2Q_ERR_INVALID, "null cache");
    *c = *in;
    if (c->dtype != B2Q_TYPE_F16 && c->dtype != B2Q_TYPE_BF16)
        return set_error(B2Q_ERR_INVALID, "the cache must be F16 or BF16");
    if (c->n_pages <= 0 || c->n_kv_head <= 0) return set_error(B2Q_ERR_SHAPE, "bad n_pages / n_kv_head");
    if (c->page_size <= 0 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return set_error(B2Q_ERR_SHAPE, "page_size must be a power of two up to 1024");
    if (static_cast<int64_t>(c->n_pages) * c->page_size > INT32_MAX)
        return set_error(B2Q_ERR_SHAPE, "more cache slots than an int32 holds");
    if (c->d_head <= 0 || c->d_head > 256 || c->d_head % 8)
        return set_error(B2Q_ERR_SHAPE, "d_head must be a multiple of 8 up to 256");
    if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0)
        return set_error(B2Q_ERR_SHAPE, "cache strides must not be negative");
    if (!c->token_stride) c->token_stride = c->d_head;
    if (!c->head_stride) c->head_stride = static_cast<int64_t>(c->page_size) * c->d_head;
    if (!c->page_stride) c->page_stride = static_cast<int64_t>(c->n_kv_head) * c->page_size * c->d_head;
    if (c->token_stride < c->d_head) return set_error(B2Q_ERR_SHAPE, "token_stride smaller than d_head");
    if (c->token_stride % 8 || c->head_stride % 8 || c->page_stride % 8 || !ptr_aligned(c->k, 16) ||
        !ptr_aligned(c->v, 16))
        return set_error(B2Q_ERR_ALIGN, "cache rows need 16-byte alignment");
    return B2Q_OK;
}

template <class T>
inline CacheView<T> view_of(const b2q_kv_cache& c) {
    return {static_cast<T*>(c.k), static_cast<T*>(c.v), c.page_stride, c.head_stride, c.token_stride,
            c.n_pages,            log2_of(c.page_size), c.page_size - 1};
}

}  // namespace b2q
