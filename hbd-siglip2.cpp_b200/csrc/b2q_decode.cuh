// b2q_decode.cuh — what the decode kernels share: element types, the paged
// cache as a kernel sees it, and the check of a caller's cache description.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "b2q_internal.h"
#include "b2q_ptx.cuh"

namespace b2q {

inline bool ptr_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
// Arrays of 32-bit entries (null ones too).
template <class... P>
inline bool words(const P*... p) {
    return (ptr_aligned(p, 4) && ...);
}
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

// ---- warp-level tensor-core pieces -------------------------------------------
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// d += a (16 x 16, row) * b (16 x 8, column) with fp32 sums; T picks the operand type.
template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a * b in fp16 operands, sums from zero.
__device__ __forceinline__ void mma_16816_from0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Two floats rounded to a pair of T (x in the low half), and what the rounding left of them.
template <class T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
// 16 bytes to shared memory; zeros where !valid (gmem stays a readable address).
__device__ __forceinline__ void cp_async_16(uint32_t smem, const void* gmem, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16u : 0u)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The paged cache in a kernel.  Offsets are 64-bit: a cache passes 2^32
// elements long before it passes the GPU's memory.
template <class T>
struct CacheView {
    T* k;
    T* v;
    int64_t page_stride, head_stride, token_stride;
    int n_pages, page_shift, page_mask;
};

// Lets `kernel` use `bytes` of dynamic shared memory: once per device, `done` (one
// per kernel, device d its bit d) keeps the call off the launch path.
template <class Kernel>
inline b2q_status allow_smem(Kernel* kernel, int bytes, std::atomic<uint64_t>& done, int device) {
    const uint64_t bit = uint64_t(1) << device;
    if (done.load(std::memory_order_acquire) & bit) return B2Q_OK;
    const b2q_status st = cuda_check(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory of a kernel");
    if (!st) done.fetch_or(bit, std::memory_order_release);
    return st;
}

// ---- pairs of CTAs (clusters of two) ------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address of this shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster_128(uint32_t addr, uint4 v) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ void st_cluster_64(uint32_t addr, uint2 v) {
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void st_cluster_32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void max_cluster_32(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void or_cluster_32(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// All threads of the cluster; orders their shared-memory accesses.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- back-to-back launches ---------------------------------------------------
// The decode kernels are launched so that one may start while the one before it
// in the stream still runs (programmatic dependent launch): it lets its successor
// start (`let_next_start`) and waits for its predecessors' results
// (`wait_for_previous`) before it touches anything that they may read or write.
// What comes before that wait reads only its arguments and registered weights,
// which are complete when their registration returns.  A kernel launched any other
// way keeps its full order.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... Params, class... Args>
inline cudaError_t launch_after(int cluster, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                                cudaStream_t s, const Args&... args) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}
template <class... Params, class... Args>
inline cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                const Args&... args) {
    return launch_after(1, kernel, grid, block, smem, s, args...);
}

// B2Q_OK and the strides filled in, or the error of a bad description.
inline b2q_status check_cache(const b2q_kv_cache* in, b2q_kv_cache* c) {
    if (!in || !in->k || !in->v) return set_error(B2Q_ERR_INVALID, "null cache");
    *c = *in;
    if (c->dtype != B2Q_TYPE_F16 && c->dtype != B2Q_TYPE_BF16)
        return set_error(B2Q_ERR_INVALID, "the cache must be F16 or BF16");
    if (c->n_pages <= 0 || c->n_kv_head <= 0 || c->n_kv_head > 65535) return set_error(B2Q_ERR_SHAPE, "bad n_pages / n_kv_head");
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
