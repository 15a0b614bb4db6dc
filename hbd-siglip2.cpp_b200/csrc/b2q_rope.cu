// b2q_rope.cu — RMS norm of query and key heads, rotation by position, and the
// keys' and values' way into the paged cache, in one pass (b2q_qk_norm_rope).
#include "b2q_decode.cuh"

namespace b2q {
namespace {

constexpr int kRopeWarps = 8;

template <class Tin, class Tc>
struct RopeArgs {
    const Tin* x;
    int64_t ld, n_rows;
    int n_head, n_kv, d, rot, interleaved, n_pos;
    float eps;
    const float *qw, *kw, *rope;
    const int32_t *pos, *slot;
    Tc* q;
    int64_t ldq;
    CacheView<Tc> c;
    int n_slots;
    uint32_t* err;
};

// One warp per (row, head); element d of the head in lane d % 32.
template <class Tin, class Tc>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_kernel(RopeArgs<Tin, Tc> a) {
    __shared__ float sx[kRopeWarps][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = a.n_head + 2 * a.n_kv;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kRopeWarps + warp;
    if (item >= a.n_rows * heads) return;
    const int64_t t = item / heads;
    const int h = static_cast<int>(item % heads);
    int pos = a.pos[t], slot = a.slot[t];
    const bool pad = pos == -1;
    if (!pad && a.rot && (pos < 0 || pos >= a.n_pos)) {
        if (lane == 0) report(a.err, kDevBadPosition);
        pos = 0;
        slot = -1;
    }
    if (slot < -1 || slot >= a.n_slots) {
        if (lane == 0) report(a.err, kDevBadPosition);
        slot = -1;
    }
    if (pad) slot = -1;
    Tc* dst;
    if (h < a.n_head) {
        dst = a.q + t * a.ldq + static_cast<int64_t>(h) * a.d;
    } else {
        if (slot < 0) return;
        const bool is_v = h >= a.n_head + a.n_kv;
        const int hk = h - a.n_head - (is_v ? a.n_kv : 0);
        dst = (is_v ? a.c.v : a.c.k) + (slot >> a.c.page_shift) * a.c.page_stride + hk * a.c.head_stride +
              (slot & a.c.page_mask) * a.c.token_stride;
    }
    const Tin* src = a.x + t * a.ld + static_cast<int64_t>(h) * a.d;
    float* x = sx[warp];
    float ss = 0.f;
    for (int i = lane; i < a.d; i += 32) {
        const float v = pad ? 0.f : to_f32(src[i]);
        x[i] = v;
        ss = fmaf(v, v, ss);
    }
    __syncwarp();
    const bool turned = h < a.n_head + a.n_kv && !pad;
    const float* w = h < a.n_head ? a.qw : a.kw;
    if (turned && w) {
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = 1.0f / sqrtf(ss / a.d + a.eps);
        for (int i = lane; i < a.d; i += 32) x[i] = x[i] * r * w[i];
        __syncwarp();
    }
    const int half = a.rot / 2;
    const float* cs = a.rope + static_cast<int64_t>(pad ? 0 : pos) * a.rot;
    for (int i = lane; i < a.d; i += 32) {
        float y = x[i];
        if (turned && i < a.rot) {
            const int p = a.interleaved ? i >> 1 : (i < half ? i : i - half);
            const bool second = a.interleaved ? (i & 1) : i >= half;
            const float other = x[a.interleaved ? i ^ 1 : (second ? i - half : i + half)];
            y = second ? y * cs[p] + other * cs[half + p] : y * cs[p] - other * cs[half + p];
        }
        dst[i] = from_f32<Tc>(y);
    }
}

template <class Tin, class Tc>
cudaError_t launch(const RopeArgs<Tin, Tc>& a, cudaStream_t s) {
    const int64_t items = a.n_rows * (a.n_head + 2 * a.n_kv);
    rope_kernel<Tin, Tc><<<static_cast<unsigned>((items + kRopeWarps - 1) / kRopeWarps), kRopeWarps * 32, 0, s>>>(a);
    count_launch();
    return cudaGetLastError();
}

}  // namespace
}  // namespace b2q

using namespace b2q;

extern "C" b2q_status b2q_qk_norm_rope(const void* qkv, int32_t dtype, int64_t ld, int64_t n_rows, int32_t n_head,
                                       const float* q_weight, const float* k_weight, float eps, const float* rope,
                                       int32_t n_pos, int32_t rot_dim, int32_t interleaved, const int32_t* pos,
                                       const int32_t* slot, void* q_out, int64_t ldq, const b2q_kv_cache* cache,
                                       void* stream) {
    B2Q_REQUIRE_STATE();
    b2q_kv_cache c;
    b2q_status st = check_cache(cache, &c);
    if (st) return st;
    if (dtype != B2Q_TYPE_F32 && dtype != B2Q_TYPE_F16 && dtype != B2Q_TYPE_BF16)
        return set_error(B2Q_ERR_INVALID, "rows must be F32, F16 or BF16");
    if (n_rows < 0 || n_rows > (1 << 30) || n_head <= 0 || n_head > 65535)
        return set_error(B2Q_ERR_SHAPE, "bad n_rows / n_head");
    const int64_t heads = n_head + 2 * static_cast<int64_t>(c.n_kv_head);
    if (ld < heads * c.d_head || ldq < static_cast<int64_t>(n_head) * c.d_head)
        return set_error(B2Q_ERR_SHAPE, "row strides shorter than the heads");
    if (rot_dim < 0 || rot_dim > c.d_head || rot_dim % 2) return set_error(B2Q_ERR_SHAPE, "bad rot_dim");
    if (rot_dim > 0 && n_pos <= 0) return set_error(B2Q_ERR_SHAPE, "bad n_pos");
    if (!(eps >= 0.f)) return set_error(B2Q_ERR_INVALID, "eps must not be negative");
    if (n_rows == 0) return B2Q_OK;
    if (!qkv || !pos || !slot || !q_out || (rot_dim > 0 && !rope)) return set_error(B2Q_ERR_INVALID, "null pointer");
    const size_t es = dtype == B2Q_TYPE_F32 ? 4 : 2;
    if (!ptr_aligned(qkv, es) || !ptr_aligned(q_out, 2)) return set_error(B2Q_ERR_ALIGN, "misaligned rows");
    if (n_rows * heads > (int64_t(1) << 33)) return set_error(B2Q_ERR_SHAPE, "too many heads in one call");
    auto go = [&](auto tin, auto tc) {
        using Tin = decltype(tin);
        using Tc = decltype(tc);
        RopeArgs<Tin, Tc> a{static_cast<const Tin*>(qkv), ld, n_rows, n_head, c.n_kv_head, c.d_head, rot_dim,
                            interleaved, n_pos, eps, q_weight, k_weight, rope, pos, slot, static_cast<Tc*>(q_out),
                            ldq, view_of<Tc>(c), c.n_pages * c.page_size, ds->err};
        return cuda_check(launch(a, static_cast<cudaStream_t>(stream)), "norm + rotation launch");
    };
    auto with_cache = [&](auto tin) {
        return c.dtype == B2Q_TYPE_F16 ? go(tin, __half{}) : go(tin, __nv_bfloat16{});
    };
    return dtype == B2Q_TYPE_F32   ? with_cache(float{})
           : dtype == B2Q_TYPE_F16 ? with_cache(__half{})
                                   : with_cache(__nv_bfloat16{});
}
