// b2q_rope.cu — RMS norm of query and key heads, rotation by position, and the
// keys' and values' way into the paged cache, in one pass (b2q_qk_norm_rope).
//
// Bound: bytes; every element is read and written once, about six operations
// apart.  Norm, rotation and the cache write in one pass because each of them
// alone would read and write the same bytes.
//
// A head belongs to a group of up to 32 lanes, each with two pieces of kVec
// elements: in the half-and-half pairing a piece and the one half a rotation
// further, so that a lane holds both elements of its pairs and the only exchange is
// the sum of squares.  A group takes two heads of its row, both loaded before the
// first is used; the row's position, slot and rotation values are fetched once for
// both.  Norm and pairing are compiled in and lanes without a piece read the first
// one's: instructions, not bytes, were the limit before (19 an element).
// Measured on one B200 (copy bandwidth 6.53 TB/s): 20,011 rows of 24 + 2 x 4 heads of
// 128, fp16, half rotated, 333 MB: 60 us, 5.54 TB/s (one head a group 67, four 69);
// 20,000 rows of 32 + 2 x 8 heads, bf16, normed and rotated, 502 MB: 100 us, 5.0 TB/s
// (141, 153); 20,000 rows of 48 heads of 72, fp32 in, normed and rotated, 421 MB: 119
// us, 3.5 TB/s (pieces of 4 instead of 12: 146); 256 rows: 2.8 us, the launch.
#include "b2q_decode.cuh"

#include <type_traits>

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

// A row's position and slot, checked; pad: a padding row.
struct RowPlace {
    int pos, slot;
    bool pad;
};
template <class Tin, class Tc>
__device__ __forceinline__ RowPlace place_of(const RopeArgs<Tin, Tc>& a, int64_t t, bool reports) {
    RowPlace o{a.pos[t], a.slot[t], false};
    o.pad = o.pos == -1;
    if (!o.pad && a.rot && (o.pos < 0 || o.pos >= a.n_pos)) {
        if (reports) report(a.err, kDevBadPosition);
        o.pos = 0;
        o.slot = -1;
    }
    if (o.slot < -1 || o.slot >= a.n_slots) {
        if (reports) report(a.err, kDevBadPosition);
        o.slot = -1;
    }
    if (o.pad) {
        o.pos = 0;
        o.slot = -1;
    }
    return o;
}

// kVec elements in 16-byte accesses, or 8-byte ones where they are not a multiple
template <class T, int kVec>
struct Piece {
    static constexpr int kWords = kVec * sizeof(T) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWords / 2; ++i) {
                const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p) + i);
                w[2 * i] = v.x, w[2 * i + 1] = v.y;
            }
        }
    }
    __device__ __forceinline__ void get(float (&x)[kVec]) const {
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
            float2 f;
            if constexpr (sizeof(T) == 4) f = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            else f = unpack2<T>(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
};
template <class T, int kVec>
__device__ __forceinline__ void store_piece(T* p, const float (&x)[kVec]) {
    uint32_t w[kVec / 2];
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    if constexpr (kVec == 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < kVec / 4; ++i) reinterpret_cast<uint2*>(p)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
    }
}
template <int kN>
__device__ __forceinline__ void load_f32(const float* p, float (&x)[kN]) {
    if constexpr (kN % 4) {
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) {
            const float2 v = __ldg(reinterpret_cast<const float2*>(p) + i);
            x[2 * i] = v.x, x[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN / 4; ++i) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
    }
}

// Block (lanes of a group, groups of a row, rows), grid (rows, runs of heads).
// Lane s of a group holds pieces s and s + half/kVec of the rotated part, the lanes
// after those two neighbouring pieces each of what is left.
template <class Tin, class Tc, int kVec, int kHeads, bool kNorm, bool kInter>
__global__ void __launch_bounds__(256, kHeads == 2 ? 4 : 1) rope_kernel(RopeArgs<Tin, Tc> a) {
    const int group = blockDim.x, s = threadIdx.x, heads = a.n_head + 2 * a.n_kv, n_turned = a.n_head + a.n_kv;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.z + threadIdx.z;
    const int step = blockDim.y, h0 = blockIdx.y * step * kHeads + threadIdx.y;
    const bool live = t < a.n_rows;
    const int pieces = a.d / kVec, paired = kInter ? 0 : a.rot / (2 * kVec);
    int pa = s < paired ? s : 2 * s, pb = s < paired ? s + paired : 2 * s + 1;   // (2 paired + 2 (s - paired))
    const bool has_a = pa < pieces, has_b = pb < pieces;   // a lane without a piece reads the first and stores none
    if (!has_a) pa = 0;
    if (!has_b) pb = 0;
    let_next_start();
    wait_for_previous();
    Piece<Tin, kVec> ra[kHeads], rb[kHeads];
    const Tin* src = a.x + (live ? t : a.n_rows - 1) * a.ld;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        const Tin* p = src + min(h0 + k * step, heads - 1) * a.d;
        ra[k].load(p + pa * kVec);
        rb[k].load(p + pb * kVec);
    }
    const RowPlace o = live ? place_of(a, t, s == 0 && h0 == 0) : RowPlace{0, -1, true};
    // this lane's rotation values: of piece a and b in the interleaved pairing, of their pairs in the other;
    // (1, 0) where nothing turns
    const float* cs = a.rope + static_cast<int64_t>(o.pos) * a.rot;
    const int half = a.rot / 2;
    float c[kVec], sn[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        c[i] = 1.f;
        sn[i] = 0.f;
    }
    if constexpr (kInter) {
        constexpr int kHalf = kVec / 2;
        float u[kHalf];
        if (pa * kVec < a.rot) {
            load_f32(cs + pa * kHalf, u);
#pragma unroll
            for (int i = 0; i < kHalf; ++i) c[i] = u[i];
            load_f32(cs + half + pa * kHalf, u);
#pragma unroll
            for (int i = 0; i < kHalf; ++i) sn[i] = u[i];
        }
        if (pb * kVec < a.rot) {
            load_f32(cs + pb * kHalf, u);
#pragma unroll
            for (int i = 0; i < kHalf; ++i) c[kHalf + i] = u[i];
            load_f32(cs + half + pb * kHalf, u);
#pragma unroll
            for (int i = 0; i < kHalf; ++i) sn[kHalf + i] = u[i];
        }
    } else if (s < paired) {
        load_f32(cs + pa * kVec, c);
        load_f32(cs + half + pa * kVec, sn);
    }
    const int64_t cache_row = (o.slot >> a.c.page_shift) * a.c.page_stride + (o.slot & a.c.page_mask) * a.c.token_stride;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * step;
        float xa[kVec], xb[kVec];
        ra[k].get(xa);
        rb[k].get(xb);
        if constexpr (kNorm) {   // (every lane takes part in the sum)
            float sa = 0.f, sb = 0.f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                sa = fmaf(xa[i], xa[i], sa);
                sb = fmaf(xb[i], xb[i], sb);
            }
            float ss = (has_a ? sa : 0.f) + (has_b ? sb : 0.f);
            for (int x = group >> 1; x; x >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, x);
            const float* w = h < a.n_head ? a.qw : a.kw;
            if (h < n_turned && w) {
                const float r = 1.0f / sqrtf(ss / a.d + a.eps);
                float v[kVec];
                load_f32(w + pa * kVec, v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) xa[i] = xa[i] * r * v[i];
                load_f32(w + pb * kVec, v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) xb[i] = xb[i] * r * v[i];
            }
        }
        if (!live || h >= heads) continue;
        Tc* dst;
        if (h < a.n_head) {
            dst = a.q + t * a.ldq + h * a.d;
        } else {
            if (o.slot < 0) continue;
            dst = h < n_turned ? a.c.k + (h - a.n_head) * a.c.head_stride : a.c.v + (h - n_turned) * a.c.head_stride;
            dst += cache_row;
        }
        if (h < n_turned) {
            if constexpr (kInter) {
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) {
                    float u = xa[2 * i], v = xa[2 * i + 1];
                    xa[2 * i] = u * c[i] - v * sn[i];
                    xa[2 * i + 1] = v * c[i] + u * sn[i];
                    u = xb[2 * i], v = xb[2 * i + 1];
                    xb[2 * i] = u * c[kVec / 2 + i] - v * sn[kVec / 2 + i];
                    xb[2 * i + 1] = v * c[kVec / 2 + i] + u * sn[kVec / 2 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float u = xa[i], v = xb[i];
                    xa[i] = u * c[i] - v * sn[i];
                    xb[i] = v * c[i] + u * sn[i];
                }
            }
            if (o.pad) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) xa[i] = xb[i] = 0.f;
            }
        }
        if (has_a) store_piece<Tc, kVec>(dst + pa * kVec, xa);
        if (has_b) store_piece<Tc, kVec>(dst + pb * kVec, xb);
    }
}

// Any alignment and any even rotation: one warp per (row, head), element d of the
// head in lane d % 32.
template <class Tin, class Tc>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_any_kernel(RopeArgs<Tin, Tc> a) {
    __shared__ float sx[kRopeWarps][256];
    let_next_start();
    wait_for_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = a.n_head + 2 * a.n_kv;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kRopeWarps + warp;
    if (item >= a.n_rows * heads) return;
    const int64_t t = item / heads;
    const int h = static_cast<int>(item % heads);
    const RowPlace o = place_of(a, t, lane == 0);
    Tc* dst;
    if (h < a.n_head) {
        dst = a.q + t * a.ldq + static_cast<int64_t>(h) * a.d;
    } else {
        if (o.slot < 0) return;
        const bool is_v = h >= a.n_head + a.n_kv;
        dst = (is_v ? a.c.v + (h - a.n_head - a.n_kv) * a.c.head_stride : a.c.k + (h - a.n_head) * a.c.head_stride) +
              (o.slot >> a.c.page_shift) * a.c.page_stride + (o.slot & a.c.page_mask) * a.c.token_stride;
    }
    const Tin* src = a.x + t * a.ld + static_cast<int64_t>(h) * a.d;
    float* x = sx[warp];
    float ss = 0.f;
    for (int i = lane; i < a.d; i += 32) {
        const float v = o.pad ? 0.f : to_f32(src[i]);
        x[i] = v;
        ss = fmaf(v, v, ss);
    }
    __syncwarp();
    const bool turned = h < a.n_head + a.n_kv && !o.pad;
    const float* w = h < a.n_head ? a.qw : a.kw;
    if (turned && w) {
        for (int k = 16; k; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
        const float r = 1.0f / sqrtf(ss / a.d + a.eps);
        for (int i = lane; i < a.d; i += 32) x[i] = x[i] * r * w[i];
        __syncwarp();
    }
    const int half = a.rot / 2;
    const float* cs = a.rope + static_cast<int64_t>(o.pos) * a.rot;
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

// Pieces of 8 elements where every row, cache row and rotation half is made of
// whole aligned ones, else of 12 or of 4 where that holds for them (halves of 36, in
// heads of 72: three of four lanes at work instead of nine of sixteen), else the
// element-wise kernel.
template <class Tin, class Tc>
cudaError_t launch(const RopeArgs<Tin, Tc>& a, cudaStream_t s) {
    const int64_t items = a.n_rows * (a.n_head + 2 * a.n_kv);
    auto fits = [&](int vec) {
        const size_t in = vec * sizeof(Tin) % 16 ? 8 : 16, out = vec * 2 % 16 ? 8 : 16;
        const int unit = a.interleaved ? vec : 2 * vec;
        return a.d % vec == 0 && a.rot % unit == 0 && a.d / vec <= 64 && ptr_aligned(a.x, in) && a.ld * sizeof(Tin) % in == 0 &&
               ptr_aligned(a.q, out) && a.ldq * 2 % out == 0 && ptr_aligned(a.qw, 16) && ptr_aligned(a.kw, 16) &&
               ptr_aligned(a.rope, 16);
    };
    const int heads = a.n_head + 2 * a.n_kv;
    auto go = [&](auto vec) {
        constexpr int kVec = decltype(vec)::value;
        const int pieces = a.d / kVec, paired = a.interleaved ? 0 : a.rot / (2 * kVec);
        const int lanes = paired + (pieces - 2 * paired + 1) / 2;
        int group = 1;
        while (group < lanes) group *= 2;
        auto with = [&](auto n_heads, auto norm, auto inter) {
            constexpr int kHeads = decltype(n_heads)::value;
            // whole warps: 32 / group rows, and at most 8 groups a row; as few runs of heads as that allows
            const int runs = (heads + 8 * kHeads - 1) / (8 * kHeads);
            const int groups = (heads + runs * kHeads - 1) / (runs * kHeads);
            const dim3 block(group, groups, 32 / group);
            const dim3 grid(static_cast<unsigned>((a.n_rows + block.z - 1) / block.z), runs);
            return launch_after(rope_kernel<Tin, Tc, kVec, kHeads, decltype(norm)::value, decltype(inter)::value>, grid,
                                block, 0, s, a);
        };
        auto with_heads = [&](auto norm, auto inter) {
            // two heads a group once the lanes fill the GPU (half a million); one waits less
            if constexpr (kVec <= 8)   // (pieces of 12 fill the registers with one)
                if (items * group >= (1 << 19)) return with(std::integral_constant<int, 2>{}, norm, inter);
            return with(std::integral_constant<int, 1>{}, norm, inter);
        };
        auto with_norm = [&](auto inter) {
            return a.qw || a.kw ? with_heads(std::true_type{}, inter) : with_heads(std::false_type{}, inter);
        };
        return a.interleaved ? with_norm(std::true_type{}) : with_norm(std::false_type{});
    };
    if (fits(8)) return go(std::integral_constant<int, 8>{});
    if (fits(12)) return go(std::integral_constant<int, 12>{});
    if (fits(4)) return go(std::integral_constant<int, 4>{});
    return launch_after(rope_any_kernel<Tin, Tc>, dim3(static_cast<unsigned>((items + kRopeWarps - 1) / kRopeWarps)),
                        dim3(kRopeWarps * 32), 0, s, a);
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
    if (!words(q_weight, k_weight, rope, pos, slot)) return set_error(B2Q_ERR_ALIGN, "misaligned array");
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
