// b2q_q4.cu — products of few activation rows with ggml Q4_0 / Q4_1 weights
// (b2q_weight_q4_*, b2q_mul_vec_q4).
//
// y[n] = sum_kb d[n,kb] S[n,kb] (+ m[n,kb] X[kb]), S the sum of (q - 8) x (Q4_1:
// q x) over the 32 columns of block kb, X that of x.
//
// Bound: bytes, 18 (20) per 32 weights and at most once.  At the measured copy
// rate that is 11.6 T weights/s, and the SMs issue about 36 T lane operations/s:
// three instructions a weight for everything.  Unpacking alone takes more than
// one, so even a single activation row goes to the tensor cores: mma.sync
// (16 weight rows x 16 columns x 8 activation columns) does 8 of a lane's
// products in one instruction and sums in fp32.
//
//  * The nibbles become exact 16-bit integers: OR-ed into the mantissa of 2^7
//    (bf16) or 2^10 (fp16), the power and the 8 subtracted again.
//  * fp16 and bf16 activations are operands as they are.  An fp32 activation
//    is the exact sum of three bf16 values (8 bits of its mantissa each), which
//    take three of the eight activation columns: with one row they are free.
//  * S leaves the tensor core once per block, is scaled by the fp32 value of d
//    and summed in fp32, so nothing is rounded to 16 bits on the way.
//
// The weights are laid out at registration in the order the lanes want them:
// per 16 rows a run of units of 64 columns, each 512 bytes of nibbles (lane l of
// the warp: 16 bytes) and the blocks' scales (64 bytes; Q4_1: 64 more for m).  A
// warp streams units through a ring of asynchronous copies that runs on across
// row tiles; the activations sit in shared memory for the whole launch (grid:
// one CTA of 16 warps per SM).  kSplit warps share a row tile, each taking every
// kSplit-th unit, and add up in a fixed order.
#include "b2q_decode.cuh"

#include <new>
#include <type_traits>

struct b2q_weight_q4 {
    int64_t N = 0, K = 0;
    int type = 0, device = -1;
    int64_t tiles = 0, units = 0;   // of 16 rows; of 64 columns per row tile
    uint8_t* packed = nullptr;      // [tiles][units][576 or 640 bytes]
};

namespace b2q {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxK = 28672;        // three bf16 pieces of a row still fit shared memory next to the rings
constexpr int kSmemMax = 227 * 1024 - 1024;

constexpr int unit_bytes(bool min) { return min ? 640 : 576; }

// ------------------------------------------------------------------ layout
// Lane l = 4 g + t of a unit holds, for each of its two blocks, the columns
// 8 t .. 8 t + 7 of rows g and g + 8: one 32-bit word each, column 2 j in the
// nibble at bit 4 j and column 2 j + 1 in that at bit 16 + 4 j, so that shifting
// by 4 j and masking yields the operand pair (2 j, 2 j + 1).
__global__ void pack_q4_kernel(const uint8_t* __restrict__ raw, int64_t N, int64_t Kb, int64_t row_bytes, bool min,
                               int64_t tiles, int64_t units, uint8_t* __restrict__ out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;   // one lane of one unit
    if (i >= tiles * units * 32) return;
    const int l = static_cast<int>(i & 31), g = l >> 2, t = l & 3;
    const int64_t unit = (i >> 5) % units, tile = (i >> 5) / units;
    uint8_t* dst = out + (i >> 5) * unit_bytes(min);
    uint32_t w[4];
    for (int x = 0; x < 4; ++x) {
        const int64_t n = tile * 16 + g + 8 * (x & 1), kb = unit * 2 + (x >> 1);
        w[x] = 0;
        uint16_t d = 0, m = 0;
        if (n < N && kb < Kb) {
            const uint8_t* b = raw + n * row_bytes + kb * (min ? 20 : 18);
            const uint8_t* q = b + (min ? 4 : 2);
            for (int e = 0; e < 8; ++e) {
                const int k = 8 * t + e;
                const uint32_t v = (q[k & 15] >> (k < 16 ? 0 : 4)) & 15u;
                w[x] |= v << (4 * (e >> 1) + 16 * (e & 1));
            }
            d = static_cast<uint16_t>(b[0] | (b[1] << 8));
            if (min) m = static_cast<uint16_t>(b[2] | (b[3] << 8));
        }
        if (t == 0) {
            reinterpret_cast<uint16_t*>(dst + 512 + g * 8)[x] = d;
            if (min) reinterpret_cast<uint16_t*>(dst + 576 + g * 8)[x] = m;
        }
    }
    *reinterpret_cast<uint4*>(dst + l * 16) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------ product
template <class Tx>
struct Q4Args {
    const uint8_t* w;
    int64_t N;
    int tiles, units, split;
    const Tx* x;
    int rows;               // activation rows of this launch
    int64_t x_cols, ldx;
    void* y;
    int64_t ldy;
    bool y_f32;
    const float *bias, *residual;
    int pitch, ring_at, red_at, sum_at;   // shared memory: row of an activation column, parts' offsets (bytes)
};

// The word's four pairs as exact integers q - 8 (Q4_1: q).
template <class T, bool kMin>
__device__ __forceinline__ void unpack_q4(uint32_t w, uint32_t (&r)[4]);
#define B2Q_UNPACK_BF16(kMin)                                                                             \
    template <>                                                                                           \
    __device__ __forceinline__ void unpack_q4<__nv_bfloat16, kMin>(uint32_t w, uint32_t (&r)[4]) {        \
        const __nv_bfloat162 off = __floats2bfloat162_rn(kMin ? -128.f : -136.f, kMin ? -128.f : -136.f); \
        _Pragma("unroll") for (int j = 0; j < 4; ++j) {                                                   \
            const uint32_t u = ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;                              \
            const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);          \
            r[j] = *reinterpret_cast<const uint32_t*>(&v);                                                \
        }                                                                                                 \
    }
B2Q_UNPACK_BF16(false)
B2Q_UNPACK_BF16(true)
#undef B2Q_UNPACK_BF16
// fp16 has room for a nibble at bit 4 as well (1024 + 16 q, scaled back in the
// multiply-add), which saves two of the three shifts.
#define B2Q_UNPACK_F16(kMin)                                                                      \
    template <>                                                                                   \
    __device__ __forceinline__ void unpack_q4<__half, kMin>(uint32_t w, uint32_t (&r)[4]) {       \
        const __half2 off = __float2half2_rn(kMin ? -1024.f : -1032.f);                           \
        const __half2 off16 = __float2half2_rn(kMin ? -64.f : -72.f), s16 = __float2half2_rn(0.0625f); \
        _Pragma("unroll") for (int j = 0; j < 4; j += 2) {                                        \
            const uint32_t s = w >> (4 * j);                                                      \
            const uint32_t u = (s & 0x000F000Fu) | 0x64006400u, v = (s & 0x00F000F0u) | 0x64006400u; \
            const __half2 a = __hadd2(*reinterpret_cast<const __half2*>(&u), off);                \
            const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&v), s16, off16);         \
            r[j] = *reinterpret_cast<const uint32_t*>(&a);                                        \
            r[j + 1] = *reinterpret_cast<const uint32_t*>(&b);                                    \
        }                                                                                         \
    }
B2Q_UNPACK_F16(false)
B2Q_UNPACK_F16(true)
#undef B2Q_UNPACK_F16

// The leading 8 bits of x's mantissa (cut, so that what is left is exact and a
// large x does not become infinite); infinities and NaN stay what they are.
__device__ __forceinline__ float lead_bf16(float x) {
    const uint32_t u = __float_as_uint(x) & 0xFFFF0000u;
    return x != x ? x : __uint_as_float(u);
}
__device__ __forceinline__ float finite_or_0(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.f; }
__device__ __forceinline__ uint32_t cut_pair(float x, float y) {
    const uint32_t a = x != x ? 0x7FC0u : __float_as_uint(x) >> 16, b = y != y ? 0x7FC0u : __float_as_uint(y) >> 16;
    return a | (b << 16);
}

// Activation rows into shared memory: per row its operand columns (fp32: three
// bf16 pieces), and for Q4_1 the sums over each block.
template <class Tx, bool kMin>
__device__ __forceinline__ void stage_x(const Q4Args<Tx>& a, uint8_t* smem) {
    constexpr int kPieces = std::is_same<Tx, float>::value ? 3 : 1;
    const int chunks = a.units * 8;   // of 8 columns
    const int total = a.rows * chunks;
    const bool vec = (a.ldx * sizeof(Tx)) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    for (int base = 0; base < total; base += kThreads) {
        const int i = base + threadIdx.x;
        const bool in = i < total;
        const int m = in ? i / chunks : 0, c = in ? i % chunks : 0;
        const Tx* x = a.x + m * a.ldx + c * 8;
        const int64_t left = in ? a.x_cols - c * 8 : 0;
        Tx v[8];
        if (vec && left >= 8) {
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(Tx)) / 2; ++j)
                reinterpret_cast<uint4*>(v)[j] = reinterpret_cast<const uint4*>(x)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? x[j] : from_f32<Tx>(0.f);
        }
        uint8_t* dst = smem + m * kPieces * a.pitch + c * 16;
        if (in) {
            if constexpr (kPieces == 1) {
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
            } else {
                uint32_t p[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float e[2] = {v[2 * j], v[2 * j + 1]}, h[3][2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        h[0][z] = lead_bf16(e[z]);
                        const float r = finite_or_0(e[z] - h[0][z]);
                        h[1][z] = lead_bf16(r);
                        h[2][z] = r - h[1][z];
                    }
#pragma unroll
                    for (int q = 0; q < 3; ++q) p[q][j] = cut_pair(h[q][0], h[q][1]);
                }
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    *reinterpret_cast<uint4*>(dst + q * a.pitch) = make_uint4(p[q][0], p[q][1], p[q][2], p[q][3]);
            }
        }
        if constexpr (kMin) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s += to_f32(v[j]);
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            if (in && (c & 3) == 0) reinterpret_cast<float*>(smem + a.sum_at)[(c >> 2) * a.rows + m] = s;
        }
    }
}

template <class Tx, bool kMin, int kN, int kStages>
__global__ void __launch_bounds__(kThreads, 1) mul_vec_q4_kernel(Q4Args<Tx> a) {
    using T = typename std::conditional<std::is_same<Tx, float>::value, __nv_bfloat16, Tx>::type;
    constexpr int kPieces = std::is_same<Tx, float>::value ? 3 : 1;
    constexpr int kUnit = unit_bytes(kMin);
    constexpr int kRedPitch = 8 * kN + 1, kRedWarp = 16 * kRedPitch + 1;   // odd: no bank conflicts either way
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = a.split, sub = warp % split, group = warp / split, groups = kWarps / split;
    const int first = blockIdx.x * groups + group, step = gridDim.x * groups;
    const int per_tile = (a.units - sub + split - 1) / split;   // units of this warp in each of its tiles

    // ---- the weights' stream: unit `u` of tile `lt`, kStages - 1 units ahead ----
    const uint32_t ring = smem_u32(smem + a.ring_at) + warp * kStages * kUnit;
    const uint8_t* src = a.w;
    int lt = first, lu = sub, slot = 0;
    auto issue = [&]() {
        if (lt < a.tiles) {
            const uint8_t* p = src + (static_cast<int64_t>(lt) * a.units + lu) * kUnit + lane * 16;
            const uint32_t dst = ring + slot * kUnit + lane * 16;
            cp_async_16(dst, p, true);
            if (lane < (kUnit - 512) / 16) cp_async_16(dst + 512, p + 512, true);
            lu += split;
            if (lu >= a.units) {
                lu = sub;
                lt += step;
            }
        }
        cp_commit();
        slot = slot + 1 == kStages ? 0 : slot + 1;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();
    stage_x<Tx, kMin>(a, smem);
    __syncthreads();

    // this lane's operand columns and, for Q4_1, the sums that its outputs take
    const int cols = a.rows * kPieces;
    const float* sums = reinterpret_cast<const float*>(smem + a.sum_at);
    uint32_t xb[kN];
    bool has[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        has[n] = n * 8 + g < cols;
        xb[n] = smem_u32(smem) + (has[n] ? n * 8 + g : 0) * a.pitch + t * 16;
    }
    int out_slot = 0;
    for (int tile = first; tile < a.tiles; tile += step) {
        float acc[kN][4] = {};
        int u = sub;
        for (int j = 0; j < per_tile; ++j, u += split) {
            issue();
            cp_wait<kStages - 1>();
            __syncwarp();
            const uint32_t at = ring + out_slot * kUnit;
            out_slot = out_slot + 1 == kStages ? 0 : out_slot + 1;
            const uint4 w4 = lds_128(at + lane * 16);
            const uint2 d4 = lds_64(at + 512 + g * 8);
            uint2 m4 = make_uint2(0, 0);
            if constexpr (kMin) m4 = lds_64(at + 576 + g * 8);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t lo[4], hi[4];
                unpack_q4<T, kMin>(b ? w4.z : w4.x, lo);
                unpack_q4<T, kMin>(b ? w4.w : w4.y, hi);
                const float2 d = unpack2<__half>(b ? d4.y : d4.x);
                const float2 mn = unpack2<__half>(b ? m4.y : m4.x);
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    uint4 x4 = make_uint4(0, 0, 0, 0);
                    if (has[n]) x4 = lds_128(xb[n] + (2 * u + b) * 64);
                    float s[4];
                    mma_16816_from0<T>(s, lo[0], hi[0], lo[1], hi[1], x4.x, x4.y);
                    mma_16816<T>(s, lo[2], hi[2], lo[3], hi[3], x4.z, x4.w);
                    acc[n][0] = fmaf(d.x, s[0], acc[n][0]);
                    acc[n][1] = fmaf(d.x, s[1], acc[n][1]);
                    acc[n][2] = fmaf(d.y, s[2], acc[n][2]);
                    acc[n][3] = fmaf(d.y, s[3], acc[n][3]);
                    if constexpr (kMin) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int col = n * 8 + 2 * t + e;
                            if (col < cols && col % kPieces == 0) {
                                const float xs = sums[(2 * u + b) * a.rows + col / kPieces];
                                acc[n][e] = fmaf(mn.x, xs, acc[n][e]);
                                acc[n][2 + e] = fmaf(mn.y, xs, acc[n][2 + e]);
                            }
                        }
                    }
                }
            }
            __syncwarp();   // the slot may be filled again
        }
        // ---- add up the warps of the tile and the pieces, in order ----
        float* red = reinterpret_cast<float*>(smem + a.red_at) + warp * kRedWarp;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[(g + 8 * (e >> 1)) * kRedPitch + n * 8 + 2 * t + (e & 1)] = acc[n][e];
        auto meet = [&]() {
            if (split == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(split * 32) : "memory");
        };
        meet();
        const float* all = reinterpret_cast<const float*>(smem + a.red_at) + group * split * kRedWarp;
        const int e = tid - group * split * 32, part = e % split;
        for (int base = 0; base < 16 * a.rows; base += 32) {
            const int o = base + e / split, row = o & 15, m = o >> 4;
            const int64_t n = static_cast<int64_t>(tile) * 16 + row;
            const bool in = o < 16 * a.rows && n < a.N;
            float v = 0.f;
            if (in)
#pragma unroll
                for (int p = 0; p < kPieces; ++p) v += all[part * kRedWarp + row * kRedPitch + m * kPieces + p];
            for (int x = 1; x < split; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
            if (in && part == 0) {
                if (a.bias) v += a.bias[n];
                if (a.residual) v += a.residual[m * a.ldy + n];
                if (a.y_f32) static_cast<float*>(a.y)[m * a.ldy + n] = v;
                else static_cast<Tx*>(a.y)[m * a.ldy + n] = from_f32<Tx>(v);
            }
        }
        meet();
    }
}

// ------------------------------------------------------------------ launch
// Warps per row tile: the split whose slowest warp streams the fewest units;
// of equal ones the smallest, which meets least often.
int split_of(int64_t tiles, int units, int sms) {
    int best = 1;
    int64_t best_cost = INT64_MAX;
    for (int s = 1; s <= kWarps && s <= units; s *= 2) {
        const int64_t groups = static_cast<int64_t>(sms) * (kWarps / s);
        const int64_t cost = (tiles + groups - 1) / groups * ((units + s - 1) / s);
        if (cost < best_cost) {
            best = s;
            best_cost = cost;
        }
    }
    return best;
}

struct Q4Plan {
    int stages, pitch, ring_at, red_at, sum_at, bytes;
};
// Shared memory of a launch over `rows` activation rows; stages 0 where it does not fit.
Q4Plan plan_of(int rows, int pieces, int n_tiles, int units, bool min) {
    for (int stages : {8, 4}) {
        Q4Plan p;
        p.stages = stages;
        p.pitch = units * 128 + 64;   // 64 bytes off a multiple of 128: eight columns' chunks miss one another's banks
        p.ring_at = static_cast<int>(round_up(rows * pieces * p.pitch, 128));
        p.red_at = p.ring_at + kWarps * stages * unit_bytes(min);
        p.sum_at = p.red_at + static_cast<int>(round_up(kWarps * (16 * (8 * n_tiles + 1) + 1) * 4, 128));
        p.bytes = p.sum_at + (min ? units * 2 * rows * 4 : 0);
        if (p.bytes <= kSmemMax) return p;
    }
    return Q4Plan{};
}
// Operand tiles (of 8 columns) that a launch over `rows` rows is built for, 0 = too many.
int n_tiles_of(int rows, int pieces) {
    const int n = (rows * pieces + 7) / 8;
    return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 0;
}

}  // namespace
}  // namespace b2q

using namespace b2q;

extern "C" {

b2q_status b2q_weight_q4_register(const void* blocks, int32_t ggml_type, int64_t N, int64_t K, int64_t row_bytes,
                                  int src_is_host, void* stream, b2q_weight_q4** out) {
    B2Q_REQUIRE_STATE();
    if (!blocks || !out) return set_error(B2Q_ERR_INVALID, "null pointer");
    if (ggml_type != B2Q_TYPE_Q4_0 && ggml_type != B2Q_TYPE_Q4_1)
        return set_error(B2Q_ERR_INVALID, "weights must be Q4_0 or Q4_1");
    if (N <= 0 || N > (1 << 24) || K <= 0 || K % 32 || K > kMaxK)
        return set_error(B2Q_ERR_SHAPE, "a 4-bit weight needs N in [1, 2^24] and K a multiple of 32 up to 28672");
    const bool min = ggml_type == B2Q_TYPE_Q4_1;
    if (row_bytes < K / 32 * (min ? 20 : 18))
        return set_error(B2Q_ERR_SHAPE, "row_bytes smaller than the row's blocks");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    b2q_weight_q4* w = new (std::nothrow) b2q_weight_q4();
    if (!w) return set_error(B2Q_ERR_NOMEM, "out of host memory");
    w->N = N;
    w->K = K;
    w->type = ggml_type;
    w->device = ds->device;
    w->tiles = (N + 15) / 16;
    w->units = (K + 63) / 64;
    void* staged = nullptr;
    const size_t src_bytes = static_cast<size_t>(N - 1) * row_bytes + K / 32 * (min ? 20 : 18);
    b2q_status st = B2Q_OK;
    if (cudaMalloc(reinterpret_cast<void**>(&w->packed), static_cast<size_t>(w->tiles * w->units * unit_bytes(min))) !=
            cudaSuccess ||
        (src_is_host && cudaMalloc(&staged, src_bytes) != cudaSuccess)) {
        cudaGetLastError();
        st = set_error(B2Q_ERR_NOMEM, "cudaMalloc of a 4-bit weight failed");
    }
    if (!st && src_is_host)
        st = cuda_check(cudaMemcpyAsync(staged, blocks, src_bytes, cudaMemcpyHostToDevice, s), "4-bit weight upload");
    if (!st) {
        const int64_t lanes = w->tiles * w->units * 32;
        pack_q4_kernel<<<static_cast<unsigned>((lanes + 255) / 256), 256, 0, s>>>(
            static_cast<const uint8_t*>(src_is_host ? staged : blocks), N, K / 32, row_bytes, min, w->tiles, w->units,
            w->packed);
        count_launch();
        st = cuda_check(cudaGetLastError(), "4-bit weight layout");
    }
    if (src_is_host) {
        const b2q_status sync = cuda_check(cudaStreamSynchronize(s), "4-bit weight layout");
        if (!st) st = sync;
        cudaFree(staged);
    }
    if (st) {
        cudaFree(w->packed);
        delete w;
        return st;
    }
    *out = w;
    return B2Q_OK;
}

b2q_status b2q_weight_q4_release(b2q_weight_q4* w) {
    if (!w) return B2Q_OK;
    cudaFree(w->packed);
    delete w;
    return B2Q_OK;
}

b2q_status b2q_mul_vec_q4(const b2q_weight_q4* w, const void* x, int32_t x_dtype, int64_t M, int64_t x_cols,
                          int64_t ldx, void* y, int32_t y_dtype, int64_t ldy, const float* bias,
                          const float* residual, void* stream) {
    B2Q_REQUIRE_STATE();
    if (!w) return set_error(B2Q_ERR_INVALID, "null weight");
    if (w->device != ds->device) return set_error(B2Q_ERR_INVALID, "weight registered on another device");
    if (x_dtype != B2Q_TYPE_F32 && x_dtype != B2Q_TYPE_F16 && x_dtype != B2Q_TYPE_BF16)
        return set_error(B2Q_ERR_INVALID, "x must be F32, F16 or BF16");
    if (y_dtype != B2Q_TYPE_F32 && y_dtype != x_dtype) return set_error(B2Q_ERR_INVALID, "y must be F32 or x's type");
    if (M < 0 || M > 65535) return set_error(B2Q_ERR_SHAPE, "bad M");
    if (x_cols <= 0 || round_up(x_cols, 32) != w->K)
        return set_error(B2Q_ERR_SHAPE, "x_cols must round up to the weight's K");
    if (ldx < x_cols || ldy < w->N) return set_error(B2Q_ERR_SHAPE, "ldx / ldy shorter than a row");
    if (M == 0) return B2Q_OK;
    if (!x || !y) return set_error(B2Q_ERR_INVALID, "null pointer");
    if (!ptr_aligned(x, x_dtype == B2Q_TYPE_F32 ? 4 : 2) || !ptr_aligned(y, y_dtype == B2Q_TYPE_F32 ? 4 : 2) ||
        !ptr_aligned(bias, 4) || !ptr_aligned(residual, 4))
        return set_error(B2Q_ERR_ALIGN, "misaligned rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool min = w->type == B2Q_TYPE_Q4_1;
    const int units = static_cast<int>(w->units);
    const int pieces = x_dtype == B2Q_TYPE_F32 ? 3 : 1;
    const size_t es = pieces == 3 ? 4 : 2, ys = y_dtype == B2Q_TYPE_F32 ? 4 : 2;
    // the most rows that a launch takes (operand tiles and shared memory), then as even launches as that allows
    int most = 1;
    while (most < M && n_tiles_of(most + 1, pieces) &&
           plan_of(most + 1, pieces, n_tiles_of(most + 1, pieces), units, min).stages)
        ++most;
    const int64_t launches = (M + most - 1) / most;
    const int split = split_of(w->tiles, units, ds->num_sms);
    const int groups = kWarps / split;
    const int64_t want = (w->tiles + groups - 1) / groups;
    const unsigned grid = static_cast<unsigned>(want < ds->num_sms ? want : ds->num_sms);
    for (int64_t i = 0, m0 = 0; i < launches; ++i) {
        const int rows = static_cast<int>((M - m0 + launches - i - 1) / (launches - i));
        const int n_tiles = n_tiles_of(rows, pieces);
        const Q4Plan p = plan_of(rows, pieces, n_tiles, units, min);
        if (!p.stages) return set_error(B2Q_ERR_SHAPE, "an activation row does not fit shared memory");
        auto go = [&](auto tx, auto mn, auto nt, auto stages) {
            using Tx = decltype(tx);
            Q4Args<Tx> a{w->packed, w->N, static_cast<int>(w->tiles), units, split,
                         reinterpret_cast<const Tx*>(static_cast<const uint8_t*>(x) + m0 * ldx * es), rows, x_cols, ldx,
                         static_cast<uint8_t*>(y) + m0 * ldy * ys, ldy, y_dtype == B2Q_TYPE_F32, bias,
                         residual ? residual + m0 * ldy : nullptr, p.pitch, p.ring_at, p.red_at, p.sum_at};
            auto* kernel = mul_vec_q4_kernel<Tx, decltype(mn)::value, decltype(nt)::value, decltype(stages)::value>;
            b2q_status st = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                            kSmemMax), "4-bit product shared memory");
            if (st) return st;
            kernel<<<grid, kThreads, p.bytes, s>>>(a);
            count_launch();
            return cuda_check(cudaGetLastError(), "4-bit product launch");
        };
        auto with_stages = [&](auto tx, auto mn, auto nt) {
            return p.stages == 8 ? go(tx, mn, nt, std::integral_constant<int, 8>{})
                                 : go(tx, mn, nt, std::integral_constant<int, 4>{});
        };
        auto with_tiles = [&](auto tx, auto mn) {
            return n_tiles == 1   ? with_stages(tx, mn, std::integral_constant<int, 1>{})
                   : n_tiles == 2 ? with_stages(tx, mn, std::integral_constant<int, 2>{})
                                  : with_stages(tx, mn, std::integral_constant<int, 4>{});
        };
        auto with_min = [&](auto tx) {
            return min ? with_tiles(tx, std::true_type{}) : with_tiles(tx, std::false_type{});
        };
        const b2q_status st = x_dtype == B2Q_TYPE_F32   ? with_min(float{})
                              : x_dtype == B2Q_TYPE_F16 ? with_min(__half{})
                                                        : with_min(__nv_bfloat16{});
        if (st) return st;
        m0 += rows;
    }
    return B2Q_OK;
}

}  // extern "C"
