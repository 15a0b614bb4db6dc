// b2q_q4.cu — products of few activation rows with ggml Q4_0 / Q4_1 weights
// (b2q_weight_q4_*, b2q_mul_vec_q4).
//
// y[n] = sum_kb d[n,kb] S[n,kb] (+ m[n,kb] X[kb]), S the sum of (q - 8) x (Q4_1: q x)
// over the 32 columns of block kb, X that of x.
//
// Bound: bytes, 18 (20) per 32 weights and at most once.  At the measured copy
// rate that is 11.6 T weights/s, and the SMs issue about 36 T lane operations/s:
// three instructions a weight for everything, which unpacking to floats and
// multiplying alone would take.  So even a single activation row goes to the
// tensor cores: one mma.sync (16 weight rows x 16 columns x 8 activation columns)
// does 8 of a lane's products and sums in fp32, and almost nothing is unpacked:
//
//  * A nibble OR-ed into the mantissa of 2^10 is the fp16 number 1024 + q (in bits 0-3
//    of a half) or 1024 + 16 q (bits 4-7), and one exact addition or multiply-add
//    makes it q - 8 (Q4_1: q): nine instructions for eight weights.  (Left in place as
//    fp16 subnormals q 2^-24 and q 2^-20 they take five, and 256000 x 1152 35 us; but the
//    tensor core aligns a sum's products by the operands' exponents, of which a
//    subnormal has the largest, and cuts off seven bits: relative errors of 1e-6, and
//    of 1e-5 beside a large activation.)
//  * An activation row is scaled by a power of two and becomes fp16 operands: fp16 and
//    bf16 values one, an fp32 value two, x rounded to 11 bits and the rest rounded to
//    11 bits, which leaves nothing of three values in four and at most 2^-23 |x|; they
//    take as many of the eight activation columns.  The row has one scale, so nothing
//    is held closer than 2^-34 of its largest value (fp16 ends at 2^-24, and that value
//    lies at 2^9 or above): beside one 1e6 times as large values keep 14 bits.
//  * S leaves the tensor core once per block and is summed in fp32, d S.
// Relative error against 64 bits: 1 x 1152 x 4320, Q4_0, 9e-8 (plain fp32 products
// 1.9e-7); 1 x 256000 x 1152, Q4_1, 1.6e-7 to 2.6e-7 by the row (1.3e-7: with the minima
// apart, d S and m X are each several times their sum, and so are their roundings, of
// which that of X is the same for every output).
//
// The weights are laid out at registration in the order the lanes want them:
// per 16 rows a run of units of 128 columns, each 1024 bytes of nibbles (lane l of
// the warp: twice 16 bytes) and the blocks' scales (128 bytes; Q4_1: 128 more for
// m).  A warp streams units through its own ring of asynchronous copies, which runs
// on across row tiles (with one bulk copy and a barrier per unit the stream took 64
// of 176 instructions a unit); the activations sit in shared memory for the whole
// launch (a fixed grid of one CTA of 16, 24 or 32 warps per SM).  `split` warps share a row
// tile, each taking every split-th unit, and add up in a fixed order.
//
// Measured on one B200 (copy bandwidth 6.53 TB/s), device time: 1 x 256000 x 1152, Q4_1,
// fp32, 185 MB: 36.4 us, 5.1 TB/s, issue slots 69% busy; 7 x 28672 x 8192, bf16, 133 MB:
// 34.3 us, 3.9 TB/s, of which 7 until the rows are staged; 1 x 28672 x 8192: 29.6 us; 1 x
// 4096 x 4096: 4.6 us; 1 x 1152 x 4320, fp32: 4.4 us, the launch and one trip to memory.
#include "b2q_decode.cuh"

#include <cstddef>
#include <new>
#include <type_traits>

struct b2q_weight_q4 {
    int64_t N = 0, K = 0;
    int type = 0, device = -1;
    int64_t tiles = 0, units = 0;   // of 16 rows; of 128 columns per row tile
    uint8_t* packed = nullptr;      // [tiles][units][unit_bytes]
};

namespace b2q {
namespace {

constexpr int kMaxRows = 32;        // of one launch
constexpr int kMaxK = 28672;        // two pieces of a row still fit shared memory next to the rings
constexpr int kSmemMax = 227 * 1024 - 1024;   // next to the static part

constexpr int unit_bytes(bool min) { return min ? 1280 : 1152; }
inline __host__ __device__ int red_pitch(int cols) { return cols | 1; }   // odd: rows in different banks

// ------------------------------------------------------------------ layout
// Lane l = 4 g + t of a unit holds, for each of its four blocks, the columns
// 8 t .. 8 t + 7 of rows g and g + 8: one 32-bit word each, column 2 j in the
// nibble at bit 4 j and column 2 j + 1 in that at bit 16 + 4 j.  Blocks 0 and 1
// fill the first 512 bytes, 2 and 3 the next; then per g the scales of
// (block, row g), (block, row g + 8), ..., and in Q4_1 the same for m.
__global__ void pack_q4_kernel(const uint8_t* __restrict__ raw, int64_t N, int64_t Kb, int64_t row_bytes, bool min,
                               int64_t tiles, int64_t units, uint8_t* __restrict__ out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;   // one lane of one unit
    if (i >= tiles * units * 32) return;
    const int l = static_cast<int>(i & 31), g = l >> 2, t = l & 3;
    const int64_t unit = (i >> 5) % units, tile = (i >> 5) / units;
    uint8_t* dst = out + (i >> 5) * unit_bytes(min);
    uint32_t w[8];
    for (int x = 0; x < 8; ++x) {
        const int64_t n = tile * 16 + g + 8 * (x & 1), kb = unit * 4 + (x >> 1);
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
            reinterpret_cast<uint16_t*>(dst + 1024 + g * 16)[x] = d;
            if (min) reinterpret_cast<uint16_t*>(dst + 1152 + g * 16)[x] = m;
        }
    }
    *reinterpret_cast<uint4*>(dst + l * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + 512 + l * 16) = make_uint4(w[4], w[5], w[6], w[7]);
}

// ------------------------------------------------------------------ product
struct Q4Args {
    const uint8_t* w;
    int64_t N;
    int tiles, units, split;
    int part_log2;          // 2^part_log2 lanes add up the warps of an output
    bool pair;              // two CTAs stage the activations for one another
    const void* x;
    int x_type, pieces;
    int rows;               // activation rows of this launch
    int64_t x_cols, ldx;
    void* y;
    int64_t ldy;
    bool y_f32;
    const float *bias, *residual;
    int pitch, ring_at, red_at, sum_at;   // shared memory: bytes of an operand column, parts' offsets
    uint32_t magic = 0x64006400u;         // 2^10 twice.  An argument, so that it stays in a register: with two
                                          // constants in sight the compiler makes two instructions of (w & a) | b
};

// The word's four pairs of a lane as fp16 integers q - 8 (Q4_1: q): OR-ed into the
// mantissa of 2^10 a nibble gives 1024 + q (bits 0-3) or 1024 + 16 q (bits 4-7), and
// one exact addition or multiply-add takes the rest off.
template <bool kMin>
__device__ __forceinline__ void unpack_q4(uint32_t w, uint32_t magic, uint32_t (&r)[4]) {
    const __half2 off = __float2half2_rn(kMin ? -1024.f : -1032.f);
    const __half2 off16 = __float2half2_rn(kMin ? -64.f : -72.f), s16 = __float2half2_rn(0.0625f);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const uint32_t s = w >> (4 * j), u = (s & 0x000F000Fu) | magic, v = (s & 0x00F000F0u) | magic;
        const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&u), off);
        const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&v), s16, off16);
        r[j] = *reinterpret_cast<const uint32_t*>(&x);
        r[j + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// What the rows' staging leaves in shared memory beside the operands.
struct RowState {
    uint32_t peak[kMaxRows];   // bits of the largest finite |x|
    int shift[kMaxRows];       // the operands are x 2^shift
    float back[kMaxRows][2];   // factors that take a row's sums back: 2^-shift, in two
    uint32_t odd;              // rows that hold an infinity or a NaN (left out of the operands)
};
// x 2^top_shift(peak) has its largest value in [2^14, 2^15); peaks below 2^-113 stay smaller.
__device__ __forceinline__ int top_shift(uint32_t peak) { return min(141 - static_cast<int>(peak >> 23), 127); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

// Eight values as they lie in memory.
template <class Tx>
struct Eight {
    uint4 r[sizeof(Tx) / 2];
    __device__ __forceinline__ void load(const Tx* x, int left, bool vec) {
        if (vec && left >= 8) {
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(Tx)) / 2; ++j) r[j] = reinterpret_cast<const uint4*>(x)[j];
        } else {
            Tx* e = reinterpret_cast<Tx*>(r);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = j < left ? x[j] : from_f32<Tx>(0.f);
        }
    }
    __device__ __forceinline__ float2 pair(int j) const {   // values 2 j, 2 j + 1
        const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
        if constexpr (sizeof(Tx) == 4) return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
        else return unpack2<Tx>(w[j]);
    }
    __device__ __forceinline__ uint32_t peak_bits() const {   // of the largest |x|, infinities and NaN on top
        const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
        uint32_t m = 0;
        if constexpr (sizeof(Tx) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, w[j] & 0x7FFFFFFFu);
            return m;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
            return __float_as_uint(unpack2<Tx>(max(m & 0xFFFFu, m >> 16)).x);
        }
    }
};

// Activation rows into shared memory: operand column p * rows + m holds piece p
// of row m, x 2^shift.  Q4_1: `sum_at` gets the sums X of each block's scaled values,
// times 2^-5, as operands of the product with m: three fp16 pieces side by side in
// k, four blocks x 8 bytes per unit and row.
//
// A warp takes 256 columns of a row at a time.  A row's power of two is a guess
// from its first 32 values, the largest of them taken to [2^9, 2^10): that leaves
// the row's largest value a factor of 32, and loses no more than 2^-34 of it.  The
// same pass takes the peaks; a row that needs more room is staged again with the
// power that its peak gives (`again`).  Two CTAs of a cluster (`pair`) stage half of
// the work each and store it in both shared memories.
template <class Tx, int kPieces, bool kMin, int kWarps>
__device__ __forceinline__ void stage_x(const Q4Args& a, uint8_t* smem, RowState& st, bool again) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = a.units * 16, segs = (chunks + 31) / 32;   // of 8 columns; of 32 chunks
    const Tx* px = static_cast<const Tx*>(a.x);
    const bool vec = (a.ldx * sizeof(Tx)) % 16 == 0 && (reinterpret_cast<uintptr_t>(px) & 15) == 0;
    const uint32_t rank = a.pair ? cluster_rank() : 0, here = smem_u32(smem), state = smem_u32(&st);
    const uint32_t there = a.pair ? in_cta(here, rank ^ 1) : 0, state_there = a.pair ? in_cta(state, rank ^ 1) : 0;
    const int workers = a.pair ? 2 * kWarps : kWarps, worker = warp + (rank ? kWarps : 0);
    const int row_step = workers / segs, seg_step = workers % segs;
    int m = worker / segs, seg = worker % segs;
    Eight<Tx> next;
    Tx next_sample = from_f32<Tx>(0.f);
    auto load = [&]() {
        const Tx* row = px + m * a.ldx;
        const int c = seg * 32 + lane;
        next.load(row + c * 8, static_cast<int>(a.x_cols) - c * 8, vec);
        if (lane < a.x_cols) next_sample = row[lane];
    };
    if (m < a.rows) load();
#pragma unroll 1
    while (m < a.rows) {
        const Eight<Tx> v = next;
        const Tx sample = next_sample;
        const int row = m, c = seg * 32 + lane;
        m += row_step;
        seg += seg_step;
        if (seg >= segs) {
            seg -= segs;
            ++m;
        }
        if (m < a.rows) load();
        uint32_t peak = __reduce_max_sync(0xffffffffu, v.peak_bits());
        const bool odd = peak >= 0x7F800000u;
        int shift;
        if (again) {
            shift = st.shift[row];
        } else {
            if (odd) {
                peak = 0;
                for (int j = 0; j < 4; ++j) {
                    const float2 x = v.pair(j);
                    if (is_finite(x.x)) peak = max(peak, __float_as_uint(fabsf(x.x)));
                    if (is_finite(x.y)) peak = max(peak, __float_as_uint(fabsf(x.y)));
                }
                peak = __reduce_max_sync(0xffffffffu, peak);
            }
            const float f = fabsf(to_f32(sample));
            shift = top_shift(__reduce_max_sync(0xffffffffu, is_finite(f) ? __float_as_uint(f) : 0u)) - 5;
            if (lane == 0) {
                atomicMax(&st.peak[row], peak);
                if (odd) atomicOr(&st.odd, 1u << row);
                st.shift[row] = shift;   // every warp of the row finds the same
                if (a.pair) {
                    max_cluster_32(state_there + offsetof(RowState, peak) + 4 * row, peak);
                    if (odd) or_cluster_32(state_there + offsetof(RowState, odd), 1u << row);
                    st_cluster_32(state_there + offsetof(RowState, shift) + 4 * row, static_cast<uint32_t>(shift));
                }
            }
        }
        const float s = pow2(shift);
        float sum = 0.f;
        uint32_t p[kPieces][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 x = v.pair(j);
            if (odd) {
                if (!is_finite(x.x)) x.x = 0.f;
                if (!is_finite(x.y)) x.y = 0.f;
            }
            x.x *= s;
            x.y *= s;
            if constexpr (kMin) sum += x.x + x.y;
#pragma unroll
            for (int z = 0; z + 1 < kPieces; ++z) {
                p[z][j] = pack2<__half>(x.x, x.y);
                const float2 h = unpack2<__half>(p[z][j]);
                x.x -= h.x;
                x.y -= h.y;
            }
            p[kPieces - 1][j] = pack2<__half>(x.x, x.y);
        }
        if constexpr (kMin) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        }
        if (c < chunks) {
            const int dst = row * a.pitch + c * 16;
#pragma unroll
            for (int z = 0; z < kPieces; ++z) {
                const uint4 v = make_uint4(p[z][0], p[z][1], p[z][2], p[z][3]);
                *reinterpret_cast<uint4*>(smem + dst + z * a.rows * a.pitch) = v;
                if (a.pair) st_cluster_128(there + dst + z * a.rows * a.pitch, v);
            }
            if (kMin && (c & 3) == 0) {
                __half h[4];
                sum *= 0.03125f;
#pragma unroll
                for (int z = 0; z < 3; ++z) {
                    h[z] = __float2half_rn(sum);
                    sum -= __half2float(h[z]);
                }
                h[3] = __float2half_rn(0.f);
                const int at = a.sum_at + (((c >> 4) * a.rows + row) * 4 + ((c >> 2) & 3)) * 8;
                *reinterpret_cast<uint2*>(smem + at) = *reinterpret_cast<const uint2*>(h);
                if (a.pair) st_cluster_64(there + at, *reinterpret_cast<const uint2*>(h));
            }
        }
    }
    // what columns of other pieces take
    if (kMin && threadIdx.x < 8) reinterpret_cast<float*>(smem + a.sum_at)[a.units * a.rows * 8 + threadIdx.x] = 0.f;
}

template <bool kMin, int kWarps>
__device__ __forceinline__ void stage_rows(const Q4Args& a, uint8_t* smem, RowState& st) {
    const int tid = threadIdx.x;
    auto meet = [&]() {
        if (a.pair) cluster_sync();
        else __syncthreads();
    };
    if (tid < kMaxRows) st.peak[tid] = 0;
    if (tid == 0) st.odd = 0;
    meet();
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        if (a.x_type == B2Q_TYPE_F32) stage_x<float, 2, kMin, kWarps>(a, smem, st, pass);
        else if (a.x_type == B2Q_TYPE_BF16) stage_x<__nv_bfloat16, 1, kMin, kWarps>(a, smem, st, pass);
        else stage_x<__half, 1, kMin, kWarps>(a, smem, st, pass);
        meet();   // (peaks and shifts are the same in both CTAs of a pair, and so is what follows)
        const bool mine = pass == 0 && tid < a.rows;
        const bool over = mine && st.shift[tid] > top_shift(st.peak[tid]);
        if (over) st.shift[tid] = top_shift(st.peak[tid]);
        if (mine) {
            const int e = -st.shift[tid];
            st.back[tid][0] = pow2(e >> 1);
            st.back[tid][1] = pow2(e - (e >> 1));
        }
        if (!__syncthreads_or(over)) break;
    }
}

// w[n][k] as registered
template <bool kMin>
__device__ float weight_at(const Q4Args& a, int64_t n, int64_t k) {
    const uint8_t* u = a.w + ((n >> 4) * a.units + (k >> 7)) * unit_bytes(kMin);
    const int g = n & 7, high = (n >> 3) & 1, b = (k >> 5) & 3, t = (k >> 3) & 3, e = k & 7;
    const uint32_t word = reinterpret_cast<const uint32_t*>(u)[(b >> 1) * 128 + (4 * g + t) * 4 + 2 * (b & 1) + high];
    const int q = (word >> (4 * (e >> 1) + 16 * (e & 1))) & 15;
    const float d = __half2float(reinterpret_cast<const __half*>(u + 1024)[8 * g + 2 * b + high]);
    if (!kMin) return d * static_cast<float>(q - 8);
    return d * static_cast<float>(q) + __half2float(reinterpret_cast<const __half*>(u + 1152)[8 * g + 2 * b + high]);
}
// What a row's infinities and NaN add to output n.
template <bool kMin>
__device__ __noinline__ float odd_terms(const Q4Args& a, int64_t n, int m) {
    float v = 0.f;
    for (int64_t k = 0; k < a.x_cols; ++k) {
        const int64_t i = m * a.ldx + k;
        const float x = a.x_type == B2Q_TYPE_F32   ? static_cast<const float*>(a.x)[i]
                        : a.x_type == B2Q_TYPE_F16 ? to_f32(static_cast<const __half*>(a.x)[i])
                                                   : to_f32(static_cast<const __nv_bfloat16*>(a.x)[i]);
        if (!is_finite(x)) v += weight_at<kMin>(a, n, k) * x;
    }
    return v;
}

// kGroup units of a tile are waited for together, where kStages rings of them fit.
template <bool kMin, int kN, int kGroup, int kStages, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 1) mul_vec_q4_kernel(const __grid_constant__ Q4Args a) {
    constexpr int kUnit = unit_bytes(kMin);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RowState st;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = a.split, sub = warp % split, group = warp / split, groups = kWarps / split;
    const int first = group * gridDim.x + blockIdx.x, step = gridDim.x * groups;   // every SM gets its share of the tiles
    const int per_tile = (a.units - sub + split - 1) / split;   // units of this warp in each of its tiles

    // ---- the weights' stream: a unit is asked for as soon as its slot is free ----
    constexpr int kSlot = kGroup * kUnit;
    const int ring = a.ring_at + warp * kStages * kSlot;
    const uint8_t* tile_src = a.w + (static_cast<int64_t>(first) * a.units + sub) * kUnit + lane * 16;
    const uint8_t* src = tile_src;
    const int64_t unit_step = static_cast<int64_t>(split) * kUnit;
    const int64_t tile_step = static_cast<int64_t>(step) * a.units * kUnit;
    int tiles_left = first < a.tiles ? (a.tiles - first + step - 1) / step : 0;   // tiles still to ask for
    int left = per_tile;                                                          // units of this one
    auto issue = [&](int slot) {
        if (tiles_left > 0) {
            const uint32_t dst = smem_u32(smem) + slot + lane * 16;
#pragma unroll
            for (int u = 0; u < kGroup; ++u)
                if (u == 0 || left > u) {
                    cp_async_16(dst + u * kUnit, src, true);
                    cp_async_16(dst + u * kUnit + 512, src + 512, true);
                    if (lane < (kUnit - 1024) / 16) cp_async_16(dst + u * kUnit + 1024, src + 1024, true);
                    src += unit_step;
                }
            left -= kGroup;
            if (left <= 0) {
                left = per_tile;
                --tiles_left;
                tile_src += tile_step;
                src = tile_src;
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue(ring + i * kSlot);
    // the weights are on their way; the activations may be another kernel's results
    let_next_start();
    wait_for_previous();
    stage_rows<kMin, kWarps>(a, smem, st);

    // This lane's operand columns.  A column that no row has computes on the
    // first one's values; its results are not read.
    const int cols = a.rows * a.pieces;
    int x0[kN], sum0[kN], sum_step[kN];   // sums (Q4_1): of this lane's column, block t
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const int col = n * 8 + g < cols ? n * 8 + g : 0;
        const bool own = n * 8 + g < a.rows;   // X goes with a row's first piece
        x0[n] = col * a.pitch + t * 16 + sub * 256;
        sum_step[n] = own ? a.rows * 32 : 0;
        sum0[n] = a.sum_at + (own ? (sub * a.rows + col) * 32 : a.units * a.rows * 32) + t * 8;
    }
    int slot = ring, buf = 0;
    for (int tile = first; tile < a.tiles; tile += step, buf ^= 1) {
        float acc[kN][4] = {};
        int xo = 0, so[kN];
#pragma unroll
        for (int n = 0; n < kN; ++n) so[n] = sum0[n];
        for (int j = 0; j < per_tile; j += kGroup) {
            cp_wait<kStages - 1>();
            __syncwarp();   // every lane's part of the units has come
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                if (u && j + u >= per_tile) break;
                const uint8_t* use = smem + slot + u * kUnit;
                const uint4 wa = *reinterpret_cast<const uint4*>(use + lane * 16);
                const uint4 wb = *reinterpret_cast<const uint4*>(use + 512 + lane * 16);
                const uint4 dd = *reinterpret_cast<const uint4*>(use + 1024 + g * 16);
                const uint32_t w8[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                const uint32_t d4[4] = {dd.x, dd.y, dd.z, dd.w};
                if constexpr (kMin) {   // block t's m three times in k, against the pieces of its X
                    const uint32_t mm = *reinterpret_cast<const uint32_t*>(use + 1152 + g * 16 + t * 4);
                    const uint32_t m0 = __byte_perm(mm, 0, 0x1010), m8 = __byte_perm(mm, 0, 0x3232);
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        const uint2 xp = *reinterpret_cast<const uint2*>(smem + so[n]);
                        float v[4];
                        mma_16816_from0(v, m0, m8, m0, m8, xp.x, xp.y);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][e] = fmaf(v[e], 32.f, acc[n][e]);   // (X was scaled by 2^-5)
                        so[n] += split * sum_step[n];
                    }
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t lo[4], hi[4];
                    unpack_q4<kMin>(w8[2 * b], a.magic, lo);
                    unpack_q4<kMin>(w8[2 * b + 1], a.magic, hi);
                    const float2 d = unpack2<__half>(d4[b]);
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        const uint4 xv = *reinterpret_cast<const uint4*>(smem + x0[n] + xo + b * 64);
                        float s[4];
                        mma_16816_from0(s, lo[0], hi[0], lo[1], hi[1], xv.x, xv.y);
                        mma_16816<__half>(s, lo[2], hi[2], lo[3], hi[3], xv.z, xv.w);
                        acc[n][0] = fmaf(d.x, s[0], acc[n][0]);
                        acc[n][1] = fmaf(d.x, s[1], acc[n][1]);
                        acc[n][2] = fmaf(d.y, s[2], acc[n][2]);
                        acc[n][3] = fmaf(d.y, s[3], acc[n][3]);
                    }
                }
                xo += split * 256;
            }
            __syncwarp();   // the slot may be filled again
            issue(slot);
            slot += kSlot;
            if (slot == ring + kStages * kSlot) slot = ring;
        }
        auto put = [&](int m, int n, float v) {
            if (n >= a.N) return;
            v = v * st.back[m][0] * st.back[m][1];
            if ((st.odd >> m) & 1) v += odd_terms<kMin>(a, n, m);
            const int64_t at = m * a.ldy + n;
            if (a.bias) v += a.bias[n];
            if (a.residual) v += a.residual[at];
            if (a.y_f32) static_cast<float*>(a.y)[at] = v;
            else if (a.x_type == B2Q_TYPE_F16) static_cast<__half*>(a.y)[at] = from_f32<__half>(v);
            else static_cast<__nv_bfloat16*>(a.y)[at] = from_f32<__nv_bfloat16>(v);
        };
        if (split == 1 && a.rows == 1) {   // a lane has all of an output: its row's pieces, columns 0 and 1
            if (t == 0) {
                put(0, tile * 16 + g, a.pieces == 1 ? acc[0][0] : acc[0][0] + acc[0][1]);
                put(0, tile * 16 + g + 8, a.pieces == 1 ? acc[0][2] : acc[0][2] + acc[0][3]);
            }
            continue;
        }
        // ---- add up the tile's warps and the pieces, in order; two buffers, so that
        // one meeting a tile suffices ----
        const int pitch = red_pitch(cols), part_floats = 16 * pitch;
        float* all = reinterpret_cast<float*>(smem + a.red_at) + (buf * kWarps + group * split) * part_floats;
        float* red = all + sub * part_floats + g * pitch + 2 * t;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n * 8 + 2 * t + (e & 1) < cols) red[8 * (e >> 1) * pitch + n * 8 + (e & 1)] = acc[n][e];
        if (split == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(group), "r"(split * 32) : "memory");
        // 2^part_log2 neighbouring lanes take an output, each some of its warps' parts
        const int me = tid - group * split * 32, part = me & ((1 << a.part_log2) - 1);
        for (int base = 0; base < 16 * a.rows; base += split * 32 >> a.part_log2) {
            const int o = base + (me >> a.part_log2), row = o & 15, m = o >> 4;
            const bool in = m < a.rows;
            float v = 0.f;
            if (in) {
                const float* p = all + part * part_floats + row * pitch + m;
                for (int w = part; w < split; w += 1 << a.part_log2, p += part_floats << a.part_log2)
                    v += a.pieces == 1 ? p[0] : p[0] + p[a.rows];
            }
            for (int x = 1 << a.part_log2 >> 1; x; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
            if (in && !part) put(m, tile * 16 + row, v);
        }
    }
}

// ------------------------------------------------------------------ launch
// What the fullest SM has to do, in half units of all its warps: two a unit that a
// warp streams, and per tile three for its end, four where `split` warps meet there.
int64_t cost_of(int64_t tiles, int units, int sms, int warps, int split) {
    const int64_t rounds = ((tiles + sms - 1) / sms * split + warps - 1) / warps;
    return rounds * (2 * ((units + split - 1) / split) + (split > 1 ? 4 : 3)) * warps;
}
// log2 of the lanes that share an output at a tile's end: all warps' parts side by
// side where the outputs leave that many lanes.
int part_log2_of(int split, int rows) {
    int l = 0;
    while ((2 << l) <= split && 16 * rows * (2 << l) <= split * 32) ++l;
    return l;
}

struct Q4Plan {
    int group, stages, pitch, ring_at, red_at, sum_at, bytes;
};
// Shared memory of a launch over `rows` activation rows, with as deep a ring as
// it holds; stages 0 where it does not fit.
Q4Plan plan_of(int rows, int pieces, int warps, int units, bool min) {
    Q4Plan p{};
    p.pitch = units * 256 + 64;   // 64 bytes off a multiple of 128: eight columns' chunks miss one another's banks
    p.red_at = static_cast<int>(round_up(rows * pieces * p.pitch, 128));
    p.sum_at = p.red_at + static_cast<int>(round_up(2 * warps * 16 * red_pitch(rows * pieces) * 4, 128));
    p.ring_at = p.sum_at + (min ? static_cast<int>(round_up((units * rows + 1) * 32, 128)) : 0);
    constexpr int kRings[][2] = {{2, 3}, {2, 2}, {1, 2}};   // units of a group, stages
    for (const auto& r : kRings) {
        if (warps > 16 && r[1] == 3) continue;   // (as many warps fill shared memory with two)
        p.bytes = p.ring_at + warps * unit_bytes(min) * r[0] * r[1];
        if (p.bytes <= kSmemMax) {
            p.group = r[0];
            p.stages = r[1];
            break;
        }
    }
    return p;
}
// Operand tiles (of 8 columns) that a launch over `rows` rows is built for, 0 = too many.
int n_tiles_of(int rows, int pieces) {
    const int n = rows <= kMaxRows ? (rows * pieces + 7) / 8 : 5;
    return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 0;
}
// The warps of a CTA (one per SM), the split and the shared memory of a launch.  One
// operand tile leaves the registers for 24 or 32 warps, and what suits the number
// of tiles costs least: 256000 x 1152 takes 37.8 us with 32 warps and 35.8 with 24,
// 7 x 28672 x 8192 33.9 and 35.2.  16 warps start 0.7 us sooner: where an SM has no
// more than four units for each (1 x 1152 x 4320: 4.4 against 5.1 us), where two
// or four operand tiles need the registers, and where long rows leave no room for 24
// warps' rings of two stages (4 x 28672 x 8640, Q4_1, fp32: 41.0 us; 24 warps with one
// stage each 73.5).
struct Choice {
    int n_tiles, warps, split;
    Q4Plan plan;
};
Choice choose(int rows, int pieces, int64_t tiles, int units, int sms, bool min) {
    Choice best{};
    const int n = n_tiles_of(rows, pieces);
    if (!n) return best;
    const bool few = n > 1 || (tiles + sms - 1) / sms * units <= 64;
    const bool full = !few && !plan_of(rows, pieces, 24, units, min).stages;
    int64_t best_cost = INT64_MAX;
    for (int warps : {16, 24, 32}) {
        if (warps == 16 ? !few && !full : few) continue;
        const Q4Plan p = plan_of(rows, pieces, warps, units, min);
        if (!p.stages || p.stages < best.plan.stages) continue;
        for (int split = 1; warps % split == 0 && split <= units; split *= 2) {
            const int64_t cost = cost_of(tiles, units, sms, warps, split);
            if (cost >= best_cost && p.stages == best.plan.stages) continue;
            best = Choice{n, warps, split, p};
            best_cost = cost;
        }
    }
    return best;
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
    w->units = (K + 127) / 128;
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
    // complete when this returns: the product reads weights before it waits for other kernels
    const b2q_status sync = cuda_check(cudaStreamSynchronize(s), "4-bit weight layout");
    if (!st) st = sync;
    if (staged) cudaFree(staged);
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
        !words(bias, residual))
        return set_error(B2Q_ERR_ALIGN, "misaligned rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool min = w->type == B2Q_TYPE_Q4_1;
    const int units = static_cast<int>(w->units);
    const int pieces = x_dtype == B2Q_TYPE_F32 ? 2 : 1;
    const size_t es = x_dtype == B2Q_TYPE_F32 ? 4 : 2, ys = y_dtype == B2Q_TYPE_F32 ? 4 : 2;
    auto choice = [&](int rows) { return choose(rows, pieces, w->tiles, units, ds->num_sms, min); };
    // the most rows that a launch takes (operand tiles and shared memory), then as even launches as that allows
    int most = 1;
    while (most < M && choice(most + 1).plan.stages) ++most;
    const int64_t launches = (M + most - 1) / most;
    for (int64_t i = 0, m0 = 0; i < launches; ++i) {
        const int rows = static_cast<int>((M - m0 + launches - i - 1) / (launches - i));
        const Choice c = choice(rows);
        const Q4Plan& p = c.plan;
        const int n_tiles = c.n_tiles, warps = c.warps, split = c.split;
        if (!p.stages) return set_error(B2Q_ERR_SHAPE, "an activation row does not fit shared memory");
        // Pairs where each warp would stage more than two pieces of 256 columns by itself
        // (7 x 32 x 8192: 11.1 -> 8.4 us); an SM may stay idle where their number is odd.
        const bool pair = rows * ((units + 1) / 2) > 2 * warps && w->tiles > 1 && ds->num_sms >= 2;
        unsigned grid = static_cast<unsigned>(w->tiles < ds->num_sms ? w->tiles : ds->num_sms);
        if (pair) grid = grid / 2 * 2;
        const Q4Args a{w->packed, w->N, static_cast<int>(w->tiles), units, split,
                       part_log2_of(split, rows), pair,
                       static_cast<const uint8_t*>(x) + m0 * ldx * es, x_dtype, pieces, rows, x_cols, ldx,
                       static_cast<uint8_t*>(y) + m0 * ldy * ys, ldy, y_dtype == B2Q_TYPE_F32, bias,
                       residual ? residual + m0 * ldy : nullptr, p.pitch, p.ring_at, p.red_at, p.sum_at};
        auto go = [&](auto mn, auto nt, auto group, auto stages, auto wp) {
            auto* kernel = mul_vec_q4_kernel<decltype(mn)::value, decltype(nt)::value, decltype(group)::value,
                                             decltype(stages)::value, decltype(wp)::value>;
            static std::atomic<uint64_t> allowed{0};
            const b2q_status st = allow_smem(kernel, kSmemMax, allowed, ds->device);
            if (st) return st;
            return cuda_check(launch_after(pair ? 2 : 1, kernel, dim3(grid), dim3(warps * 32), p.bytes, s, a),
                              "4-bit product launch");
        };
        constexpr std::integral_constant<int, 1> one{};
        constexpr std::integral_constant<int, 2> two{};
        auto with_stages = [&](auto mn, auto nt, auto wp) {
            if (p.group == 2 && p.stages == 3) {
                if constexpr (decltype(wp)::value == 16) return go(mn, nt, two, std::integral_constant<int, 3>{}, wp);
            }
            return p.group == 2 ? go(mn, nt, two, two, wp) : go(mn, nt, one, two, wp);
        };
        constexpr std::integral_constant<int, 16> w16{};
        constexpr std::integral_constant<int, 24> w24{};
        constexpr std::integral_constant<int, 32> w32{};
        auto with_tiles = [&](auto mn) {
            return n_tiles == 1   ? (warps == 32   ? with_stages(mn, one, w32)
                                     : warps == 24 ? with_stages(mn, one, w24)
                                                   : with_stages(mn, one, w16))
                   : n_tiles == 2 ? with_stages(mn, std::integral_constant<int, 2>{}, w16)
                                  : with_stages(mn, std::integral_constant<int, 4>{}, w16);
        };
        const b2q_status st = min ? with_tiles(std::true_type{}) : with_tiles(std::false_type{});
        if (st) return st;
        m0 += rows;
    }
    return B2Q_OK;
}

}  // extern "C"
