// b2q_paged.cu — attention of single tokens over a paged key-value cache
// (b2q_attention_paged).
//
// out = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q.k_j - ref), c = scale log2(e),
// in one pass over the keys: a running maximum fixes ref, and the sums so far
// are multiplied by 2^(old ref - new ref) when it moves.  Partial results over
// disjoint keys (ref, sum p, sum p v) join the same way, so the keys of one
// request may be split anywhere.
//
// Bound: bytes.  Every key costs 4 d bytes of cache and 4 d operations per query
// head of its group, so even 16 heads on one key are 16 operations a byte.
//
// Work split.  A unit is 64 keys (a tile) of one (row, key head, block of query
// rows).  The units of all rows in order are dealt to a fixed grid of CTAs in
// equal contiguous shares, whatever the lengths: one request of 100,000 keys
// and hundreds of ragged ones load every SM alike, lengths are read on the
// device, and a captured launch stays valid as they grow.  A CTA's share holds
// the end of one group, whole groups, and the start of another; what is not
// whole goes to scratch as a partial result, and the last CTA to arrive at a
// group joins its parts in their order (so the bits repeat).  Nobody waits.
//
// Inside a CTA each of four warps takes 16 keys of every tile and keeps its own
// ref, sum and output; they meet only where a group ends.  Keys and values
// come by 16-byte asynchronous copies, each warp filling its own ring of
// stages, so loads run on across tiles, groups and rows with no block barrier.
// Shared rows have an odd number of 16-byte chunks, which keeps ldmatrix free of
// bank conflicts for every head width.
//
// Products run on mma.sync (16 query rows x 8 keys): a decode step has 1 to 16
// query rows per key head, far from the 64 to 128 of a tcgen05 tile, and the
// bytes bind long before the tensor pipe.  Probabilities enter the second
// product as a 16-bit head and remainder(s), 22 to 24 bits in all: rounding
// them to 16 bits would cost as much as the output's own rounding.  With at
// most 8 query rows the head takes rows 0-7 of the operand and the remainder
// rows 8-15, so the exact product costs no more instructions than the rounded
// one would.
#include "b2q_decode.cuh"

#include <cmath>
#include <type_traits>

namespace b2q {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16 * kWarps;     // keys of a unit
constexpr int kMaxCtas = 1024;         // join counters at the start of the scratch
constexpr size_t kCounterBytes = kMaxCtas * sizeof(uint32_t);

// Per head width (padded to DP): stages of the ring and CTAs per SM, as many as
// the 227 KB of shared memory hold next to the join buffer.
template <int DP>
struct Shape {
    static constexpr int kChunks = (DP / 8) | 1;            // 16-byte chunks of a shared row
    static constexpr int kPitch = kChunks * 16;
    static constexpr int kStageBytes = 2 * 16 * kPitch;     // one warp's keys and values
    static constexpr int kStages = DP > 128 ? 3 : 3;
    static constexpr int kCtas = DP > 128 ? 1 : (DP > 64 ? 2 : 3);
    static constexpr int kLanes = DP <= 64 ? 8 : (DP <= 128 ? 16 : 32);   // lanes that copy one row
    static constexpr int kOutPitch = DP + 8;
};
template <int DP, int kRows>
constexpr size_t smem_bytes() {
    return static_cast<size_t>(kWarps) * Shape<DP>::kStages * Shape<DP>::kStageBytes +
           static_cast<size_t>(kRows) * Shape<DP>::kOutPitch * 4;
}
// floats of one partial result: output rows, then refs and sums
template <int DP, int kRows>
constexpr int part_floats() { return kRows * DP + 2 * kRows; }

template <class T>
struct PagedArgs {
    const T* q;
    int64_t ldq;
    int n_rows, n_head, group, row_blocks, d, max_blocks, n_table_rows, window;
    CacheView<T> c;
    const int32_t* table;
    int64_t bt_stride;
    const int32_t *seq_of, *kv_len;
    float scale_log2;
    void* out;
    int64_t ldo;
    float* lse;
    uint32_t* counters;
    float* parts;
    uint32_t* err;
};

// The keys row r reads: [first, len) of request seq, in nt tiles from tile t0.
struct Span {
    int seq, first, len, t0, nt;
};
template <class T>
__device__ __forceinline__ Span span_of(const PagedArgs<T>& a, int r) {
    Span s;
    s.len = a.kv_len[r];
    s.seq = a.seq_of ? a.seq_of[r] : r;
    const int room = a.max_blocks << a.c.page_shift;   // fits: checked at the call
    if (s.seq == -1) s.len = 0;
    if (s.len < 0 || (s.len > 0 && (s.seq < 0 || s.seq >= a.n_table_rows))) {
        report(a.err, kDevBadPage);
        s.len = 0;
    }
    if (s.len > room) {
        report(a.err, kDevBadPage);
        s.len = room;
    }
    s.first = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
    s.t0 = s.first / kTile;
    s.nt = s.len > 0 ? (s.len - 1) / kTile + 1 - s.t0 : 0;
    return s;
}

// A place in the sequence of units: tile t of head-and-row-block hm of row r.
struct Cursor {
    int r, hm, t;
    Span s;
};
template <class T>
__device__ __forceinline__ void next_unit(const PagedArgs<T>& a, Cursor& c, int per_row) {
    if (++c.t < c.s.nt) return;
    c.t = 0;
    if (++c.hm < per_row) return;
    c.hm = 0;
    c.s.nt = 0;
    while (c.s.nt == 0 && ++c.r < a.n_rows) c.s = span_of(a, c.r);
}

template <class To>
__device__ __forceinline__ void store_out(To* p, float v) { *p = from_f32<To>(v); }

template <class T, class To, int DP, int kRows>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kCtas) paged_kernel(PagedArgs<T> a) {
    using S = Shape<DP>;
    constexpr int kSteps = DP / 16;           // of 16 elements in q.k
    constexpr int kCols = DP / 8;             // 8-wide column tiles of the output
    constexpr bool kPacked = kRows == 8;      // head and remainder share one operand
    // a third piece where a bf16 cache meets 32-bit results: 16 bits of a probability are not enough there
    constexpr bool kThird = std::is_same<T, __nv_bfloat16>::value && std::is_same<To, float>::value;
    // fp16 remainders of small probabilities stay in the normal range
    constexpr float kLift = std::is_same<T, __half>::value ? 10.0f : 0.0f;

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_valid[kWarps][S::kStages];
    __shared__ float s_ref[kWarps][16], s_sum[kWarps][16], s_row_ref[16], s_row_sum[16];
    __shared__ long long s_base[kWarps];
    __shared__ long long s_u0;
    __shared__ int s_row;
    __shared__ uint32_t s_last;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int per_row = (a.n_head / a.group) * a.row_blocks;
    float* s_out = reinterpret_cast<float*>(smem + kWarps * S::kStages * S::kStageBytes);
    const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStageBytes;

    // columns d..DP-1 of the shared rows stay zero for good
    if (a.d < DP)
        for (int i = tid; i < kWarps * S::kStages * S::kStageBytes / 16; i += kThreads)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);

    // ---- the units of all rows, and this CTA's share ----
    const int per = (a.n_rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.n_rows), r1 = min(r0 + per, a.n_rows);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += span_of(a, r).nt;
    long long incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) s_base[warp] = incl;
    __syncthreads();
    long long base = incl - mine, total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) base += s_base[w];
        total += s_base[w];
    }
    total *= per_row;
    base *= per_row;
    mine *= per_row;
    const long long ctas = min(static_cast<long long>(gridDim.x), total), cta = blockIdx.x;

    // rows with nothing to read
    for (int r = blockIdx.x * kWarps + warp; r < a.n_rows; r += gridDim.x * kWarps) {
        if (span_of(a, r).nt) continue;
        To* o = static_cast<To*>(a.out) + r * a.ldo;
        for (int i = lane; i < a.n_head * a.d; i += 32) store_out(o + i, 0.f);
        if (a.lse)
            for (int i = lane; i < a.n_head; i += 32) a.lse[static_cast<int64_t>(r) * a.n_head + i] = -INFINITY;
    }
    if (cta >= ctas) return;

    const long long u0 = total * cta / ctas, u1 = total * (cta + 1) / ctas;
    if (u0 >= base && u0 < base + mine) {   // exactly one thread
        long long b = base;
        for (int r = r0; r < r1; ++r) {
            const long long n = static_cast<long long>(span_of(a, r).nt) * per_row;
            if (u0 < b + n) {
                s_row = r;
                s_u0 = b;
                break;
            }
            b += n;
        }
    }
    __syncthreads();
    Cursor ld;
    ld.r = s_row;
    ld.s = span_of(a, ld.r);
    ld.hm = static_cast<int>((u0 - s_u0) / ld.s.nt);
    ld.t = static_cast<int>((u0 - s_u0) % ld.s.nt);
    Cursor cu = ld;
    const int n_units = static_cast<int>(min(u1 - u0, 0x7FFFFFFFll));
    long long group_u0 = u0 - cu.t;           // first unit of the current group

    // ---- loading: lane l < 16 looks up key l's page one tile ahead of its copies ----
    int pg = -1, key = 0;
    bool live = false;
    auto look_up = [&](int i) {
        live = false;
        if (i < n_units && lane < 16) {
            key = (ld.s.t0 + ld.t) * kTile + warp * 16 + lane;
            live = key >= ld.s.first && key < ld.s.len;
            if (live) pg = a.table[ld.s.seq * a.bt_stride + (key >> a.c.page_shift)];
        }
    };
    auto issue = [&](int i) {
        if (i < n_units) {
            bool ok = live && pg >= 0 && pg < a.c.n_pages;
            if (live && !ok) report(a.err, kDevBadPage);
            int64_t off = 0;
            if (ok)
                off = pg * a.c.page_stride + (ld.hm / a.row_blocks) * a.c.head_stride +
                      (key & a.c.page_mask) * a.c.token_stride;
            const uint32_t valid = __ballot_sync(0xffffffffu, ok);
            const int stage = i % S::kStages;
            if (lane == 0) s_valid[warp][stage] = valid;
            if (valid) {
                const int chunk = lane % S::kLanes;
                const uint32_t dst = ring + stage * S::kStageBytes + chunk * 16;
#pragma unroll
                for (int row0 = 0; row0 < 16; row0 += 32 / S::kLanes) {
                    const int row = row0 + lane / S::kLanes;
                    const int64_t o = __shfl_sync(0xffffffffu, off, row);
                    const bool in = (valid >> row) & 1;
                    if (chunk * 8 < a.d) {
                        cp_async_16(dst + row * S::kPitch, a.c.k + o + chunk * 8, in);
                        cp_async_16(dst + (16 + row) * S::kPitch, a.c.v + o + chunk * 8, in);
                    }
                }
            }
            next_unit(a, ld, per_row);
        }
        cp_commit();
    };
    if (a.d < DP) __syncthreads();            // the zeros are in place
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
        look_up(i);
        issue(i);
    }
    look_up(S::kStages - 1);

    uint32_t qf[kSteps][4];
    float o[kCols][4];
    float ref[2], sum[2];
    bool fresh = true;

    for (int i = 0; i < n_units; ++i) {
        issue(i + S::kStages - 1);
        look_up(i + S::kStages);
        if (fresh) {   // a new group: its queries, empty sums
            fresh = false;
            const int hk = cu.hm / a.row_blocks, q0 = (cu.hm % a.row_blocks) * kRows;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = q0 + g + 8 * x;
                const bool in = row < a.group && (x == 0 || !kPacked);
                const T* q = a.q + cu.r * a.ldq + static_cast<int64_t>(hk * a.group + (in ? row : 0)) * a.d;
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int col = k * 16 + y * 8 + 2 * t4;
                        qf[k][x + 2 * y] = in && col < a.d ? *reinterpret_cast<const uint32_t*>(q + col) : 0u;
                    }
                ref[x] = -INFINITY;
                sum[x] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
        }
        cp_wait<S::kStages - 1>();
        __syncwarp();
        const int stage = i % S::kStages;
        const uint32_t valid = s_valid[warp][stage];
        if (valid) {
            const uint32_t sk = ring + stage * S::kStageBytes, sv = sk + 16 * S::kPitch;
            float s[2][4] = {};
            const uint32_t ka = sk + ((lane & 7) + (lane >> 4) * 8) * S::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldsm_x4(b, ka + k * 32);
                mma_16816<T>(s[0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                mma_16816<T>(s[1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
            }
            constexpr int kHalves = kPacked ? 1 : 2;
            bool moved = false;
            float factor[2] = {1.f, 1.f};
#pragma unroll
            for (int x = 0; x < kHalves; ++x) {
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& v = s[n][2 * x + e];
                        v = (valid >> (n * 8 + 2 * t4 + e)) & 1 ? v * a.scale_log2 : -INFINITY;
                        mx = fmaxf(mx, v);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float nr = fmaxf(ref[x], mx - kLift);
                if (nr > ref[x]) {
                    factor[x] = exp2_approx(ref[x] - nr);
                    ref[x] = nr;
                    moved = true;
                }
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    o[n][0] *= factor[0];
                    o[n][1] *= factor[0];
                    o[n][2] *= factor[kPacked ? 0 : 1];
                    o[n][3] *= factor[kPacked ? 0 : 1];
                }
                sum[0] *= factor[0];
                sum[1] *= factor[1];
            }
            // p = 2^(s - ref), split into 16-bit pieces in operand order
            uint32_t hi[4], lo[4], th[4];
#pragma unroll
            for (int x = 0; x < kHalves; ++x) {
                const float rf = ref[x] == -INFINITY ? 0.f : ref[x];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p0 = exp2_approx(s[n][2 * x] - rf), p1 = exp2_approx(s[n][2 * x + 1] - rf);
                    sum[x] += p0 + p1;
                    const uint32_t h = pack2<T>(p0, p1);
                    const float2 hf = unpack2<T>(h);
                    const float d0 = p0 - hf.x, d1 = p1 - hf.y;
                    const uint32_t l = pack2<T>(d0, d1);
                    hi[x + 2 * n] = h;
                    lo[x + 2 * n] = l;
                    if constexpr (kThird) {
                        const float2 lf = unpack2<T>(l);
                        th[x + 2 * n] = pack2<T>(d0 - lf.x, d1 - lf.y);
                    }
                }
            }
            const uint32_t va = sv + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kPitch + (lane >> 4) * 16;
#pragma unroll
            for (int n = 0; n < kCols; n += 2) {
                uint32_t b[4];
                ldsm_x4_trans(b, va + n * 16);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t b0 = b[2 * y], b1 = b[2 * y + 1];
                    if constexpr (kPacked) {
                        mma_16816<T>(o[n + y], hi[0], lo[0], hi[2], lo[2], b0, b1);
                        if constexpr (kThird) mma_16816<T>(o[n + y], th[0], 0u, th[2], 0u, b0, b1);
                    } else {
                        mma_16816<T>(o[n + y], hi[0], hi[1], hi[2], hi[3], b0, b1);
                        mma_16816<T>(o[n + y], lo[0], lo[1], lo[2], lo[3], b0, b1);
                        if constexpr (kThird) mma_16816<T>(o[n + y], th[0], th[1], th[2], th[3], b0, b1);
                    }
                }
            }
        }
        __syncwarp();

        // ---- the end of a group, or of the share: join the warps ----
        const bool group_end = cu.t + 1 == cu.s.nt;
        if (group_end || i + 1 == n_units) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
                sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
                if (t4 == 0) {
                    s_ref[warp][g + 8 * x] = ref[x];
                    s_sum[warp][g + 8 * x] = sum[x];
                }
            }
            __syncthreads();
            float fac[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float m = -INFINITY;
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ref[w][g + 8 * x]);
                fac[x] = ref[x] == -INFINITY ? 0.f : exp2_approx(ref[x] - m);
            }
            if (tid < kRows) {
                float m = -INFINITY, l = 0.f;
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ref[w][tid]);
                for (int w = 0; w < kWarps; ++w)
                    l += s_ref[w][tid] == -INFINITY ? 0.f : s_sum[w][tid] * exp2_approx(s_ref[w][tid] - m);
                s_row_ref[tid] = m;
                s_row_sum[tid] = l;
            }
            for (int w = 0; w < kWarps; ++w) {   // in turn: a fixed order of the additions
                if (warp == w) {
#pragma unroll
                    for (int n = 0; n < kCols; ++n) {
                        float2* p = reinterpret_cast<float2*>(s_out + g * S::kOutPitch + n * 8 + 2 * t4);
                        if constexpr (kPacked) {
                            float2 v = make_float2((o[n][0] + o[n][2]) * fac[0], (o[n][1] + o[n][3]) * fac[0]);
                            if (w) v = make_float2(p->x + v.x, p->y + v.y);
                            *p = v;
                        } else {
                            float2* p8 = p + 4 * S::kOutPitch;
                            float2 v = make_float2(o[n][0] * fac[0], o[n][1] * fac[0]);
                            float2 v8 = make_float2(o[n][2] * fac[1], o[n][3] * fac[1]);
                            if (w) {
                                v = make_float2(p->x + v.x, p->y + v.y);
                                v8 = make_float2(p8->x + v8.x, p8->y + v8.y);
                            }
                            *p = v;
                            *p8 = v8;
                        }
                    }
                }
                __syncthreads();
            }
            const int hk = cu.hm / a.row_blocks, q0 = (cu.hm % a.row_blocks) * kRows;
            const int rows = min(kRows, a.group - q0), head0 = hk * a.group + q0;
            const bool whole = group_end && group_u0 >= u0;
            bool write = whole;
            const long long last_u = group_u0 + cu.s.nt - 1;
            const int c0 = static_cast<int>(((group_u0 + 1) * ctas - 1) / total);
            const int c1 = static_cast<int>(((last_u + 1) * ctas - 1) / total);
            const int n_parts = c1 - c0 + 1;
            constexpr int kPart = part_floats<DP, kRows>();
            if (!whole) {
                float* part = a.parts + (2 * cta + (group_u0 >= u0 ? 1 : 0)) * kPart;
                for (int e = tid; e < rows * (DP / 4); e += kThreads) {
                    const int row = e / (DP / 4), c = e % (DP / 4) * 4;
                    __stcg(reinterpret_cast<float4*>(part + row * DP + c),
                           *reinterpret_cast<const float4*>(s_out + row * S::kOutPitch + c));
                }
                if (tid < rows) {
                    __stcg(part + kRows * DP + tid, s_row_ref[tid]);
                    __stcg(part + kRows * DP + kRows + tid, s_row_sum[tid]);
                }
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    const uint32_t before = atomicAdd(a.counters + c0, 1u);
                    s_last = before + 1 == static_cast<uint32_t>(n_parts);
                    if (s_last) a.counters[c0] = 0;   // for the next launch: all parts have arrived
                }
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    const auto part_of = [&](int p) {
                        return a.parts + (2 * static_cast<int64_t>(c0 + p) + (p == 0 ? 1 : 0)) * kPart;
                    };
                    for (int row = warp; row < rows; row += kWarps) {
                        float m = -INFINITY, l = 0.f;
                        for (int p = lane; p < n_parts; p += 32) m = fmaxf(m, __ldcg(part_of(p) + kRows * DP + row));
                        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                        for (int p = lane; p < n_parts; p += 32) {
                            const float* q = part_of(p) + kRows * DP + row;
                            const float rf = __ldcg(q);
                            l += rf == -INFINITY ? 0.f : __ldcg(q + kRows) * exp2_approx(rf - m);
                        }
                        for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
                        if (lane == 0) {
                            s_row_ref[row] = m;
                            s_row_sum[row] = l;
                        }
                    }
                    __syncthreads();
                    for (int e = tid; e < rows * (DP / 4); e += kThreads) {
                        const int row = e / (DP / 4), c = e % (DP / 4) * 4;
                        const float m = s_row_ref[row];
                        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                        for (int p = 0; p < n_parts; ++p) {
                            const float* q = part_of(p);
                            const float rf = __ldcg(q + kRows * DP + row);
                            const float f = rf == -INFINITY ? 0.f : exp2_approx(rf - m);
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(q + row * DP + c));
                            acc.x = fmaf(f, v.x, acc.x);
                            acc.y = fmaf(f, v.y, acc.y);
                            acc.z = fmaf(f, v.z, acc.z);
                            acc.w = fmaf(f, v.w, acc.w);
                        }
                        *reinterpret_cast<float4*>(s_out + row * S::kOutPitch + c) = acc;
                    }
                    __syncthreads();
                    write = true;
                }
            }
            if (write) {
                To* out = static_cast<To*>(a.out) + cu.r * a.ldo + static_cast<int64_t>(head0) * a.d;
                for (int e = tid; e < rows * DP; e += kThreads) {
                    const int row = e / DP, c = e % DP;
                    const float l = s_row_sum[row], v = s_out[row * S::kOutPitch + c];
                    if (c < a.d) store_out(out + static_cast<int64_t>(row) * a.d + c, l == 0.f ? 0.f : v / l);
                }
                if (a.lse && tid < rows) {
                    const float l = s_row_sum[tid];
                    a.lse[static_cast<int64_t>(cu.r) * a.n_head + head0 + tid] =
                        l == 0.f ? -INFINITY : (s_row_ref[tid] + log2f(l)) * 0.69314718055994531f;
                }
            }
            __syncthreads();   // s_out and the sums are free again
            fresh = true;
        }
        if (group_end) group_u0 += cu.s.nt;
        next_unit(a, cu, per_row);
    }
}

// Head width and query rows as the kernel is built for them.
int padded_width(int d) { return d <= 64 ? 64 : d <= 80 ? 80 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

// fn(DP, rows of a block) of the variant for a head width and group: 8 query rows
// where they suffice (head and remainder of a probability in one operand), else 16.
template <class Fn>
auto with_shape(int d, int group, Fn fn) {
    auto rows = [&](auto dp) {
        return group <= 8 ? fn(dp, std::integral_constant<int, 8>{}) : fn(dp, std::integral_constant<int, 16>{});
    };
    switch (padded_width(d)) {
        case 64: return rows(std::integral_constant<int, 64>{});
        case 80: return rows(std::integral_constant<int, 80>{});
        case 96: return rows(std::integral_constant<int, 96>{});
        case 128: return rows(std::integral_constant<int, 128>{});
        case 192: return rows(std::integral_constant<int, 192>{});
        default: return rows(std::integral_constant<int, 256>{});
    }
}

int grid_of(int num_sms, int ctas) { return num_sms * ctas < kMaxCtas ? num_sms * ctas : kMaxCtas; }

}  // namespace
}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_attention_paged_scratch_bytes(int32_t n_head, int32_t n_kv_head, int32_t d_head) {
    if (n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head || d_head <= 0 || d_head > 256) return 0;
    DeviceState* ds = state();
    const int sms = ds ? ds->num_sms : 148;
    return with_shape(d_head, n_head / n_kv_head, [&](auto dp, auto rows) {
        constexpr int kPart = part_floats<decltype(dp)::value, decltype(rows)::value>();
        return kCounterBytes + sizeof(float) * 2 * kPart * grid_of(sms, Shape<decltype(dp)::value>::kCtas);
    });
}

b2q_status b2q_attention_paged(const void* q, int64_t ldq, int64_t n_rows, int32_t n_head, const b2q_kv_cache* cache,
                               const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                               int32_t n_table_rows, const int32_t* seq_of, const int32_t* kv_len, float scale,
                               int32_t window, void* out, int32_t out_dtype, int64_t ldo, float* lse, void* scratch,
                               void* stream) {
    B2Q_REQUIRE_STATE();
    b2q_kv_cache c;
    b2q_status st = check_cache(cache, &c);
    if (st) return st;
    if (out_dtype != B2Q_TYPE_F32 && out_dtype != c.dtype)
        return set_error(B2Q_ERR_INVALID, "out must be F32 or the cache's type");
    if (n_rows < 0 || n_rows > (1 << 20) || n_head <= 0 || n_head > 65535 || n_head % c.n_kv_head)
        return set_error(B2Q_ERR_SHAPE, "bad n_rows / n_head");
    if (ldq < static_cast<int64_t>(n_head) * c.d_head || ldo < static_cast<int64_t>(n_head) * c.d_head)
        return set_error(B2Q_ERR_SHAPE, "row strides shorter than the heads");
    if (max_blocks < 0 || bt_stride < max_blocks || n_table_rows < 0)
        return set_error(B2Q_ERR_SHAPE, "bad block table width / stride / rows");
    if (static_cast<int64_t>(max_blocks) * c.page_size > INT32_MAX)
        return set_error(B2Q_ERR_SHAPE, "block table rows hold more tokens than an int32");
    if (!seq_of && n_rows > n_table_rows) return set_error(B2Q_ERR_SHAPE, "more rows than block table rows");
    if (!std::isfinite(scale) || window < 0) return set_error(B2Q_ERR_INVALID, "bad scale / window");
    if (n_rows == 0) return B2Q_OK;
    if (!q || !kv_len || !out || !scratch || (max_blocks > 0 && n_table_rows > 0 && !block_table))
        return set_error(B2Q_ERR_INVALID, "null pointer");
    if (!ptr_aligned(scratch, 256)) return set_error(B2Q_ERR_ALIGN, "scratch must be 256-byte aligned");
    if (ldq % 8 || !ptr_aligned(q, 16)) return set_error(B2Q_ERR_ALIGN, "query rows need 16-byte alignment");
    if (!ptr_aligned(out, out_dtype == B2Q_TYPE_F32 ? 4 : 2)) return set_error(B2Q_ERR_ALIGN, "misaligned out");
    const int group = n_head / c.n_kv_head;
    auto go = [&](auto t, auto to) {
        using T = decltype(t);
        using To = decltype(to);
        return with_shape(c.d_head, group, [&](auto dp, auto rows) {
            constexpr int DP = decltype(dp)::value, kRows = decltype(rows)::value;
            constexpr size_t smem = smem_bytes<DP, kRows>();
            PagedArgs<T> a{static_cast<const T*>(q), ldq, static_cast<int>(n_rows), n_head, group,
                           (group + kRows - 1) / kRows, c.d_head, max_blocks, n_table_rows, window, view_of<T>(c),
                           block_table, bt_stride, seq_of, kv_len, scale * 1.44269504088896340736f, out, ldo, lse,
                           static_cast<uint32_t*>(scratch),
                           reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + kCounterBytes), ds->err};
            auto* kernel = paged_kernel<T, To, DP, kRows>;
            static std::atomic<uint64_t> allowed{0};
            const b2q_status s = allow_smem(kernel, static_cast<int>(smem), allowed, ds->device);
            if (s) return s;
            kernel<<<grid_of(ds->num_sms, Shape<DP>::kCtas), kThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
            count_launch();
            return cuda_check(cudaGetLastError(), "paged attention launch");
        });
    };
    auto with_out = [&](auto t) { return out_dtype == B2Q_TYPE_F32 ? go(t, float{}) : go(t, t); };
    return c.dtype == B2Q_TYPE_F16 ? with_out(__half{}) : with_out(__nv_bfloat16{});
}

}  // extern "C"
