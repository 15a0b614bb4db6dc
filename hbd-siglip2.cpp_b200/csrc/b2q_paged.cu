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
// Work split.  A unit is a tile of 64 to 128 keys (16 a warp) of one (row, key head, block of query
// rows).  The units of all rows in order are dealt to a fixed grid of CTAs in
// equal contiguous shares, whatever the lengths: one request of 100,000 keys
// and hundreds of ragged ones load every SM alike, lengths are read on the
// device, and a captured launch stays valid as they grow.  A CTA's share holds
// the end of one group, whole groups, and the start of another; what is not
// whole goes to scratch as a partial result.  At its end the CTA reports its one or
// two partial groups, and the last to report a group joins the parts in their order
// whichever CTA that is (so the bits repeat).  Nobody waits.
//
// Inside a CTA each of four to eight warps takes 16 keys of every tile and keeps its own
// ref, sum and output; they meet only where a group ends, each leaving its output
// in the ring slot that it has just read.  Keys and values come by 16-byte
// asynchronous copies, each warp filling its own ring of stages, so loads run on
// across tiles, groups and rows with no block barrier; page ids are looked up a tile
// before they are needed.  Shared rows have an odd number of 16-byte chunks, which
// keeps ldmatrix free of bank conflicts for every head width.
//
// Products run on mma.sync (16 query rows x 8 keys): a decode step has 1 to 16
// query rows per key head, far from the 64 to 128 of a tcgen05 tile, and the
// bytes bind long before the tensor pipe.  Probabilities enter the second
// product as a 16-bit head and remainder(s), 22 to 24 bits in all: rounding
// them to 16 bits would cost as much as the output's own rounding.  With at
// most 8 query rows the head takes rows 0-7 of the operand and the remainder
// rows 8-15, so the exact product costs no more instructions than the rounded
// one would.  The tensor core cuts its sums off rather than rounding them, so a tile's
// products are summed from zero there and added to the output in fp32: a chain over
// thousands of keys would shrink it (131,071 keys: relative error 4.0e-6 against 1.1e-6).
//
// Measured on one B200 (copy bandwidth 6.53 TB/s), device time: 3 requests of 131,071
// keys, 40/8 heads of 128, fp16, 1.61 GB: 270 us, 6.0 TB/s; 61 ragged ones of 17 to 8,191,
// 32/8 heads of 128, bf16, 0.99 GB: 167 us, 5.9 TB/s; 256 rows with a window of 1,024, 8/1
// heads of 256, 264 MB: 62 us, 4.3 TB/s (with four warps and three stages 70, as one warp a
// scheduler waits for its own products); one request of 997 keys, 16 heads of 72: 9.1 us,
// round trips one after the other.  Two stages or three a warp: 268 and 275, 166 and 169 us.
#include "b2q_decode.cuh"

#include <cmath>
#include <type_traits>

namespace b2q {
namespace {

constexpr int kMaxCtas = 444;          // three per SM of a full GPU (148)
constexpr size_t kCounterBytes = 2048;   // a join counter per CTA, at the start of the scratch

// Per head width (padded to DP): warps of a CTA and CTAs per SM.  Two stages a warp are
// enough bytes in flight; what the 227 KB of shared memory and the registers hold beyond
// that goes to more warps.
template <int DP>
struct Shape {
    static constexpr int kChunks = (DP / 8) | 1;            // 16-byte chunks of a shared row
    static constexpr int kPitch = kChunks * 16;
    static constexpr int kStageBytes = 2 * 16 * kPitch;     // one warp's keys and values
    static constexpr int kStages = 2;
    static constexpr int kWarps = DP > 192 ? 6 : (DP > 128 ? 8 : 4);
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kTile = 16 * kWarps;               // keys of a unit
    static constexpr int kCtas = DP > 128 ? 1 : (DP > 64 ? 2 : 3);
    static constexpr int kLanes = DP <= 64 ? 8 : (DP <= 128 ? 16 : 32);   // lanes that copy one row
    static constexpr int kOutPitch = DP + 8;
    static_assert(16 * kOutPitch * 4 <= kStageBytes, "a warp's output fits the ring slot that it has just read");
};
// The ring, which at the end also holds a join's weights, sums and half-way outputs.
template <int DP, int kRows>
constexpr int smem_bytes() {
    constexpr int ring = Shape<DP>::kWarps * Shape<DP>::kStages * Shape<DP>::kStageBytes;
    constexpr int join = 2 * kRows * (kMaxCtas + 2) * 4 + 2 * Shape<DP>::kThreads * 16;
    return ring > join ? ring : join;
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
template <int kTile, class T>
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
template <int kTile, class T>
__device__ __forceinline__ void next_unit(const PagedArgs<T>& a, Cursor& c, int per_row) {
    if (++c.t < c.s.nt) return;
    c.t = 0;
    if (++c.hm < per_row) return;
    c.hm = 0;
    c.s.nt = 0;
    while (c.s.nt == 0 && ++c.r < a.n_rows) c.s = span_of<kTile>(a, c.r);
}

// x / y for y that fits an int: 32-bit wherever x does too (64-bit division is some
// hundred dependent instructions, and the start of a short call waits for it).
__device__ __forceinline__ long long divide(long long x, int y) {
    return x <= 0xFFFFFFFFll ? static_cast<long long>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y)) : x / y;
}
// `total` units dealt to `ctas` CTAs in contiguous shares that differ by one at most.
struct Shares {
    long long each;
    int more, ctas;   // the first `more` CTAs have one unit more
    __device__ __forceinline__ void init(long long total, int grid) {
        ctas = total < grid ? static_cast<int>(total) : grid;
        each = ctas ? divide(total, ctas) : 0;
        more = static_cast<int>(total - each * ctas);
    }
    __device__ __forceinline__ long long start(int cta) const { return each * cta + min(cta, more); }
    __device__ __forceinline__ int owner(long long u) const {
        const long long first = (each + 1) * more;   // units of the longer shares
        if (each > 0x7FFFFFFEll) return static_cast<int>(u < first ? u / (each + 1) : more + (u - first) / each);
        return static_cast<int>(u < first ? divide(u, static_cast<int>(each) + 1)
                                          : more + divide(u - first, static_cast<int>(each)));
    }
};
struct Start {
    int r;
    long long in_row;   // units before the share within row r
    Span s;
};
struct Partial {
    int live, r, head0, rows, nt;
    long long u0;       // the group's first unit
    int c0;             // and the CTA that has it
};

__device__ __forceinline__ uint32_t add_acq_rel(uint32_t* p, uint32_t v) {
    uint32_t old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}

// What stands for an element whose sum is NaN although every weight is a number: then
// values that are none are among those weighted, and what they make is looked at again
// at the end (no arithmetic or conversion yields this NaN).
template <class To>
__device__ __forceinline__ To open_mark();
template <>
__device__ __forceinline__ float open_mark<float>() { return __uint_as_float(0x7FC0B2B2u); }
template <>
__device__ __forceinline__ __half open_mark<__half>() { return __ushort_as_half(0x7EB2u); }
template <>
__device__ __forceinline__ __nv_bfloat16 open_mark<__nv_bfloat16>() { return __ushort_as_bfloat16(0x7FD2u); }
__device__ __forceinline__ bool is_open(float x) { return __float_as_uint(x) == 0x7FC0B2B2u; }
__device__ __forceinline__ bool is_open(__half x) { return __half_as_ushort(x) == 0x7EB2u; }
__device__ __forceinline__ bool is_open(__nv_bfloat16 x) { return __bfloat16_as_ushort(x) == 0x7FD2u; }

// v f, f = 1 / l, for a sum of l; no key: zeros.  Sets *open where it leaves a mark.
template <class To, class T>
__device__ __forceinline__ void write_out(const PagedArgs<T>& a, int r, int head, int c, float4 v, float l, float f,
                                          uint32_t* open) {
    if (c >= a.d) return;   // d is a multiple of 8
    To* o = static_cast<To*>(a.out) + r * a.ldo + static_cast<int64_t>(head) * a.d + c;
    v = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    o[0] = from_f32<To>(v.x);
    o[1] = from_f32<To>(v.y);
    o[2] = from_f32<To>(v.z);
    o[3] = from_f32<To>(v.w);
    if ((v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w) && l == l) {
        *open = 1;
        if (v.x != v.x) o[0] = open_mark<To>();
        if (v.y != v.y) o[1] = open_mark<To>();
        if (v.z != v.z) o[2] = open_mark<To>();
        if (v.w != v.w) o[3] = open_mark<To>();
    }
}

// The marks in the results of `rows` query heads (of one key head) from head0 of row r,
// all threads of the CTA: a probability's remainder is zero or negative as often as not,
// and makes NaN of an infinity that the probability would leave alone.  By the definition
// infinities of one sign make that infinity; both signs, or a NaN, make NaN.  Reads the
// row's values once more where there is a mark (3 x 131,071 keys, one infinity: 3.7 ms
// a call).  flags: one word a column, shared.
template <class To, class T>
__device__ __noinline__ void settle(const PagedArgs<T>& a, int r, int head0, int rows, uint32_t* flags) {
    constexpr int kTogether = 16;   // loads of a thread in flight
    const int tid = threadIdx.x, n = rows * a.d;
    To* out = static_cast<To*>(a.out) + r * a.ldo + static_cast<int64_t>(head0) * a.d;
    bool any = false;
    for (int i = tid; i < n; i += blockDim.x) any |= is_open(out[i]);
    if (!__syncthreads_or(any)) return;
    for (int c = tid; c < a.d; c += blockDim.x) flags[c] = 0;
    __syncthreads();
    const Span s = span_of<64>(a, r);
    const int chunks = a.d / 8, step = blockDim.x / chunks, c = tid % chunks * 8;
    const T* col = a.c.v + head0 / a.group * a.c.head_stride + c;
    uint32_t seen[8] = {};   // 1: +inf, 2: -inf, 4: NaN, of column c + e
    if (tid / chunks < step && tid / chunks < s.len - s.first)
        for (int key0 = s.first + tid / chunks; key0 < s.len;
             key0 = s.len - key0 > kTogether * step ? key0 + kTogether * step : s.len) {
            uint4 raw[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {   // (the first key again behind the end: nothing new)
                const int key = k * step < s.len - key0 ? key0 + k * step : key0;
                const int page = a.table[s.seq * a.bt_stride + (key >> a.c.page_shift)];
                const bool ok = page >= 0 && page < a.c.n_pages;
                const T* p = col + (ok ? page : 0) * a.c.page_stride + (key & a.c.page_mask) * a.c.token_stride;
                raw[k] = ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 x2 = unpack2<T>(w[e / 2]);
                    const float x = e % 2 ? x2.y : x2.x;
                    seen[e] |= (x == INFINITY ? 1u : 0u) | (x == -INFINITY ? 2u : 0u) | (x != x ? 4u : 0u);
                }
            }
        }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (seen[e]) atomicOr(flags + c + e, seen[e]);
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x)
        if (is_open(out[i])) {
            const uint32_t f = flags[i % a.d];
            out[i] = from_f32<To>(f == 1 ? INFINITY : f == 2 ? -INFINITY : __uint_as_float(0x7FFFFFFFu));
        }
}
template <class T>
__device__ __forceinline__ void write_lse(const PagedArgs<T>& a, int r, int head, float ref, float l) {
    if (a.lse)
        a.lse[static_cast<int64_t>(r) * a.n_head + head] =
            l == 0.f ? -INFINITY : (ref + log2f(l)) * 0.69314718055994531f;
}

template <class T, class To, int DP, int kRows>
__global__ void __launch_bounds__(Shape<DP>::kThreads, Shape<DP>::kCtas) paged_kernel(const __grid_constant__ PagedArgs<T> a) {
    using S = Shape<DP>;
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTile = S::kTile;
    constexpr int kSteps = DP / 16;           // of 16 elements in q.k
    constexpr int kCols = DP / 8;             // 8-wide column tiles of the output
    constexpr bool kPacked = kRows == 8;      // head and remainder share one operand
    // a third piece where a bf16 cache meets 32-bit results: 16 bits of a probability are not enough there
    constexpr bool kThird = std::is_same<T, __nv_bfloat16>::value && std::is_same<To, float>::value;
    // fp16 remainders of small probabilities stay in the normal range
    constexpr float kLift = std::is_same<T, __half>::value ? 10.0f : 0.0f;

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_valid[kWarps][S::kStages];
    __shared__ float s_ref[kWarps][16], s_sum[kWarps][16];
    __shared__ long long s_base[kWarps];
    __shared__ Start s_start;
    __shared__ Partial s_partial[2];
    __shared__ uint32_t s_last[2], s_open;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int per_row = (a.n_head / a.group) * a.row_blocks;
    const int ring_at = warp * S::kStages * S::kStageBytes;
    const uint32_t ring = smem_u32(smem) + ring_at;
    constexpr int kPart = part_floats<DP, kRows>();

    // columns d..DP-1 of the shared rows stay zero for good
    if (a.d < DP) {
        const int from = a.d / 8, n = S::kChunks - from;
        for (int i = tid; i < kWarps * S::kStages * 32 * n; i += kThreads)
            *reinterpret_cast<uint4*>(smem + i / n * S::kPitch + (from + i % n) * 16) = make_uint4(0, 0, 0, 0);
    }
    if (tid < 2) s_partial[tid].live = 0;
    if (tid == 0) s_open = 0;
    let_next_start();
    wait_for_previous();

    // ---- the units of all rows, and this CTA's share ----
    const int per = (a.n_rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.n_rows), r1 = min(r0 + per, a.n_rows);
    Span mine_span{};
    long long mine = 0;
    for (int r = r0; r < r1; ++r) {
        mine_span = span_of<kTile>(a, r);
        mine += mine_span.nt;
    }
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
    Shares sh;
    sh.init(total * per_row, gridDim.x);
    const bool works = static_cast<int>(blockIdx.x) < sh.ctas;
    const long long u0 = sh.start(blockIdx.x), u1 = sh.start(blockIdx.x + 1);
    base *= per_row;
    if (works && u0 >= base && u0 < base + mine * per_row) {   // exactly one thread
        for (int r = r0; r < r1; ++r) {
            if (per > 1) mine_span = span_of<kTile>(a, r);
            const long long n = static_cast<long long>(mine_span.nt) * per_row;
            if (u0 < base + n) {
                s_start = Start{r, u0 - base, mine_span};
                break;
            }
            base += n;
        }
    }
    __syncthreads();

    if (works) {
        Cursor ld;
        ld.r = s_start.r;
        ld.s = s_start.s;
        ld.hm = static_cast<int>(divide(s_start.in_row, ld.s.nt));
        ld.t = static_cast<int>(s_start.in_row - static_cast<long long>(ld.hm) * ld.s.nt);
        Cursor cu = ld;
        const int n_units = static_cast<int>(min(u1 - u0, 0x7FFFFFFFll));
        long long group_u0 = u0 - cu.t;           // first unit of the current group

        // ---- loading: a warp's 16 keys are looked up one tile ahead of their copies ----
        struct Pending {
            int page;        // of lane's key (of all 16 where a page holds that many), -1 = none
            uint32_t live;   // the 16 keys that are the row's
            int64_t rest;    // offset of head and row within the page: of lane's key, or of the first
        };
        const bool one_page = a.c.page_mask >= 15;
        int looked = 0;
        auto look_up = [&]() {
            Pending p{-1, 0u, 0};
            if (looked < n_units) {
                ++looked;
                const int tile0 = (ld.s.t0 + ld.t) * kTile;   // below len; a warp's keys may pass an int32 behind it
                const int lo = max(ld.s.first - tile0 - warp * 16, 0), hi = min(ld.s.len - tile0 - warp * 16, 16);
                if (lo < hi) p.live = ((1u << hi) - 1) & ~((1u << lo) - 1);
                const int key = static_cast<int>(static_cast<uint32_t>(tile0) + warp * 16 + (one_page ? 0 : lane));
                const bool mine = one_page ? p.live != 0 : lane < 16 && ((p.live >> lane) & 1);
                if (mine) p.page = a.table[ld.s.seq * a.bt_stride + (key >> a.c.page_shift)];
                const int head = a.row_blocks == 1 ? ld.hm : ld.hm / a.row_blocks;
                p.rest = head * a.c.head_stride + (key & a.c.page_mask) * a.c.token_stride;
                next_unit<kTile>(a, ld, per_row);
            }
            return p;
        };
        const int chunk = lane % S::kLanes, row_of_lane = lane / S::kLanes;
        const bool copies = chunk * 8 < a.d;
        auto issue = [&](const Pending& p, int stage) {
            const bool ok = p.page >= 0 && p.page < a.c.n_pages;
            const int64_t off = (ok ? p.page : 0) * a.c.page_stride + p.rest;
            uint32_t valid = p.live;
            if (one_page) {
                if (!ok && valid) {
                    if (lane == 0) report(a.err, kDevBadPage);
                    valid = 0;
                }
            } else {
                if (!ok && lane < 16 && ((p.live >> lane) & 1)) report(a.err, kDevBadPage);
                valid &= __ballot_sync(0xffffffffu, ok);
            }
            if (lane == 0) s_valid[warp][stage] = valid;
            if (valid) {
                const uint32_t dst = ring + stage * S::kStageBytes + row_of_lane * S::kPitch + chunk * 16;
                constexpr int kStep = 32 / S::kLanes;   // rows of one copy instruction
                if (one_page) {
                    const T* k = a.c.k + off + row_of_lane * a.c.token_stride + chunk * 8;
                    const T* v = a.c.v + off + row_of_lane * a.c.token_stride + chunk * 8;
#pragma unroll
                    for (int row = 0; row < 16; row += kStep) {
                        const bool in = (valid >> (row + row_of_lane)) & 1;
                        if (copies) {
                            cp_async_16(dst + row * S::kPitch, k, in);
                            cp_async_16(dst + (16 + row) * S::kPitch, v, in);
                        }
                        k += kStep * a.c.token_stride;
                        v += kStep * a.c.token_stride;
                    }
                } else {
#pragma unroll
                    for (int row = 0; row < 16; row += kStep) {
                        const int64_t o = __shfl_sync(0xffffffffu, off, row + row_of_lane);
                        const bool in = (valid >> (row + row_of_lane)) & 1;
                        if (copies) {   // (a row that is not read is named by the cache's first)
                            cp_async_16(dst + row * S::kPitch, a.c.k + (in ? o : 0) + chunk * 8, in);
                            cp_async_16(dst + (16 + row) * S::kPitch, a.c.v + (in ? o : 0) + chunk * 8, in);
                        }
                    }
                }
            }
            cp_commit();
        };
        uint32_t qf[kSteps][4];
        constexpr int kHalves = kPacked ? 1 : 2;   // sets of 8 query rows
        float o[kCols][2 * kHalves];
        float ref[2], sum[2];
        auto new_group = [&]() {   // its queries, empty sums
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
                for (int x = 0; x < 2 * kHalves; ++x) o[n][x] = 0.f;
        };
        Pending next = look_up();
        bool fresh = true;
        int stage = 1;   // of tile i; tile i + kStages - 1 goes to the one before it

        // (The ring is filled by the same instructions: code that runs once is fetched at
        // memory latency, and a few warps have nothing to hide that behind.)
#pragma unroll 1
        for (int i = 1 - S::kStages; i < n_units; ++i) {
            issue(next, stage == 0 ? S::kStages - 1 : stage - 1);
            next = look_up();
            if (fresh) {   // (at the start: before the rest of the ring's keys fill the queues)
                fresh = false;
                new_group();
            }
            if (i < 0) {
                if (++stage == S::kStages) stage = 0;
                continue;
            }
            cp_wait<S::kStages - 1>();
            __syncwarp();
            const uint32_t valid = s_valid[warp][stage];
            if (valid) {
                const uint32_t sk = ring + stage * S::kStageBytes, sv = sk + 16 * S::kPitch;
                float sc[2][2][4] = {};   // two chains of dependent products a result
                const uint32_t ka = sk + ((lane & 7) + (lane >> 4) * 8) * S::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t b[4];
                    ldsm_x4(b, ka + k * 32);
                    mma_16816<T>(sc[k % 2][0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                    mma_16816<T>(sc[k % 2][1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
                }
                float (&s)[2][4] = sc[0];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] += sc[1][n][x];
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
                    for (int n = 0; n < kCols; ++n)
#pragma unroll
                        for (int x = 0; x < 2 * kHalves; ++x) o[n][x] *= factor[x / 2];
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
                        float d[4] = {};
                        if constexpr (kPacked) {
                            if constexpr (kThird) mma_16816<T>(d, th[0], 0u, th[2], 0u, b0, b1);
                            mma_16816<T>(d, hi[0], lo[0], hi[2], lo[2], b0, b1);
                            o[n + y][0] += d[0] + d[2];
                            o[n + y][1] += d[1] + d[3];
                        } else {
                            if constexpr (kThird) mma_16816<T>(d, th[0], th[1], th[2], th[3], b0, b1);
                            mma_16816<T>(d, lo[0], lo[1], lo[2], lo[3], b0, b1);
                            mma_16816<T>(d, hi[0], hi[1], hi[2], hi[3], b0, b1);
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[n + y][x] += d[x];
                        }
                    }
                }
            }
            __syncwarp();

            // ---- the end of a group, or of the share: join the warps ----
            const bool group_end = cu.t + 1 == cu.s.nt;
            if (group_end || i + 1 == n_units) {
                // into the slot that has just been read: nothing fills it before the next tile
                const int slot_at = stage * S::kStageBytes;
                float* so = reinterpret_cast<float*>(smem + ring_at + slot_at) + g * S::kOutPitch + 2 * t4;
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    *reinterpret_cast<float2*>(so + n * 8) = make_float2(o[n][0], o[n][1]);
                    if constexpr (!kPacked)
                        *reinterpret_cast<float2*>(so + 8 * S::kOutPitch + n * 8) = make_float2(o[n][2], o[n][3]);
                }
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
                const int hk = cu.hm / a.row_blocks, q0 = (cu.hm % a.row_blocks) * kRows;
                const int rows = min(kRows, a.group - q0), head0 = hk * a.group + q0;
                const bool starts_here = group_u0 >= u0, whole = group_end && starts_here;
                float* part = a.parts + (2 * static_cast<int64_t>(blockIdx.x) + starts_here) * kPart;
                for (int e = tid; e < rows * (DP / 4); e += kThreads) {
                    const int row = e / (DP / 4), c = e % (DP / 4) * 4;
                    float m = s_ref[0][row], l = 0.f;
#pragma unroll
                    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_ref[w][row]);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float rw = s_ref[w][row], f = rw == -INFINITY ? 0.f : exp2_approx(rw - m);
                        const float4 x = *reinterpret_cast<const float4*>(
                            smem + w * S::kStages * S::kStageBytes + slot_at + (row * S::kOutPitch + c) * 4);
                        l = fmaf(f, s_sum[w][row], l);
                        v.x = fmaf(f, x.x, v.x);
                        v.y = fmaf(f, x.y, v.y);
                        v.z = fmaf(f, x.z, v.z);
                        v.w = fmaf(f, x.w, v.w);
                    }
                    if (whole) {
                        write_out<To>(a, cu.r, head0 + row, c, v, l, 1.0f / l, &s_open);
                        if (c == 0) write_lse(a, cu.r, head0 + row, m, l);
                    } else {
                        __stcg(reinterpret_cast<float4*>(part + row * DP + c), v);
                        if (c == 0) {
                            __stcg(part + kRows * DP + row, m);
                            __stcg(part + kRows * DP + kRows + row, l);
                        }
                    }
                }
                if (!whole && tid == 0) s_partial[starts_here] = Partial{1, cu.r, head0, rows, cu.s.nt, group_u0};
                __syncthreads();   // the slots, refs and sums are free again
                if (a.d < DP) {    // ... and the slot's padding columns zero again
                    const int from = a.d / 8;
                    for (int e = lane; e < 32 * (S::kChunks - from); e += 32)
                        *reinterpret_cast<uint4*>(smem + ring_at + slot_at + e / (S::kChunks - from) * S::kPitch +
                                                  (from + e % (S::kChunks - from)) * 16) = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
                fresh = true;
            }
            if (group_end) group_u0 += cu.s.nt;
            next_unit<kTile>(a, cu, per_row);
            if (++stage == S::kStages) stage = 0;
        }

        // ---- report the partial groups; the last to report one joins it ----
        // (the parts are all threads' stores: the group's barrier orders them before
        // this thread's release, its acquire before what the next barrier lets run)
        if (lane == 0 && warp < 2) {
            Partial& pt = s_partial[warp];
            int parts = 0;
            if (pt.live) {
                pt.c0 = sh.owner(pt.u0);
                const int n = sh.owner(pt.u0 + pt.nt - 1) - pt.c0 + 1;
                if (add_acq_rel(a.counters + pt.c0, 1u) + 1 == static_cast<uint32_t>(n)) {
                    a.counters[pt.c0] = 0;   // for the next launch: all parts have arrived
                    parts = n;
                }
            }
            s_last[warp] = parts;
        }
        __syncthreads();
        // One group: all threads join it.  Two: half of the threads each.
        const int n0 = s_last[0], n1 = s_last[1], teams = (n0 != 0) + (n1 != 0);
        if (teams) {
            const int team_threads = kThreads / teams, team = tid / team_threads, me = tid % team_threads;
            const int x = teams == 2 ? team : n0 ? 0 : 1;
            const Partial pt = s_partial[x];
            const int n_parts = x ? n1 : n0, n_out = pt.rows * (DP / 4);
            const auto part_of = [&](int p) {
                return a.parts + (2 * static_cast<int64_t>(pt.c0 + p) + (p == 0 ? 1 : 0)) * kPart;
            };
            // shared: per team refs (then weights) and sums of all parts, and half-way outputs (the ring is free now)
            constexpr int kTeamFloats = 2 * kRows * (kMaxCtas + 2);
            float* wt = reinterpret_cast<float*>(smem) + (x ? 2 * kRows * (n0 ? n0 : 0) : 0);
            float* sm = wt + n_parts * pt.rows;
            float4* red = reinterpret_cast<float4*>(smem + kTeamFloats * 4) + team * kThreads;
            // Few outputs: the parts too are dealt to `subs` sums of an output, added up in
            // a second step.  Their number goes by the sizes alone and not by the team at
            // hand, which depends on who reported last: half the threads take two each.
            const int half = kThreads / 2 / n_out;
            const int subs = half ? min(2 * half, n_parts) : 1;
            const int at_once = half ? min(team_threads / n_out, subs) : 1;
            const int sub = subs > 1 ? me / n_out : 0, e0 = subs > 1 ? me % n_out : me;
            constexpr int kEach = (kRows * DP / 4 + kThreads / 2 - 1) / (kThreads / 2);   // outputs of a thread, at most
            constexpr int kFirst = kEach <= 8 ? 2 : 1;   // its parts that are asked for at once, with the refs
            float4 early[kFirst][kEach];
#pragma unroll
            for (int k = 0; k < kFirst; ++k)
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int p = sub + k * subs, e = e0 + i * team_threads;
                    if (sub < at_once && p < n_parts && e < n_out)
                        early[k][i] = __ldcg(reinterpret_cast<const float4*>(part_of(p)) + e);
                }
            for (int i = me; i < n_parts * pt.rows; i += team_threads) {
                const float* q = part_of(i / pt.rows) + kRows * DP + i % pt.rows;
                wt[i] = __ldcg(q);
                sm[i] = __ldcg(q + kRows);
            }
            __syncthreads();
            // eight lanes a row: all rows of a group at once
            for (int row = me / 8; row < pt.rows; row += team_threads / 8) {
                const uint32_t eight = 0xFFu << (lane & 24);
                float m = -INFINITY, l = 0.f;
                for (int p = lane & 7; p < n_parts; p += 8) m = fmaxf(m, wt[p * pt.rows + row]);
                for (int k = 4; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(eight, m, k));
                for (int p = lane & 7; p < n_parts; p += 8) {
                    float& w = wt[p * pt.rows + row];
                    w = w == -INFINITY ? 0.f : exp2_approx(w - m);
                    l = fmaf(w, sm[p * pt.rows + row], l);
                }
                for (int k = 4; k; k >>= 1) l += __shfl_xor_sync(eight, l, k);
                if ((lane & 7) == 0) {
                    s_sum[x][row] = l;
                    s_ref[x][row] = 1.0f / l;
                    write_lse(a, pt.r, pt.head0 + row, m, l);
                }
            }
            __syncthreads();
            float4 acc[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            auto add = [&](int i, int p, int e, float4 v) {
                const float f = wt[p * pt.rows + e / (DP / 4)];
                acc[i].x = fmaf(f, v.x, acc[i].x);
                acc[i].y = fmaf(f, v.y, acc[i].y);
                acc[i].z = fmaf(f, v.z, acc[i].z);
                acc[i].w = fmaf(f, v.w, acc[i].w);
            };
            if (sub < at_once) {
#pragma unroll
                for (int k = 0; k < kFirst; ++k)
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const int p = sub + k * subs, e = e0 + i * team_threads;
                        if (p < n_parts && e < n_out) add(i, p, e, early[k][i]);
                    }
            }
            if (subs == 1) {
#pragma unroll 4
                for (int p = kFirst; p < n_parts; ++p) {
                    const float4* q = reinterpret_cast<const float4*>(part_of(p));
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const int e = e0 + i * team_threads;
                        if (e < n_out) add(i, p, e, __ldcg(q + e));
                    }
                }
            } else if (sub < at_once) {
                // eight loads in flight (the last part again behind the end, not added)
                static_assert(kEach >= 2, "two sums of a thread");
                const auto rest = [&](auto sums) {
                    constexpr int kSums = decltype(sums)::value, kBatch = 8 / kSums;
                    int at[2] = {sub + kFirst * subs, sub + at_once};   // next parts of the sums
                    const int stop = kSums == 2 && at[1] >= subs ? 0 : n_parts;
                    while (at[kSums - 1] < stop || at[0] < n_parts) {
                        float4 v[kBatch][kSums];
#pragma unroll
                        for (int k = 0; k < kBatch; ++k)
#pragma unroll
                            for (int i = 0; i < kSums; ++i)
                                v[k][i] = __ldcg(reinterpret_cast<const float4*>(
                                                     part_of(min(at[i] + k * subs, n_parts - 1))) + e0);
#pragma unroll
                        for (int k = 0; k < kBatch; ++k)
#pragma unroll
                            for (int i = 0; i < kSums; ++i)
                                if (at[i] + k * subs < (i ? stop : n_parts)) add(i, at[i] + k * subs, e0, v[k][i]);
#pragma unroll
                        for (int i = 0; i < kSums; ++i) at[i] += kBatch * subs;
                    }
                    red[sub * n_out + e0] = acc[0];
                    if (kSums == 2 && stop) red[(sub + at_once) * n_out + e0] = acc[1];
                };
                if (at_once < subs) rest(std::integral_constant<int, 2>{});
                else rest(std::integral_constant<int, 1>{});
            }
            __syncthreads();
            if (subs > 1 && sub == 0) {
                acc[0] = red[e0];
                for (int k = 1; k < subs; ++k) {
                    const float4 v = red[k * n_out + e0];
                    acc[0].x += v.x;
                    acc[0].y += v.y;
                    acc[0].z += v.z;
                    acc[0].w += v.w;
                }
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int e = e0 + i * team_threads;
                if (sub == 0 && e < n_out)
                    write_out<To>(a, pt.r, pt.head0 + e / (DP / 4), e % (DP / 4) * 4, acc[i], s_sum[x][e / (DP / 4)],
                                  s_ref[x][e / (DP / 4)], &s_open);
            }
        }

        // ---- infinities and NaN among the values: what they make of the results ----
        __syncthreads();
        if (s_open) {
            const auto settle_group = [&](int r, int hm) {
                const int q0 = hm % a.row_blocks * kRows;
                settle<To>(a, r, hm / a.row_blocks * a.group + q0, min(kRows, a.group - q0),
                           reinterpret_cast<uint32_t*>(smem));
            };
            Cursor c;   // the share's whole groups
            c.r = s_start.r;
            c.s = s_start.s;
            c.hm = static_cast<int>(divide(s_start.in_row, c.s.nt));
            for (long long u = u0 - (s_start.in_row - static_cast<long long>(c.hm) * c.s.nt); u < u0 + n_units;) {
                const long long next = u + c.s.nt;
                if (u >= u0 && next <= u0 + n_units) settle_group(c.r, c.hm);
                u = next;
                c.t = c.s.nt - 1;
                next_unit<kTile>(a, c, per_row);
            }
            for (int x = 0; x < 2; ++x)   // and those that it joined
                if (s_last[x])
                    settle<To>(a, s_partial[x].r, s_partial[x].head0, s_partial[x].rows, reinterpret_cast<uint32_t*>(smem));
        }
    }

    // rows with nothing to read
    for (int r = blockIdx.x * kWarps + warp; r < a.n_rows; r += gridDim.x * kWarps) {
        if (span_of<kTile>(a, r).nt) continue;
        To* o = static_cast<To*>(a.out) + r * a.ldo;
        for (int i = lane; i < a.n_head * a.d; i += 32) o[i] = from_f32<To>(0.f);
        if (a.lse)
            for (int i = lane; i < a.n_head; i += 32) a.lse[static_cast<int64_t>(r) * a.n_head + i] = -INFINITY;
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
    if (!words(block_table, seq_of, kv_len, lse)) return set_error(B2Q_ERR_ALIGN, "misaligned array");
    const int group = n_head / c.n_kv_head;
    auto go = [&](auto t, auto to) {
        using T = decltype(t);
        using To = decltype(to);
        return with_shape(c.d_head, group, [&](auto dp, auto rows) {
            constexpr int DP = decltype(dp)::value, kRows = decltype(rows)::value;
            constexpr int smem = smem_bytes<DP, kRows>();
            PagedArgs<T> a{static_cast<const T*>(q), ldq, static_cast<int>(n_rows), n_head, group,
                           (group + kRows - 1) / kRows, c.d_head, max_blocks, n_table_rows, window, view_of<T>(c),
                           block_table, bt_stride, seq_of, kv_len, scale * 1.44269504088896340736f, out, ldo, lse,
                           static_cast<uint32_t*>(scratch),
                           reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + kCounterBytes), ds->err};
            auto* kernel = paged_kernel<T, To, DP, kRows>;
            static std::atomic<uint64_t> allowed{0};
            const b2q_status s = allow_smem(kernel, smem, allowed, ds->device);
            if (s) return s;
            return cuda_check(launch_after(kernel, dim3(grid_of(ds->num_sms, Shape<DP>::kCtas)), dim3(Shape<DP>::kThreads), smem,
                                           static_cast<cudaStream_t>(stream), a),
                              "paged attention launch");
        });
    };
    auto with_out = [&](auto t) { return out_dtype == B2Q_TYPE_F32 ? go(t, float{}) : go(t, t); };
    return c.dtype == B2Q_TYPE_F16 ? with_out(__half{}) : with_out(__nv_bfloat16{});
}

}  // extern "C"
