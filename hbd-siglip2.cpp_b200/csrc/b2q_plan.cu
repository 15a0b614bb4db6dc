// b2q_plan.cu — block tables, positions and cache slots of a decode step from
// the requests' lengths (b2q_kv_plan).
//
// With P the page size, request s holds have_s = ceil(ctx_s / P) pages and
// needs need_s = ceil((ctx_s + new_s) / P); its missing pages come from the
// free list at first_s = sum over r < s of (need_r - have_r), its rows start at
// row_s = sum over r < s of new_r.  Both sums are exclusive scans over the
// requests.  There is next to no data (about 16 bytes a row), so latency is
// what counts: one launch, no CTA waits for another.  Every CTA scans all
// requests for itself (n_seq is at most a few thousand: a few reads a thread,
// out of L2) and then fills its share of the rows and of the taken pages, each
// found by bisection in the scanned sums.  A row's page comes from the free
// list itself where it is one that this step enters, so no row waits for a
// table entry that another CTA writes.
// Measured on one B200, device time: 33 requests of one token 3.2 us, 509 requests of
// 260,000 rows (4.2 MB) 4.8 us (one row of a thread at a time 6.6; more than one CTA an
// SM 7.5 to 9).
#include "b2q_decode.cuh"

namespace b2q {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxSeq = 16384;
// The scanned sums stop here: beyond it no row and no page exists (both counts
// are int32), and min(a + b, cap) of values up to cap fits an int32 and is
// associative.
constexpr int kPlanCap = 1 << 30;

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, kPlanCap); }

struct PlanArgs {
    const int32_t *ctx, *add;
    const int32_t* free_pages;
    int32_t* table;
    int64_t bt_stride;
    int32_t *seq_of, *pos, *slot, *kv_len, *counts;
    uint32_t* err;
    int n_seq, shift, n_free, max_blocks, max_tokens;
};

// What request s has and brings, cut to what its table row can hold.
__device__ __forceinline__ void lengths_of(const PlanArgs& a, int s, int& ctx, int& add, bool& bad) {
    ctx = a.ctx[s];
    add = a.add[s];
    if (ctx < 0 || add < 0) bad = true;
    ctx = max(ctx, 0);
    add = max(add, 0);
    const int room = a.max_blocks << a.shift;   // fits: checked at the call
    if (static_cast<int64_t>(ctx) + add > room) bad = true;
    ctx = min(ctx, room);
}

__device__ __forceinline__ int blocks_of(const PlanArgs& a, int64_t tokens) {
    const int64_t b = (tokens + (1ll << a.shift) - 1) >> a.shift;
    return static_cast<int>(b < a.max_blocks ? b : a.max_blocks);
}

// Whether a page has slots of its own: not negative, and its slots fit an int32 (those
// of a larger one would wrap round to other pages' slots).
__device__ __forceinline__ bool is_page(const PlanArgs& a, int page) {
    return static_cast<uint32_t>(page) <= static_cast<uint32_t>(INT32_MAX >> a.shift);
}

// last s < n with base[s] <= i of each i (base ascending, base[0] = 0 <= i); searched
// side by side, as every step is one read from shared memory
template <int kN>
__device__ __forceinline__ void find_seqs(const int* base, int n, const int (&i)[kN], int (&s)[kN]) {
#pragma unroll
    for (int k = 0; k < kN; ++k) s[k] = 0;
    for (int left = n; left > 1;) {
        const int half = left >> 1;
#pragma unroll
        for (int k = 0; k < kN; ++k)
            if (base[s[k] + half] <= i[k]) s[k] += half;
        left -= half;
    }
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(PlanArgs a) {
    extern __shared__ int sums[];             // row_s [n_seq + 1], first_s [n_seq + 1], ctx_s [n_seq]
    __shared__ int warp_rows[kPlanThreads / 32], warp_pages[kPlanThreads / 32];
    let_next_start();
    wait_for_previous();
    int* rows = sums;
    int* pages = rows + a.n_seq + 1;
    int* ctxs = pages + a.n_seq + 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
    bool bad = false;
    int nr = 0, np = 0;
    for (int s = s0; s < s1; ++s) {
        int ctx, add;
        lengths_of(a, s, ctx, add, bad);
        nr = sat_add(nr, min(add, kPlanCap));
        np = sat_add(np, blocks_of(a, static_cast<int64_t>(ctx) + add) - blocks_of(a, ctx));
    }
    int ir = nr, ip = np;                     // inclusive over the threads
    for (int o = 1; o < 32; o <<= 1) {
        const int r = __shfl_up_sync(0xffffffffu, ir, o), p = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) {
            ir = sat_add(ir, r);
            ip = sat_add(ip, p);
        }
    }
    if (lane == 31) {
        warp_rows[warp] = ir;
        warp_pages[warp] = ip;
    }
    __syncthreads();
    int br = __shfl_up_sync(0xffffffffu, ir, 1), bp = __shfl_up_sync(0xffffffffu, ip, 1);
    if (lane == 0) br = bp = 0;
    for (int w = 0; w < warp; ++w) {
        br = sat_add(br, warp_rows[w]);
        bp = sat_add(bp, warp_pages[w]);
    }
    for (int s = s0; s < s1; ++s) {
        int ctx, add;
        bool again = false;
        lengths_of(a, s, ctx, add, again);
        rows[s] = br;
        pages[s] = bp;
        ctxs[s] = ctx;
        br = sat_add(br, min(add, kPlanCap));
        bp = sat_add(bp, blocks_of(a, static_cast<int64_t>(ctx) + add) - blocks_of(a, ctx));
    }
    if (s1 == a.n_seq && (s0 < s1 || (tid == 0))) {   // the thread that holds the last request
        rows[a.n_seq] = br;
        pages[a.n_seq] = bp;
    }
    __syncthreads();
    const int n_rows = rows[a.n_seq], n_pages = pages[a.n_seq];
    const int step = gridDim.x * kPlanThreads, at = blockIdx.x * kPlanThreads + tid;
    if (blockIdx.x == 0 && tid == 0) {
        a.counts[0] = n_rows;
        a.counts[1] = min(n_pages, a.n_free);
    }
    if (bad || n_rows > a.max_tokens || n_pages > a.n_free) report(a.err, kDevPlanFull);

    for (int i = at; i < n_pages; i += step) {
        const int one[1] = {i};
        int s[1];
        find_seqs(pages, a.n_seq, one, s);
        const int b = blocks_of(a, ctxs[s[0]]) + (i - pages[s[0]]);
        const int page = i < a.n_free ? a.free_pages[i] : -1;
        const bool ok = is_page(a, page);
        if (!ok) report(a.err, kDevPlanFull);   // such an entry is no page; those behind it are still taken
        a.table[s[0] * a.bt_stride + b] = ok ? page : -1;
    }
    // Four rows of a thread at a time, so that their searches and page reads overlap.
    constexpr int kEach = 4;
    for (int t0 = at; t0 < a.max_tokens; t0 += kEach * step) {
        int t[kEach], seq[kEach], pos[kEach], page[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) t[k] = t0 + min(k, (a.max_tokens - 1 - t0) / step) * step;
        find_seqs(rows, a.n_seq, t, seq);   // (0 for a row behind the last; not used)
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            page[k] = -1;
            if (t[k] >= n_rows) continue;
            const int ctx = ctxs[seq[k]];
            // a row behind the table's room has no page; its position stays an int32
            const int64_t p = static_cast<int64_t>(ctx) + (t[k] - rows[seq[k]]);
            pos[k] = p < INT32_MAX ? static_cast<int>(p) : INT32_MAX - 1;
            const int b = pos[k] >> a.shift, have = blocks_of(a, ctx);
            if (b < have) {
                page[k] = a.table[seq[k] * a.bt_stride + b];
            } else if (b < a.max_blocks) {
                const int i = pages[seq[k]] + (b - have);
                if (i < a.n_free) page[k] = a.free_pages[i];
            }
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (k && t[k] == t[k - 1]) break;
            const bool in = t[k] < n_rows;
            a.seq_of[t[k]] = in ? seq[k] : -1;
            a.pos[t[k]] = in ? pos[k] : -1;
            const bool ok = is_page(a, page[k]);
            a.slot[t[k]] = ok ? (page[k] << a.shift) + (pos[k] & ((1 << a.shift) - 1)) : -1;
            a.kv_len[t[k]] = in ? pos[k] + 1 : 0;
            if (!ok && page[k] >= 0) report(a.err, kDevPlanFull);
        }
    }
}

}  // namespace
}  // namespace b2q

using namespace b2q;

extern "C" b2q_status b2q_kv_plan(const int32_t* ctx_len, const int32_t* new_len, int32_t n_seq, int32_t page_size,
                                  const int32_t* free_pages, int32_t n_free, int32_t* block_table, int64_t bt_stride,
                                  int32_t max_blocks, int32_t max_tokens, int32_t* seq_of, int32_t* pos, int32_t* slot,
                                  int32_t* kv_len, int32_t* counts, void* stream) {
    B2Q_REQUIRE_STATE();
    if (n_seq < 0 || n_seq > kPlanMaxSeq || n_free < 0 || max_tokens < 0 || max_tokens > kPlanCap)
        return set_error(B2Q_ERR_SHAPE, "bad n_seq / n_free / max_tokens");
    if (page_size <= 0 || page_size > 1024 || (page_size & (page_size - 1)))
        return set_error(B2Q_ERR_SHAPE, "page_size must be a power of two up to 1024");
    if (max_blocks < 0 || bt_stride < max_blocks) return set_error(B2Q_ERR_SHAPE, "bad block table width / stride");
    if (static_cast<int64_t>(max_blocks) * page_size > INT32_MAX)
        return set_error(B2Q_ERR_SHAPE, "block table rows hold more tokens than an int32");
    if (!counts || (n_seq > 0 && (!ctx_len || !new_len)) || (n_seq > 0 && max_blocks > 0 && !block_table) ||
        (n_free > 0 && !free_pages) || (max_tokens > 0 && (!seq_of || !pos || !slot || !kv_len)))
        return set_error(B2Q_ERR_INVALID, "null pointer");
    if (!words(ctx_len, new_len, free_pages, block_table, seq_of, pos, slot, kv_len, counts))
        return set_error(B2Q_ERR_ALIGN, "misaligned array");
    PlanArgs a{ctx_len, new_len, free_pages, block_table, bt_stride, seq_of, pos, slot, kv_len, counts, ds->err,
               n_seq, log2_of(page_size), n_free, max_blocks, max_tokens};
    const size_t smem = sizeof(int) * (3 * static_cast<size_t>(n_seq) + 2);
    b2q_status st;
    if (smem > 40960 &&
        (st = cuda_check(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              static_cast<int>(sizeof(int) * (3 * kPlanMaxSeq + 2))),
                         "plan shared memory")))
        return st;
    const int64_t work = max_tokens > n_seq ? max_tokens : n_seq;
    int64_t grid = (work + 2 * kPlanThreads - 1) / (2 * kPlanThreads);
    grid = grid < 1 ? 1 : (grid > ds->num_sms ? ds->num_sms : grid);
    return cuda_check(launch_after(kv_plan_kernel, dim3(static_cast<unsigned>(grid)), dim3(kPlanThreads), smem,
                                   static_cast<cudaStream_t>(stream), a),
                      "plan launch");
}
