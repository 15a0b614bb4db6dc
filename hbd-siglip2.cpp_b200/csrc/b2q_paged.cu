// b2q_paged.cu — attention of single tokens over a paged key-value cache
// (b2q_attention_paged).
#include "b2q_decode.cuh"

#include <cmath>

namespace b2q {
namespace {

constexpr int kPagedWarps = 4;

template <class T>
struct PagedArgs {
    const T* q;
    int64_t ldq;
    int n_rows, n_head, group, d, max_blocks, n_table_rows, window;
    CacheView<T> c;
    const int32_t* table;
    int64_t bt_stride;
    const int32_t *seq_of, *kv_len;
    float scale;
    void* out;
    int64_t ldo;
    float* lse;
    uint32_t* err;
};

// One CTA per (row, head); keys over the warps, elements over the lanes.
template <class T, class To>
__global__ void __launch_bounds__(kPagedWarps * 32) paged_kernel(PagedArgs<T> a) {
    __shared__ float sm[kPagedWarps], sl[kPagedWarps], so[kPagedWarps][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.y, h = blockIdx.x, hk = h / a.group;
    int len = a.kv_len[r];
    const int seq = a.seq_of ? a.seq_of[r] : r;
    if (len > 0 && seq != -1 && (seq < 0 || seq >= a.n_table_rows)) {
        report(a.err, kDevBadPage);
        len = 0;
    }
    if (seq == -1) len = 0;
    const int64_t room = static_cast<int64_t>(a.max_blocks) * (a.c.page_mask + 1);
    if (len < 0 || len > room) {
        report(a.err, kDevBadPage);
        len = len < 0 ? 0 : static_cast<int>(room);
    }
    const int first = a.window > 0 && len > a.window ? len - a.window : 0;
    float q[8], o[8];
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < a.d ? to_f32(a.q[r * a.ldq + static_cast<int64_t>(h) * a.d + d]) * a.scale : 0.f;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = first + warp; j < len; j += kPagedWarps) {
        const int page = a.table[seq * a.bt_stride + (j >> a.c.page_shift)];
        if (page < 0 || page >= a.c.n_pages) {
            if (lane == 0) report(a.err, kDevBadPage);
            continue;
        }
        const int64_t at = page * a.c.page_stride + hk * a.c.head_stride + (j & a.c.page_mask) * a.c.token_stride;
        float s = 0.f;
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d < a.d) s = fmaf(q[i], to_f32(a.c.k[at + d]), s);
        }
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m, s), f = m == mn ? 1.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
        l = l * f + p;
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d < a.d) o[i] = o[i] * f + p * to_f32(a.c.v[at + d]);
        }
        m = mn;
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
    for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mx = -INFINITY, lt = 0.f;
    for (int w = 0; w < kPagedWarps; ++w) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < kPagedWarps; ++w) lt += sm[w] == -INFINITY ? 0.f : sl[w] * expf(sm[w] - mx);
    for (int d = threadIdx.x; d < a.d; d += kPagedWarps * 32) {
        float v = 0.f;
        for (int w = 0; w < kPagedWarps; ++w) v += sm[w] == -INFINITY ? 0.f : so[w][d] * expf(sm[w] - mx);
        static_cast<To*>(a.out)[r * a.ldo + static_cast<int64_t>(h) * a.d + d] = from_f32<To>(lt > 0.f ? v / lt : v);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[static_cast<int64_t>(r) * a.n_head + h] = lt > 0.f ? mx + logf(lt) : -INFINITY;
}

}  // namespace
}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_attention_paged_scratch_bytes(int32_t n_head, int32_t n_kv_head, int32_t d_head) {
    if (n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head || d_head <= 0) return 0;
    return 256;
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
    if (n_rows < 0 || n_rows > 65535 || n_head <= 0 || n_head > 65535 || n_head % c.n_kv_head)
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto go = [&](auto t) {
        using T = decltype(t);
        PagedArgs<T> a{static_cast<const T*>(q), ldq, static_cast<int>(n_rows), n_head, n_head / c.n_kv_head,
                       c.d_head, max_blocks, n_table_rows, window, view_of<T>(c), block_table, bt_stride, seq_of,
                       kv_len, scale, out, ldo, lse, ds->err};
        const dim3 grid(n_head, static_cast<unsigned>(n_rows));
        if (out_dtype == B2Q_TYPE_F32) paged_kernel<T, float><<<grid, kPagedWarps * 32, 0, s>>>(a);
        else paged_kernel<T, T><<<grid, kPagedWarps * 32, 0, s>>>(a);
        count_launch();
        return cuda_check(cudaGetLastError(), "paged attention launch");
    };
    return c.dtype == B2Q_TYPE_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

}  // extern "C"
