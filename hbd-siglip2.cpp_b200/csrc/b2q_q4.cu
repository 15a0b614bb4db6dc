// b2q_q4.cu — products of few activation rows with ggml Q4_0 / Q4_1 weights
// (b2q_weight_q4_*, b2q_mul_vec_q4).
#include "b2q_decode.cuh"

#include <new>

struct b2q_weight_q4 {
    int64_t N = 0, K = 0;
    int type = 0, device = -1;
    uint8_t* blocks = nullptr;   // [N][K / 32] blocks, rows back to back
};

namespace b2q {
namespace {

constexpr int kQ4Warps = 8;

template <class Tx, class Ty>
struct Q4Args {
    const uint8_t* w;
    int64_t N, K;
    const Tx* x;
    int64_t x_cols, ldx;
    Ty* y;
    int64_t ldy;
    const float *bias, *residual;
};

// One warp per (output, activation row); blocks of 32 weights over the lanes.
template <bool kMin, class Tx, class Ty>
__global__ void __launch_bounds__(kQ4Warps * 32) mul_vec_q4_kernel(Q4Args<Tx, Ty> a) {
    const int lane = threadIdx.x & 31;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kQ4Warps + (threadIdx.x >> 5);
    const int64_t m = blockIdx.y;
    if (n >= a.N) return;
    constexpr int kBlock = kMin ? 20 : 18;
    const int64_t Kb = a.K / 32;
    const Tx* x = a.x + m * a.ldx;
    float acc = 0.f;
    for (int64_t kb = lane; kb < Kb; kb += 32) {
        const uint8_t* b = a.w + (n * Kb + kb) * kBlock;
        const float d = __half2float(__ushort_as_half(static_cast<uint16_t>(b[0] | (b[1] << 8))));
        float dot = 0.f, sum = 0.f;
        for (int j = 0; j < 32; ++j) {
            const int64_t k = kb * 32 + j;
            const float xv = k < a.x_cols ? to_f32(x[k]) : 0.f;
            const int q = (b[(kMin ? 4 : 2) + (j & 15)] >> (j < 16 ? 0 : 4)) & 15;
            dot = fmaf(static_cast<float>(kMin ? q : q - 8), xv, dot);
            sum += xv;
        }
        acc = fmaf(d, dot, acc);
        if (kMin) acc = fmaf(__half2float(__ushort_as_half(static_cast<uint16_t>(b[2] | (b[3] << 8)))), sum, acc);
    }
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane) return;
    if (a.bias) acc += a.bias[n];
    if (a.residual) acc += a.residual[m * a.ldy + n];
    a.y[m * a.ldy + n] = from_f32<Ty>(acc);
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
    if (N <= 0 || N > (1 << 24) || K <= 0 || K > (1 << 20) || K % 32)
        return set_error(B2Q_ERR_SHAPE, "a 4-bit weight needs N in [1, 2^24] and K a multiple of 32 up to 2^20");
    const int64_t bytes = K / 32 * (ggml_type == B2Q_TYPE_Q4_0 ? 18 : 20);
    if (row_bytes < bytes) return set_error(B2Q_ERR_SHAPE, "row_bytes smaller than the row's blocks");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    b2q_weight_q4* w = new (std::nothrow) b2q_weight_q4();
    if (!w) return set_error(B2Q_ERR_NOMEM, "out of host memory");
    w->N = N;
    w->K = K;
    w->type = ggml_type;
    w->device = ds->device;
    b2q_status st = B2Q_OK;
    if (cudaMalloc(reinterpret_cast<void**>(&w->blocks), static_cast<size_t>(N * bytes)) != cudaSuccess) {
        cudaGetLastError();
        delete w;
        return set_error(B2Q_ERR_NOMEM, "cudaMalloc of a 4-bit weight failed");
    }
    st = cuda_check(cudaMemcpy2DAsync(w->blocks, static_cast<size_t>(bytes), blocks, static_cast<size_t>(row_bytes),
                                      static_cast<size_t>(bytes), static_cast<size_t>(N),
                                      src_is_host ? cudaMemcpyHostToDevice : cudaMemcpyDeviceToDevice, s),
                    "4-bit weight copy");
    if (!st && src_is_host) st = cuda_check(cudaStreamSynchronize(s), "4-bit weight upload");
    if (st) {
        cudaFree(w->blocks);
        delete w;
        return st;
    }
    *out = w;
    return B2Q_OK;
}

b2q_status b2q_weight_q4_release(b2q_weight_q4* w) {
    if (!w) return B2Q_OK;
    cudaFree(w->blocks);
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
    auto go = [&](auto tx, auto ty) {
        using Tx = decltype(tx);
        using Ty = decltype(ty);
        Q4Args<Tx, Ty> a{w->blocks, w->N, w->K, static_cast<const Tx*>(x), x_cols, ldx, static_cast<Ty*>(y), ldy,
                         bias, residual};
        const dim3 grid(static_cast<unsigned>((w->N + kQ4Warps - 1) / kQ4Warps), static_cast<unsigned>(M));
        if (w->type == B2Q_TYPE_Q4_1) mul_vec_q4_kernel<true, Tx, Ty><<<grid, kQ4Warps * 32, 0, s>>>(a);
        else mul_vec_q4_kernel<false, Tx, Ty><<<grid, kQ4Warps * 32, 0, s>>>(a);
        count_launch();
        return cuda_check(cudaGetLastError(), "4-bit product launch");
    };
    auto with_x = [&](auto tx) { return y_dtype == B2Q_TYPE_F32 ? go(tx, float{}) : go(tx, tx); };
    return x_dtype == B2Q_TYPE_F32   ? with_x(float{})
           : x_dtype == B2Q_TYPE_F16 ? with_x(__half{})
                                     : with_x(__nv_bfloat16{});
}

}  // extern "C"
