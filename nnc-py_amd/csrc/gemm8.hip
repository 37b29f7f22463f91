// Matrix product of 8-bit integers (nnc_hip_matmul_i8): activations a
// [M][K] with a scale for each row, weights w [N][K] with a scale for each
// row,
//   out[m][n] = (sum_k a[m][k] w[n][k]) * (a_scale[m] * w_scale[n]) + bias[n].
// The sum is exact (32-bit integers: K up to 131071); the scales, the bias
// and the output's rounding follow in 32 bits. No reference counterpart.
//
// v_mfma_i32_16x16x64_i8: lane (i = lane % 16, g = lane / 16) holds 16 k of
// row i of either operand; the k order is the same in both, so it does not
// matter which 16 of the 64 a lane group has. Result register r is row
// 4g + r, column i.
#include "quant8.h"

namespace nnc {

struct Gemm8Args {
    const int8_t* a;
    const int8_t* w;
    const float* as;
    const float* ws;
    const float* bias;
    void* out;
    int64_t m, n;
    int k;
};

// 64 x 64 outputs per workgroup, each wave 16 rows; 64 k at a time through
// LDS, loaded byte by byte: any K, any alignment.
template <typename T>
__global__ void __launch_bounds__(256) gemm8_any_k(Gemm8Args p) {
    __shared__ __align__(16) int8_t as[64][80], ws[64][80];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    ix4 acc[4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 64) {
        for (int e = threadIdx.x; e < 64 * 64; e += 256) {
            const int r = e >> 6, c = e & 63;
            const bool in = k0 + c < p.k;
            as[r][c] = in && m0 + r < p.m ? p.a[(m0 + r) * p.k + k0 + c] : 0;
            ws[r][c] = in && n0 + r < p.n ? p.w[(n0 + r) * p.k + k0 + c] : 0;
        }
        __syncthreads();
        const ix4 x = *reinterpret_cast<const ix4*>(&as[16 * wave + i][16 * g]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const ix4 y = *reinterpret_cast<const ix4*>(&ws[16 * c + i][16 * g]);
            acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, acc[c], 0, 0, 0);
        }
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int64_t n = n0 + 16 * c + i;
        if (n >= p.n) continue;
        const float sn = p.ws[n], b = p.bias ? p.bias[n] : 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t m = m0 + 16 * wave + 4 * g + r;
            if (m >= p.m) continue;
            ((T*)p.out)[m * p.n + n] = (T)((float)acc[c][r] * (p.as[m] * sn) + b);
        }
    }
}

template <typename T>
static void launch_gemm8(const char* name, const Gemm8Args& p) {
    launch(name, gemm8_any_k<T>, dim3((unsigned)ceil_div(p.n, 64), (unsigned)ceil_div(p.m, 64)), dim3(256), 0, p);
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_matmul_i8(Tensor* a, Tensor* a_scale, Tensor* w, Tensor* w_scale, Tensor* bias, Tensor* out) {
    const char* name = "nnc_hip_matmul_i8";
    if (!has_data(a) || !has_data(a_scale) || !has_data(w) || !has_data(w_scale) || !has_data(out) ||
        (bias && !has_data(bias)))
        return fail(NNC_HIP_EINVAL, name, "NULL tensor or data");
    if (a->dtype != NNC_DTYPE_INT8 || w->dtype != NNC_DTYPE_INT8) return fail(NNC_HIP_EUNSUPP, name, "int8 operands only");
    if (a_scale->dtype != NNC_DTYPE_FLOAT32 || w_scale->dtype != NNC_DTYPE_FLOAT32 ||
        (bias && bias->dtype != NNC_DTYPE_FLOAT32))
        return fail(NNC_HIP_EUNSUPP, name, "float32 scales and bias only");
    if (!is_activation(out)) return fail(NNC_HIP_EUNSUPP, name, "float32 or float16 output only");
    if (!good_shape(a) || !good_shape(out) || !good_shape(w) || w->ndim != 2)
        return fail(NNC_HIP_EINVAL, name, "w must be [N][K]");
    const int64_t k = a->shape[a->ndim - 1], n = w->shape[0];
    if (w->shape[1] != k) return fail(NNC_HIP_EINVAL, name, "rows of %lld and %lld", (long long)k, (long long)w->shape[1]);
    if (out->shape[out->ndim - 1] != n) return fail(NNC_HIP_EINVAL, name, "output rows of %lld, not %lld",
                                                    (long long)out->shape[out->ndim - 1], (long long)n);
    const int64_t m = prod(a->shape, 0, a->ndim - 1);
    if (prod(out->shape, 0, out->ndim - 1) != m || numel(a_scale) != m || numel(w_scale) != n || (bias && numel(bias) != n))
        return fail(NNC_HIP_EINVAL, name, "a_scale and out need %lld rows, w_scale and bias %lld", (long long)m, (long long)n);
    if (m == 0 || n == 0) return;
    if (k < 1 || k > 131071) return fail(NNC_HIP_EUNSUPP, name, "K = %lld (1 to 131071)", (long long)k);
    if (m > (int64_t)65535 * 64 || n > (int64_t)1 << 30) return fail(NNC_HIP_EUNSUPP, name, "too many rows");
    if (!ready(name)) return;
    Gemm8Args p{(const int8_t*)a->data, (const int8_t*)w->data, (const float*)a_scale->data, (const float*)w_scale->data,
                bias ? (const float*)bias->data : nullptr, out->data, m, n, (int)k};
    set_work(2.0 * m * n * k, (double)m * k + (double)n * k + (double)m * n * activation_bytes(out));
    if (out->dtype == NNC_DTYPE_FLOAT16)
        launch_gemm8<half_t>(name, p);
    else
        launch_gemm8<float>(name, p);
}

}  // extern "C"
