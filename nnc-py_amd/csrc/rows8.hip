// Row operators of the 8-bit serving path: RMS norm with the residual's
// addition (nnc_hip_rms_norm), rows to 8 bits with a scale each
// (nnc_hip_quantize_rows) and back (nnc_hip_dequantize_rows). No reference
// counterpart.
//
//   s = in (+ res), rounded to the activations' type
//   y = s * r * w, r = 1 / sqrt(mean(s^2) + eps)           (float output)
//   t = s * w in 32 bits, u = max|t| / 127, q = t / u to the nearest even
//   whole number, scale = r * u                            (8-bit output)
//
// r cancels out of y / scale, so q does not depend on it: the whole numbers
// are exactly defined whatever order the squares are summed in.
#include "quant8.h"

namespace nnc {

enum { kRowsFloat = 0, kRowsInt8 = 1 };

struct RowArgs {
    const void* in;
    const void* res;
    const void* w;
    void* sum;
    void* out;
    float* scale;
    int64_t rows;
    int width;
    float eps;
};

// One workgroup per row, the row read from memory (its later reads come from
// the caches) for the squares, the largest value and the output.
template <typename T, int OUT, bool NORM>
__global__ void __launch_bounds__(256) row_norm_k(RowArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float part[2][4];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* in = (const T*)a.in + row * a.width;
        const T* res = a.res ? (const T*)a.res + row * a.width : nullptr;
        const T* w = (const T*)a.w;
        T* sum = a.sum ? (T*)a.sum + row * a.width : nullptr;
        float sq = 0.f, top = 0.f;
        for (int i = threadIdx.x; i < a.width; i += 256) {
            float s = (float)in[i];
            if (NORM && res) s = (float)(T)(s + (float)res[i]);
            if (NORM) sq = fmaf(s, s, sq);
            if (OUT == kRowsInt8) top = max_nan(top, fabsf(NORM ? s * (float)w[i] : s));
        }
        sq = wave_add(sq);
        top = wave_max_nan(top);
        if (lane == 0) part[0][wave] = sq, part[1][wave] = top;
        __syncthreads();
        sq = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
        top = max_nan(max_nan(part[1][0], part[1][1]), max_nan(part[1][2], part[1][3]));
        __syncthreads();
        const float r = NORM ? 1.0f / sqrtf(sq / (float)a.width + a.eps) : 1.0f;
        const float unit = unit8(top), inverse = inverse8(unit);
        if (OUT == kRowsInt8 && threadIdx.x == 0) a.scale[row] = r * unit;
        for (int i = threadIdx.x; i < a.width; i += 256) {
            float s = (float)in[i];
            if (NORM && res) s = (float)(T)(s + (float)res[i]);
            const float t = NORM ? s * (float)w[i] : s;
            if (NORM && sum) sum[i] = (T)s;
            if (OUT == kRowsInt8)
                ((int8_t*)a.out)[row * a.width + i] = (int8_t)whole8(t, unit, inverse);
            else
                ((T*)a.out)[row * a.width + i] = (T)(s * r * (float)w[i]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) row_float_k(const int8_t* in, const float* scale, T* out, int64_t rows, int width) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float u = scale[row];
        for (int i = threadIdx.x; i < width; i += 256) out[row * width + i] = (T)((float)in[row * width + i] * u);
    }
}

template <typename T, bool NORM>
static void launch_rows(const char* name, const RowArgs& a, bool int8) {
    const unsigned grid = (unsigned)(a.rows < 65536 ? a.rows : 65536);
    if (int8)
        launch(name, row_norm_k<T, kRowsInt8, NORM>, dim3(grid), dim3(256), 0, a);
    else if (NORM)
        launch(name, row_norm_k<T, kRowsFloat, true>, dim3(grid), dim3(256), 0, a);
}

static bool shapes_equal(const Tensor* a, const Tensor* b) {
    return good_shape(a) && good_shape(b) && numel(a) == numel(b) && a->shape[a->ndim - 1] == b->shape[b->ndim - 1];
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_rms_norm(Tensor* in, Tensor* res, Tensor* weight, Tensor* sum, Tensor* out, Tensor* scale, float eps) {
    const char* name = "nnc_hip_rms_norm";
    if (!has_data(in) || !has_data(weight) || !has_data(out)) return fail(NNC_HIP_EINVAL, name, "NULL tensor or data");
    if ((res && !has_data(res)) || (sum && !has_data(sum)) || (scale && !has_data(scale)))
        return fail(NNC_HIP_EINVAL, name, "NULL data");
    if (!is_activation(in)) return fail(NNC_HIP_EUNSUPP, name, "float32 or float16 input only");
    if (weight->dtype != in->dtype || (res && res->dtype != in->dtype) || (sum && sum->dtype != in->dtype))
        return fail(NNC_HIP_EUNSUPP, name, "weight, residual and sum must have the input's type");
    const bool int8 = out->dtype == NNC_DTYPE_INT8;
    if (!int8 && out->dtype != in->dtype) return fail(NNC_HIP_EUNSUPP, name, "output must be int8 or of the input's type");
    if (!shapes_equal(in, out) || (res && !shapes_equal(in, res)) || (sum && !shapes_equal(in, sum)))
        return fail(NNC_HIP_EINVAL, name, "input, residual, sum and output must have the same rows");
    if (sum && !res) return fail(NNC_HIP_EINVAL, name, "a sum without a residual");
    const int64_t width = in->shape[in->ndim - 1];
    if (numel(weight) != width) return fail(NNC_HIP_EINVAL, name, "weight is not one row");
    if (int8 != (scale != nullptr)) return fail(NNC_HIP_EINVAL, name, "an int8 output and its scales go together");
    if (!(eps > 0.f)) return fail(NNC_HIP_EINVAL, name, "eps must be positive");
    if (numel(in) == 0) return;
    const int64_t rows = numel(in) / width;
    if (width > (1 << 30)) return fail(NNC_HIP_EUNSUPP, name, "rows of %lld elements", (long long)width);
    if (scale && (scale->dtype != NNC_DTYPE_FLOAT32 || numel(scale) != rows))
        return fail(NNC_HIP_EINVAL, name, "scale must be float32, one for each row");
    if (!ready(name)) return;
    RowArgs a{in->data, res ? res->data : nullptr, weight->data, sum ? sum->data : nullptr, out->data,
              scale ? (float*)scale->data : nullptr, rows, (int)width, eps};
    const double e = activation_bytes(in);
    set_work(8.0 * rows * width, (double)rows * width * (e * (1 + !!res + !!sum) + (int8 ? 1.0 : e)));
    if (in->dtype == NNC_DTYPE_FLOAT16)
        launch_rows<half_t, true>(name, a, int8);
    else
        launch_rows<float, true>(name, a, int8);
}

void nnc_hip_quantize_rows(Tensor* in, Tensor* out, Tensor* scale) {
    const char* name = "nnc_hip_quantize_rows";
    if (!has_data(in) || !has_data(out) || !has_data(scale)) return fail(NNC_HIP_EINVAL, name, "NULL tensor or data");
    if (!is_activation(in) || out->dtype != NNC_DTYPE_INT8 || scale->dtype != NNC_DTYPE_FLOAT32)
        return fail(NNC_HIP_EUNSUPP, name, "float32 or float16 to int8 with float32 scales only");
    if (!shapes_equal(in, out)) return fail(NNC_HIP_EINVAL, name, "input and output must have the same rows");
    if (numel(in) == 0) return;
    const int64_t width = in->shape[in->ndim - 1], rows = numel(in) / width;
    if (width > (1 << 30)) return fail(NNC_HIP_EUNSUPP, name, "rows of %lld elements", (long long)width);
    if (numel(scale) != rows) return fail(NNC_HIP_EINVAL, name, "scale must be one for each row");
    if (!ready(name)) return;
    RowArgs a{in->data, nullptr, nullptr, nullptr, out->data, (float*)scale->data, rows, (int)width, 0.f};
    set_work(4.0 * rows * width, (double)rows * width * (activation_bytes(in) + 1.0));
    if (in->dtype == NNC_DTYPE_FLOAT16)
        launch_rows<half_t, false>(name, a, true);
    else
        launch_rows<float, false>(name, a, true);
}

void nnc_hip_dequantize_rows(Tensor* in, Tensor* scale, Tensor* out) {
    const char* name = "nnc_hip_dequantize_rows";
    if (!has_data(in) || !has_data(out) || !has_data(scale)) return fail(NNC_HIP_EINVAL, name, "NULL tensor or data");
    if (!is_activation(out) || in->dtype != NNC_DTYPE_INT8 || scale->dtype != NNC_DTYPE_FLOAT32)
        return fail(NNC_HIP_EUNSUPP, name, "int8 with float32 scales to float32 or float16 only");
    if (!shapes_equal(in, out)) return fail(NNC_HIP_EINVAL, name, "input and output must have the same rows");
    if (numel(in) == 0) return;
    const int64_t width = in->shape[in->ndim - 1], rows = numel(in) / width;
    if (width > (1 << 30)) return fail(NNC_HIP_EUNSUPP, name, "rows of %lld elements", (long long)width);
    if (numel(scale) != rows) return fail(NNC_HIP_EINVAL, name, "scale must be one for each row");
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
    if (!ready(name)) return;
    set_work(1.0 * rows * width, (double)rows * width * (activation_bytes(out) + 1.0));
    if (out->dtype == NNC_DTYPE_FLOAT16)
        launch(name, row_float_k<half_t>, dim3(grid), dim3(256), 0, (const int8_t*)in->data, (const float*)scale->data,
               (half_t*)out->data, rows, (int)width);
    else
        launch(name, row_float_k<float>, dim3(grid), dim3(256), 0, (const int8_t*)in->data, (const float*)scale->data,
               (float*)out->data, rows, (int)width);
}

}  // extern "C"
