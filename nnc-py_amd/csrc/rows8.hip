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
// are exactly defined whatever order the squares are summed in. Where the sum of
// squares passes the largest number (values over 2^49 at least), it is taken
// once more of values 2^80 smaller, a sum under 2^126 for rows of 2^30.
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
    bool nt;  // outputs of kNtStoreBytes or more
};

static constexpr float kSmaller = 0x1p-80f;

// r, from the sum of squares of values 2^80 smaller if SMALLER
template <bool SMALLER>
__device__ __forceinline__ float inverse_root(float squares, int width, float eps) {
    if (SMALLER) return kSmaller / sqrtf(squares / (float)width + eps * kSmaller * kSmaller);
    return 1.0f / sqrtf(squares / (float)width + eps);
}
__device__ __forceinline__ bool too_large(float squares, int width, float eps) { return !(squares / (float)width + eps < INFINITY); }

// A store of up to 16 bytes, non-temporal or not.
template <typename P>
__device__ __forceinline__ void store_pack(bool nt, P* to, const P& v) {
    if constexpr (sizeof(P) == 16) {
        const nt_u32x4 u = __builtin_bit_cast(nt_u32x4, v);
        nt ? __builtin_nontemporal_store(u, (nt_u32x4*)to) : (void)(*(nt_u32x4*)to = u);
    } else if constexpr (sizeof(P) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        nt ? __builtin_nontemporal_store(u, (uint64_t*)to) : (void)(*(uint64_t*)to = u);
    } else if constexpr (sizeof(P) == 4) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        nt ? __builtin_nontemporal_store(u, (uint32_t*)to) : (void)(*(uint32_t*)to = u);
    } else {
        *to = v;
    }
}

template <size_t BYTES>
struct HeldAs;
template <>
struct HeldAs<16> {
    typedef nt_u32x4 type;
};
template <>
struct HeldAs<4> {
    typedef uint32_t type;
};
template <>
struct HeldAs<2> {
    typedef uint16_t type;
};

// Rows that fit the registers of TPR threads (64: a wave, 256: a workgroup),
// PER packs of N elements each: one read, one write. The next row's loads go
// out before the row is worked on, and the weights stay in registers over
// all rows of a wave. Bound by HBM: about 22 vector operations per element are
// 38 us for [16384, 4096] f16.
template <typename T, int N, int TPR, int PER, int OUT, bool NORM>
__global__ void __launch_bounds__(256) row_norm_reg_k(RowArgs a) {
    typedef Pack<T, N> P;
    typedef typename HeldAs<sizeof(P)>::type Held;  // (as an array of halves it takes twice the registers)
    constexpr int ROWS = 256 / TPR;
    __shared__ float part[2][4];
    const int lane = threadIdx.x % TPR, packs = a.width / N;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    if (TPR == 64 && row >= a.rows) return;
    auto load = [&](Held (&v)[PER], const void* base, int64_t r) {
        const P* p = (const P*)((const T*)base + r * a.width);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int i = lane + TPR * q;
            v[q] = i < packs ? __builtin_bit_cast(Held, p[i]) : Held{};
        }
    };
    Held w[NORM ? PER : 1], x[PER], res[NORM ? PER : 1];
    if constexpr (NORM) load(w, a.w, 0);
    load(x, a.in, row);
    if constexpr (NORM)
        if (a.res) load(res, a.res, row);
    for (; row < a.rows; row += step) {
        // (not converted to 32 bits once for all rows: twice the registers)
        if constexpr (NORM && N > 1)
#pragma unroll
            for (int q = 0; q < PER; ++q) asm volatile("" : "+v"(w[q]));
        Held s[PER];
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            s[q] = x[q];
            if constexpr (NORM) {
                if (a.res) {
                    P v = __builtin_bit_cast(P, x[q]), u = __builtin_bit_cast(P, res[q]);
#pragma unroll
                    for (int e = 0; e < N; ++e) v.v[e] = (T)((float)v.v[e] + (float)u.v[e]);
                    s[q] = __builtin_bit_cast(Held, v);
                }
            }
        }
        if (TPR == 64 && row + step < a.rows) {
            load(x, a.in, row + step);
            if constexpr (NORM)
                if (a.res) load(res, a.res, row + step);
        }
        float sq = 0.f;
        uint32_t big = 0;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const P v = __builtin_bit_cast(P, s[q]), u = __builtin_bit_cast(P, w[NORM ? q : 0]);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float y = (float)v.v[e];
                if (NORM) sq = fmaf(y, y, sq);
                if (OUT == kRowsInt8) big = max(big, abs_bits(NORM ? y * (float)u.v[e] : y));
            }
        }
        float top = __uint_as_float(big);
        if (NORM) sq = wave_add(sq);
        if (OUT == kRowsInt8) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(__shfl_xor(top, o))));
        }
        if constexpr (TPR == 256) {
            if ((threadIdx.x & 63) == 0) part[0][threadIdx.x >> 6] = sq, part[1][threadIdx.x >> 6] = top;
            __syncthreads();
            sq = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
            top = max_nan(max_nan(part[1][0], part[1][1]), max_nan(part[1][2], part[1][3]));
            __syncthreads();
        }
        float r = NORM ? inverse_root<false>(sq, a.width, a.eps) : 1.0f;
        if (NORM && too_large(sq, a.width, a.eps)) {
            sq = 0.f;
#pragma unroll
            for (int q = 0; q < PER; ++q) {
                const P v = __builtin_bit_cast(P, s[q]);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float y = (float)v.v[e] * kSmaller;
                    sq = fmaf(y, y, sq);
                }
            }
            sq = wave_add(sq);
            if constexpr (TPR == 256) {
                if ((threadIdx.x & 63) == 0) part[0][threadIdx.x >> 6] = sq;
                __syncthreads();
                sq = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
                __syncthreads();
            }
            r = inverse_root<true>(sq, a.width, a.eps);
        }
        const float unit = unit8(top), inverse = inverse8(unit);
        if (OUT == kRowsInt8 && lane == 0) a.scale[row] = r * unit;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int i = lane + TPR * q;
            if (i >= packs) continue;
            const P v = __builtin_bit_cast(P, s[q]), u = __builtin_bit_cast(P, w[NORM ? q : 0]);
            if (NORM && a.sum) store_pack(a.nt, (P*)((T*)a.sum + row * a.width) + i, v);
            if constexpr (OUT == kRowsInt8) {
                float t[N];
#pragma unroll
                for (int e = 0; e < N; ++e) t[e] = NORM ? (float)v.v[e] * (float)u.v[e] : (float)v.v[e];
                Pack<int8_t, N> out;
                whole8_run<N>(t, unit, inverse, out.v);
                store_pack(a.nt, (Pack<int8_t, N>*)((int8_t*)a.out + row * a.width) + i, out);
            } else if constexpr (NORM) {
                P out;
#pragma unroll
                for (int e = 0; e < N; ++e) out.v[e] = (T)((float)v.v[e] * r * (float)u.v[e]);
                store_pack(a.nt, (P*)((T*)a.out + row * a.width) + i, out);
            }
        }
        if (TPR == 256 && row + step < a.rows) {
            load(x, a.in, row + step);
            if constexpr (NORM)
                if (a.res) load(res, a.res, row + step);
        }
    }
}

// Longer rows: one workgroup per row, the row read from memory (its later reads
// come from the caches) for the squares, the largest value and the output, one
// element a lane. [4096, 14336] fp32 to 8 bits 109 us, of which its bytes are 56
// at a copy's rate; [4096, 4097] f16 to floats, unaligned, 25, and 13.
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
        float r = NORM ? inverse_root<false>(sq, a.width, a.eps) : 1.0f;
        if (NORM && too_large(sq, a.width, a.eps)) {
            sq = 0.f;
            for (int i = threadIdx.x; i < a.width; i += 256) {
                float s = (float)in[i];
                if (res) s = (float)(T)(s + (float)res[i]);
                s *= kSmaller;
                sq = fmaf(s, s, sq);
            }
            sq = wave_add(sq);
            if (lane == 0) part[0][wave] = sq;
            __syncthreads();
            sq = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
            __syncthreads();
            r = inverse_root<true>(sq, a.width, a.eps);
        }
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

// N elements a thread.
template <typename T, int N>
__global__ void __launch_bounds__(256) row_float_k(const int8_t* in, const float* scale, T* out, int64_t packs, uint32_t per_row, bool nt) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += (int64_t)gridDim.x * 256) {
        const int64_t row = packs >> 32 ? i / per_row : (uint32_t)i / per_row;
        const float u = scale[row];
        const Pack<int8_t, N> q = ((const Pack<int8_t, N>*)in)[i];
        Pack<T, N> v;
#pragma unroll
        for (int e = 0; e < N; ++e) v.v[e] = (T)((float)q.v[e] * u);
        store_pack(nt, (Pack<T, N>*)out + i, v);
    }
}

template <typename T>
static void launch_float(const char* name, const int8_t* in, const float* scale, T* out, int64_t rows, int width) {
    constexpr int N = 16 / (int)sizeof(T);
    const bool nt = rows * width * (int64_t)sizeof(T) >= kNtStoreBytes;
    if (width % N == 0 && aligned16(out) && ((uintptr_t)in & (N - 1)) == 0) {
        const int64_t packs = rows * (width / N);
        launch(name, row_float_k<T, N>, dim3(grid_for(packs, 2)), dim3(256), 0, in, scale, out, packs, (uint32_t)(width / N), nt);
    } else {
        launch(name, row_float_k<T, 1>, dim3(grid_for(rows * width, 4)), dim3(256), 0, in, scale, out, rows * width, (uint32_t)width, false);
    }
}

template <typename T, int N, int TPR, int PER, bool NORM>
static void launch_rows_reg(const char* name, const RowArgs& a, bool int8) {
    // every CU its fill of waves; each then walks its rows
    const int64_t groups = ceil_div(a.rows, 256 / TPR), most = (int64_t)cu_count() * (TPR == 64 ? 8 : 16);
    const dim3 grid((unsigned)(groups < most ? groups : most));
    if (int8)
        launch(name, row_norm_reg_k<T, N, TPR, PER, kRowsInt8, NORM>, grid, dim3(256), 0, a);
    else if constexpr (NORM)
        launch(name, row_norm_reg_k<T, N, TPR, PER, kRowsFloat, true>, grid, dim3(256), 0, a);
}

// A wave to a row while rows are short and there are some for every wave of
// the GPU, else a workgroup, which has a row's elements sooner and its weights
// in fewer registers: [2048, 4096] f16 to 8 bits 11.1 us against 15.2,
// [16384, 4096] 86.0 against 93.1 (5.5 TB/s).
template <typename T, bool NORM>
static void launch_rows(const char* name, RowArgs a, bool int8) {
    constexpr int N = 16 / (int)sizeof(T);
    a.nt = a.rows * a.width * (int64_t)(int8 ? 1 : sizeof(T)) >= kNtStoreBytes;
    bool packed = a.width % N == 0 && ((uintptr_t)a.out & (int8 ? N - 1 : 15)) == 0;
    for (const void* p : {a.in, a.res, a.w, (const void*)a.sum}) packed &= aligned16(p);
    const int packs = a.width / N;
    if (packed) {
        if (a.rows >= 16 * cu_count() && packs <= 256) {
            if (packs <= 64) return launch_rows_reg<T, N, 64, 1, NORM>(name, a, int8);
            if (packs <= 128) return launch_rows_reg<T, N, 64, 2, NORM>(name, a, int8);
            if (packs <= 256) return launch_rows_reg<T, N, 64, 4, NORM>(name, a, int8);
        }
        if (packs <= 256) return launch_rows_reg<T, N, 256, 1, NORM>(name, a, int8);
        if (packs <= 512) return launch_rows_reg<T, N, 256, 2, NORM>(name, a, int8);
        if (packs <= 1024) return launch_rows_reg<T, N, 256, 4, NORM>(name, a, int8);
        if (packs <= 2048) return launch_rows_reg<T, N, 256, 8, NORM>(name, a, int8);
    } else if (a.width <= 256 * 8) {
        return launch_rows_reg<T, 1, 256, 8, NORM>(name, a, int8);
    }
    const unsigned grid = (unsigned)(a.rows < 65536 ? a.rows : 65536);
    if (int8)
        launch(name, row_norm_k<T, kRowsInt8, NORM>, dim3(grid), dim3(256), 0, a);
    else if constexpr (NORM)
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
              scale ? (float*)scale->data : nullptr, rows, (int)width, eps, false};
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
    RowArgs a{in->data, nullptr, nullptr, nullptr, out->data, (float*)scale->data, rows, (int)width, 0.f, false};
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
    if (!ready(name)) return;
    set_work(1.0 * rows * width, (double)rows * width * (activation_bytes(out) + 1.0));
    if (out->dtype == NNC_DTYPE_FLOAT16)
        launch_float(name, (const int8_t*)in->data, (const float*)scale->data, (half_t*)out->data, rows, (int)width);
    else
        launch_float(name, (const int8_t*)in->data, (const float*)scale->data, (float*)out->data, rows, (int)width);
}

}  // extern "C"
