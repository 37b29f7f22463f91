// Shared by the 8-bit serving operators (rows8.hip, gemm8.hip, kvcache.hip,
// kvattention.hip): activation types, the rounding to 8 bits, and how a
// workgroup finds the sequence that its share of a ragged batch belongs to.
#pragma once

#include <math.h>

#include "common.h"
#include "ragged.h"

namespace nnc {

typedef _Float16 half_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float fx4 __attribute__((ext_vector_type(4)));
typedef int ix4 __attribute__((ext_vector_type(4)));
typedef int ix2 __attribute__((ext_vector_type(2)));

// A row or page whose largest absolute value is below this holds zeros with
// scale 0 (its 127th, and the reciprocal of that, stay normal numbers).
static constexpr float kTiny8 = 0x1p-100f;

// The value of one 8-bit step for numbers up to `largest`: a 127th, rounded
// once. Not finite (a NaN or an infinity among the numbers): NaN, so that
// everything the step scales reads as NaN.
__device__ __forceinline__ float unit8(float largest) {
    if (!(largest < INFINITY)) return NAN;
    return largest < kTiny8 ? 0.f : largest / 127.0f;
}

// The larger of two absolute values; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

// 1 / unit for whole8, 0 where the unit is 0 or NaN (which makes every whole
// number 0)
__device__ __forceinline__ float inverse8(float unit) { return unit > 0.f ? 1.0f / unit : 0.f; }

// The whole numbers nearest to x / unit, ties to even, as if the quotient were
// exact: x * inverse is off by a few of its last bits, so the rounded product
// can be the neighbour; the remainder x - q * unit, exact in one fused
// operation, says so, and only then (one value in 2^16) is there more to do.
// |x| <= 127 units.
template <int N>
__device__ __forceinline__ void whole8_run(const float (&x)[N], float unit, float inverse, int8_t (&out)[N]) {
    float q[N];
    const float half = 0.5f * unit;
    bool near = false;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        q[e] = rintf(x[e] * inverse);
        near |= fabsf(fmaf(-q[e], unit, x[e])) >= half;
    }
    if (near) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float rest = fmaf(-q[e], unit, x[e]);
            if (fabsf(rest) > half || (fabsf(rest) == half && ((int)q[e] & 1))) q[e] += copysignf(1.0f, rest);
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = inverse == 0.f ? (int8_t)0 : (int8_t)(int)q[e];
}
__device__ __forceinline__ int whole8(float x, float unit, float inverse) {
    const float v[1] = {x};
    int8_t q[1];
    whole8_run<1>(v, unit, inverse, q);
    return q[0];
}

// N elements of a row, loaded and stored as one.
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};

// |x|'s bits: ordered like the values, NaN above infinity
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Maximum (NaN if any is) and sum over a wave's 64 lanes, in every lane.
__device__ __forceinline__ float wave_max_nan(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max_nan(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// Finds the sequence that share number `share` falls to, count(b) being how
// many shares sequence b has: -1 if there are fewer, else b, with `share` its
// number within b. Every wave of a workgroup does this for itself: 64
// sequences at a time, their counts summed along the lanes.
template <class Count>
__device__ __forceinline__ int find_share(int& share, int batch, Count count) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < batch; base += 64) {
        const int c = base + lane < batch ? count(base + lane) : 0;
        int upto = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(upto, o);
            if (lane >= o) upto += below;
        }
        const int all = __shfl(upto, 63);
        if (share < all) {
            const int at = __ffsll((unsigned long long)__ballot(upto > share)) - 1;
            share -= __shfl(upto - c, at);
            return base + at;
        }
        share -= all;
    }
    return -1;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline bool is_activation(const Tensor* t) { return t->dtype == NNC_DTYPE_FLOAT32 || t->dtype == NNC_DTYPE_FLOAT16; }
inline int activation_bytes(const Tensor* t) { return t->dtype == NNC_DTYPE_FLOAT16 ? 2 : 4; }
inline bool good_shape(const Tensor* t) {
    if (t->ndim < 1 || t->ndim > 8) return false;
    for (int d = 0; d < t->ndim; ++d)
        if (t->shape[d] < 0) return false;
    return true;
}

// The tensors that describe a paged cache and a ragged batch, checked.
struct CacheArgs {
    int64_t pages = 0;
    int kv_heads = 0, page = 0, dim = 0;
    Ragged ragged{};
    int8_t *k = nullptr, *v = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;
};
// false with an error recorded; `rows`: rows of the activations. In kvcache.hip.
bool cache_args(const char* name, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                Tensor* starts, Tensor* lengths, int64_t rows, CacheArgs* out);
// A row-major activation matrix [rows][ld] of which `width` columns from
// `col` are used; rows and ld through the pointers.
bool rows_arg(const char* name, const char* what, Tensor* t, int col, int64_t width, int64_t* rows, int64_t* ld);

}  // namespace nnc
