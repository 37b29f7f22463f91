// Values across the lanes of a wave, and rows as 16-byte words, for logprobs.hip
// and rope.hip.
#pragma once

#include "quant8.h"

namespace nnc {

typedef unsigned long long u64;

// The word of lane ^ J, without a way through LDS: by DPP within 16 lanes, beyond
// by exchanging rows of 16 and halves of 32.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
    const int v = (int)x;
    if constexpr (J == 1) return (uint32_t)__builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);  // quads 1 0 3 2
    if constexpr (J == 2) return (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);  // quads 2 3 0 1
    if constexpr (J == 4)  // 7 - i in eights, then 3 - i in quads
        return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true), 0x1b, 0xf, 0xf, true);
    if constexpr (J == 8) return (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);  // turned by 8
    if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
    if constexpr (J == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
template <int J>
__device__ __forceinline__ float lane_xor(float x) { return __uint_as_float(lane_xor<J>(__float_as_uint(x))); }
template <int J>
__device__ __forceinline__ u64 lane_xor(u64 x) { return (u64)lane_xor<J>((uint32_t)(x >> 32)) << 32 | lane_xor<J>((uint32_t)x); }
template <int J>
__device__ __forceinline__ double lane_xor(double x) { return __longlong_as_double((long long)lane_xor<J>((u64)__double_as_longlong(x))); }

// The sum of a lane's value and those of the lanes before it
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lanes_before(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 lanes_before(u64 x) {
    return (u64)lanes_before<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | lanes_before<CTRL, ROWS>((uint32_t)x);
}
template <typename K>
__device__ __forceinline__ K sum_before_unsigned(K x) {
    x += lanes_before<0x111, 0xf>(x);  // 1, 2, 4, 8 lanes up in rows of 16
    x += lanes_before<0x112, 0xf>(x);
    x += lanes_before<0x114, 0xf>(x);
    x += lanes_before<0x118, 0xf>(x);
    x += lanes_before<0x142, 0xa>(x);  // a row's last to the next row, rows 1 and 3
    x += lanes_before<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
    return x;
}
__device__ __forceinline__ u64 sum_before(u64 x) { return sum_before_unsigned(x); }
__device__ __forceinline__ int sum_before(int x) { return (int)sum_before_unsigned((uint32_t)x); }

// What `op` makes of the values of 2 J lanes side by side
template <int J = 32, typename K, class Op>
__device__ __forceinline__ K over_lanes(K x, Op op) {
    x = op(x, lane_xor<J>(x));
    if constexpr (J > 1) return over_lanes<J / 2>(x, op);
    return x;
}

// 16 bytes of a row, kept as words
template <typename T>
struct Words {
    static constexpr int V = 16 / (int)sizeof(T);
    static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xfc00fc00u;  // -infinity
    __device__ __forceinline__ static float at(nt_u32x4 w, int u) {
        if constexpr (sizeof(T) == 4) {
            const uint32_t x = w[u];
            return __uint_as_float(x);
        } else {
            const uint32_t x = w[u / 2];
            return (float)__builtin_bit_cast(f16x2, x)[u % 2];
        }
    }
    // the words with the next value first
    __device__ __forceinline__ static nt_u32x4 next(nt_u32x4 w) {
        if constexpr (sizeof(T) == 4) return nt_u32x4{w[1], w[2], w[3], w[0]};
        return nt_u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
    }
    // float64 values, rounded to float32 and then to T. (The compiler would make
    // one conversion of the two, which takes twenty operations for float16.)
    __device__ __forceinline__ static float narrow(double y) {
        float f = (float)y;
        asm("" : "+v"(f));
        return f;
    }
    __device__ __forceinline__ static nt_u32x4 of(const double (&y)[V]) {
        nt_u32x4 w;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if constexpr (sizeof(T) == 4)
                w[u] = __float_as_uint((float)y[u]);
            else
                w[u] = __builtin_bit_cast(uint32_t, f16x2{(half_t)narrow(y[2 * u]), (half_t)narrow(y[2 * u + 1])});
        }
        return w;
    }
    __device__ __forceinline__ static uint32_t max_of(uint32_t x, uint32_t y) {
        if constexpr (sizeof(T) == 4)
            return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
        else
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(f16x2, x), __builtin_bit_cast(f16x2, y)));
    }
};

}  // namespace nnc
