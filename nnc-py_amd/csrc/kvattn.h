// What the kernels that attend over the paged 8-bit cache share
// (kvattention.hip, kvtree.hip, kvtree_rows.hip): whole numbers as MFMA operands, and a softmax
// whose weights carry the scales of the values' pages. kvattention.hip has the
// formulas.
#pragma once

#include "mfma_tile.h"
#include "quant8.h"

namespace nnc {

// 8 whole numbers as f16: 1024 + (q + 128) has the byte as its low bits
__device__ __forceinline__ f16x8 widen8(uint32_t lo, uint32_t hi) {
    union {
        uint32_t u[4];
        f16x8 v;
    } x;
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    x.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    x.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    x.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    x.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    const _Float16 c = (_Float16)-1152.f;
    return x.v + f16x8{c, c, c, c, c, c, c, c};
}

// p is scaled by 2^12 before it is rounded to f16: its smallest steps are then
// 2^-36 of the row's largest. The running maximum is only moved, and what was
// summed up scaled down, when it has grown by more than 2^3 (p stays below
// 2^15). It is the largest x itself, so that the p of a key that outweighs the
// others is 2^12, exact in f16: the next power of two in its place makes f16
// results of 64 sequences of up to 8192 worse by a third (2.9e-4 for 2.2e-4).
static constexpr float kSlack = 3.f;
static constexpr float kPLog = 12.f;
// A page's factor is used up to here. A p that l needs (2^-41: 2^17 such keys
// change its last bit) is 2^-101 then, still a normal number; and as e is chosen
// where m is moved or the factor is larger only, a term of l is up to 2^75, of
// which 2^28 leave it finite.
static constexpr float kMostFactor = 0x1p60f;
// m before anything was seen: x is above, and 2^(kNone - x) is 0
static constexpr float kNone = -3.402823466e38f;
// a page of zeros has the logarithm of a scale so small that none of its p
// shows beside a page of values, and no factor
static constexpr float kZeros = -200.f;
typedef float fx2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float scale_log(float scale) {
    const float log = __builtin_amdgcn_logf(scale);
    return log < kZeros ? kZeros : log;  // (NaN stays)
}
// The s against which l is taken (2^12 of p go with e), and e for the largest s.
__device__ __forceinline__ float reference(float m, float e) { return m - (e + kPLog); }
__device__ __forceinline__ float exponent(float m, float largest) { return floorf(__builtin_amdgcn_fmed3f(m - largest, -400.f, 400.f)) - kPLog; }
// What l becomes when m and e do: times o's factor and a power of two. (In one
// exponential where either may not be a normal number: the sum is rounded, by
// less than a weight's last bit.)
__device__ __forceinline__ float rescale(float m, float e, float to_m, float to_e) { return __builtin_amdgcn_exp2f((m - to_m) + (to_e - e)); }
// e before anything was seen
static constexpr float kUnseen = 400.f - kPLog;

typedef float fx16 __attribute__((ext_vector_type(16)));

// Where a 16-byte chunk of a row of RB bytes is in LDS: permuted, so that 16 lanes
// reading a chunk of 16 rows hit all 64 banks
template <int RB>
__device__ __forceinline__ int lds_chunk(int row, int chunk) {
    const int key = RB >= 256 ? row & 15 : RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
    return row * RB + (chunk ^ key) * 16;
}

}  // namespace nnc
