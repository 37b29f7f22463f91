// What the calls that write the paged 8-bit cache share (kvcache.hip, rope.hip).
#pragma once

#include <tuple>

#include "quant8.h"

namespace nnc {

struct KvArgs {
    Ragged g;
    int8_t *k, *v;
    float *k_scale, *v_scale;
    void *k_rows, *v_rows;
    int64_t k_ld, v_ld;
    int k_col, v_col, kv_heads, dim;
};

// false with an error recorded
bool kv_args(const char* name, Tensor* k, Tensor* v, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale,
             Tensor* v_scale, Tensor* table, Tensor* starts, Tensor* lengths, int k_col, int v_col, KvArgs* a);
// nnc_hip_kv_write's kernels for arguments that are in order, rows not 0
void launch_write(const char* name, bool f16, const KvArgs& a);

// ---------------------------------------------------------------------------
// A group of TPG threads (a wave, or a workgroup) takes a page's K or V of one
// head in quads: four consecutive positions by V dims, V of the rows' type in
// 16 bytes. A quad is four 16-byte accesses of the rows; of K four runs of V
// bytes, of V (one row of `page` bytes per dim) V words of four positions,
// which go through LDS to whole 16-byte accesses of the cache.
// ---------------------------------------------------------------------------
template <typename T, int TPG>
struct Quads {
    static constexpr int THREADS = TPG < 256 ? 256 : TPG, GROUPS = THREADS / TPG;  // of a workgroup
    static constexpr int V = 16 / (int)sizeof(T);
    typedef Pack<T, V> Row;
    typedef Pack<int8_t, V> Held;
    int page, dim, chunks, count, thread;  // chunks: of V dims
    __device__ __forceinline__ Quads(const KvArgs& a) : page(a.g.page), dim(a.dim), chunks(a.dim / V), count(a.g.page / 4 * chunks), thread(threadIdx.x % TPG) {}
    // LDS bytes between two dims: a word past a multiple of 16, off the banks
    __device__ __forceinline__ int stride() const { return page + 4; }
    __device__ __forceinline__ static void sync() {
        if (TPG == 64) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
    }
};

// One page's K or V (which: 0, 1) of one head: scale, whole numbers.
template <typename T, int TPG, int QPER>
__device__ __forceinline__ void write_quads(const KvArgs& a, const Quads<T, TPG>& z, const PageShare& p, int which, int head, char* lds, float* part) {
    typedef Quads<T, TPG> Q;
    const int64_t at = (int64_t)p.page_no * a.kv_heads + head, ld = which ? a.v_ld : a.k_ld;
    const T* rows = (const T*)(which ? a.v_rows : a.k_rows) + (which ? a.v_col : a.k_col) + head * z.dim;
    int8_t* held = (which ? a.v : a.k) + at * z.page * z.dim;
    float* scale = (which ? a.v_scale : a.k_scale) + at;
    const float before = *scale;
    const int lo = p.fresh - p.begin, hi = p.stop - p.begin;
    nt_u32x4 x[QPER][4];
    uint32_t big = 0;
#pragma unroll
    for (int q = 0; q < QPER; ++q) {
        const int e = z.thread + TPG * q, t4 = e / z.chunks * 4, d = e % z.chunks * Q::V;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = e < z.count && t4 + u >= lo && t4 + u < hi;
            x[q][u] = in ? *(const nt_u32x4*)(rows + (int64_t)p.span.row(p.begin + t4 + u) * ld + d) : nt_u32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int q = 0; q < QPER; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const typename Q::Row v = __builtin_bit_cast(typename Q::Row, x[q][u]);
#pragma unroll
            for (int i = 0; i < Q::V; ++i) big = max(big, abs_bits((float)v.v[i]));
        }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o));
    float top = __uint_as_float(big);
    if constexpr (TPG > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();  // everybody has read the scale, too
        top = part[0];
#pragma unroll
        for (int i = 1; i < TPG / 64; ++i) top = max_nan(top, part[i]);
    }
    float unit = unit8(top);
    if (lo > 0) unit = max_nan(before, unit);
    if (z.thread == 0) *scale = unit;
    if (lo > 0 && !(unit == before)) {
        for (int i = z.thread; i < lo * z.dim; i += TPG) {
            int8_t* w = held + (which ? i % z.dim * z.page + i / z.dim : i);
            *w = unit > 0.f ? (int8_t)rint((double)*w * (double)before / (double)unit) : 0;
        }
    }
    const float inverse = inverse8(unit);
    char* mine = lds + threadIdx.x / TPG * z.dim * z.stride();
#pragma unroll
    for (int q = 0; q < QPER; ++q) {
        const int e = z.thread + TPG * q, t4 = e / z.chunks * 4, d = e % z.chunks * Q::V;
        if (e >= z.count) continue;
        typename Q::Held w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const typename Q::Row v = __builtin_bit_cast(typename Q::Row, x[q][u]);
            float f[Q::V];
#pragma unroll
            for (int i = 0; i < Q::V; ++i) f[i] = (float)v.v[i];
            whole8_run<Q::V>(f, unit, inverse, w[u].v);
            if (!which && t4 + u >= lo && t4 + u < hi) *(typename Q::Held*)(held + (t4 + u) * z.dim + d) = w[u];
        }
        if (which) {
#pragma unroll
            for (int i = 0; i < Q::V; ++i) {
                const uint32_t word = (uint8_t)w[0].v[i] | (uint32_t)(uint8_t)w[1].v[i] << 8 | (uint32_t)(uint8_t)w[2].v[i] << 16 | (uint32_t)(uint8_t)w[3].v[i] << 24;
                *(uint32_t*)(mine + (d + i) * z.stride() + t4) = word;
            }
        }
    }
    Q::sync();
    if (!which) return;
    if (lo == 0 && hi == z.page) {
        for (int o = z.thread * 16; o < z.dim * z.page; o += TPG * 16) {
            const uint32_t* w = (const uint32_t*)(mine + o / z.page * z.stride() + o % z.page);
            *(nt_u32x4*)(held + o) = nt_u32x4{w[0], w[1], w[2], w[3]};
        }
    } else {
        // part of a page: the positions of the call and no others
        const int from = lo & ~3, words = (hi - from + 3) / 4;
        for (int i = z.thread; i < words * z.dim; i += TPG) {
            const int d = i / words, t = from + i % words * 4;
            const char* w = mine + d * z.stride() + t;
            if (t >= lo && t + 4 <= hi) {
                *(uint32_t*)(held + d * z.page + t) = *(const uint32_t*)w;
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (t + u >= lo && t + u < hi) held[d * z.page + t + u] = (int8_t)w[u];
            }
        }
    }
}

// Whether the rows start on 16 bytes.
template <typename T>
static bool quads(const KvArgs& a) {
    for (auto [p, col, ld] : {std::tuple(a.k_rows, a.k_col, a.k_ld), std::tuple(a.v_rows, a.v_col, a.v_ld)})
        if (!aligned16(p) || col * sizeof(T) % 16 != 0 || ld * (int64_t)sizeof(T) % 16 != 0) return false;
    return true;
}

}  // namespace nnc
