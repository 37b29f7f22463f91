// The paged 8-bit cache of keys and values: rows written to it
// (nnc_hip_kv_write) and read back (nnc_hip_kv_read). No reference
// counterpart.
//
// A page holds `page` consecutive positions of one sequence. Per page and
// head there are K as [page][dim], V as [dim][page] - the attention's second
// product takes consecutive positions of one dim - and one scale each:
// value = whole number * scale.
//
// Writing a page: with u_new the 127th of the new rows' largest value, the
// page's scale becomes u = max(u_old, u_new) if it keeps positions from
// before the call, else u_new (whatever was in a page that starts over does
// not count). If the scale grows, the kept whole numbers become the nearest to
// q u_old / u; that is at most half a step more each time it does. Positions
// behind the sequence's length are left as they were.
//
// One wave or workgroup per touched page and head does all of this, so nothing
// is shared between workgroups and no atomics are needed.
#include <tuple>

#include "quant8.h"

namespace nnc {

bool rows_arg(const char* name, const char* what, Tensor* t, int col, int64_t width, int64_t* rows, int64_t* ld) {
    if (!has_data(t)) return fail(NNC_HIP_EINVAL, name, "NULL tensor or data"), false;
    if (!is_activation(t)) return fail(NNC_HIP_EUNSUPP, name, "%s: float32 or float16 only", what), false;
    if (!good_shape(t)) return fail(NNC_HIP_EINVAL, name, "%s: bad shape", what), false;
    *ld = t->shape[t->ndim - 1];
    *rows = prod(t->shape, 0, t->ndim - 1);
    if (col < 0 || col + width > *ld)
        return fail(NNC_HIP_EINVAL, name, "%s: columns [%d, %lld) outside rows of %lld", what, col,
                    (long long)(col + width), (long long)*ld), false;
    if (*rows > INT32_MAX / 64 || *ld > INT32_MAX) return fail(NNC_HIP_EUNSUPP, name, "%s: too large", what), false;
    return true;
}

bool cache_args(const char* name, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                Tensor* starts, Tensor* lengths, int64_t rows, CacheArgs* out) {
    for (Tensor* t : {k_cache, v_cache, k_scale, v_scale, table, starts, lengths})
        if (!has_data(t)) return fail(NNC_HIP_EINVAL, name, "NULL tensor or data"), false;
    for (Tensor* t : {k_cache, v_cache, k_scale, v_scale, table, starts, lengths})
        if (!good_shape(t)) return fail(NNC_HIP_EINVAL, name, "bad shape"), false;
    if (k_cache->dtype != NNC_DTYPE_INT8 || v_cache->dtype != NNC_DTYPE_INT8 || k_scale->dtype != NNC_DTYPE_FLOAT32 ||
        v_scale->dtype != NNC_DTYPE_FLOAT32 || table->dtype != NNC_DTYPE_INT32 || starts->dtype != NNC_DTYPE_INT32 ||
        lengths->dtype != NNC_DTYPE_INT32)
        return fail(NNC_HIP_EUNSUPP, name, "an int8 cache, float32 scales and int32 table, starts and lengths only"), false;
    if (k_cache->ndim != 4 || v_cache->ndim != 4 || table->ndim != 2)
        return fail(NNC_HIP_EINVAL, name, "the cache must have four extents, the table two"), false;
    const int64_t *ks = k_cache->shape, *vs = v_cache->shape;
    const int64_t page = ks[2], dim = ks[3];
    if (vs[0] != ks[0] || vs[1] != ks[1] || vs[2] != dim || vs[3] != page)
        return fail(NNC_HIP_EINVAL, name, "K must be [pages][heads][page][dim] and V [pages][heads][dim][page]"), false;
    // (a page's K and V of a head are rows of a grid of at most 65535)
    if (ks[0] < 1 || ks[1] < 1 || ks[0] > INT32_MAX || ks[1] > 32767)
        return fail(NNC_HIP_EINVAL, name, "bad page or head count"), false;
    if (page < 16 || page > 256 || page % 16 != 0)
        return fail(NNC_HIP_EUNSUPP, name, "pages of %lld positions (a multiple of 16 up to 256)", (long long)page), false;
    if (dim != 32 && dim != 64 && dim != 128 && dim != 256)
        return fail(NNC_HIP_EUNSUPP, name, "head dim %lld (32, 64, 128 or 256)", (long long)dim), false;
    if (numel(k_scale) != ks[0] * ks[1] || numel(v_scale) != ks[0] * ks[1])
        return fail(NNC_HIP_EINVAL, name, "scales must be [pages][heads]"), false;
    const int64_t batch = table->shape[0], width = table->shape[1];
    if (numel(starts) != batch + 1 || numel(lengths) != batch)
        return fail(NNC_HIP_EINVAL, name, "starts must have one more element than the table rows, lengths as many"), false;
    if (batch > (1 << 20) || width * page > INT32_MAX / 2)
        return fail(NNC_HIP_EUNSUPP, name, "table of %lld x %lld", (long long)batch, (long long)width), false;
    if (!aligned16(k_cache->data) || !aligned16(v_cache->data))
        return fail(NNC_HIP_EUNSUPP, name, "the cache must be 16-byte aligned"), false;
    out->pages = ks[0];
    out->kv_heads = (int)ks[1];
    out->page = (int)page;
    out->dim = (int)dim;
    out->k = (int8_t*)k_cache->data;
    out->v = (int8_t*)v_cache->data;
    out->k_scale = (float*)k_scale->data;
    out->v_scale = (float*)v_scale->data;
    out->ragged = Ragged{(const int*)starts->data, (const int*)lengths->data, (const int*)table->data, (int)batch,
                         (int)width, (int)rows, (int)page, ks[0]};
    return true;
}

struct KvArgs {
    Ragged g;
    int8_t *k, *v;
    float *k_scale, *v_scale;
    void *k_rows, *v_rows;
    int64_t k_ld, v_ld;
    int k_col, v_col, kv_heads, dim;
};

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

template <typename T, int TPG, int QPER>
__global__ void __launch_bounds__((Quads<T, TPG>::THREADS)) kv_write_quads_k(KvArgs a) {
    typedef Quads<T, TPG> Q;
    extern __shared__ __align__(16) char lds[];
    __shared__ float part[Q::THREADS / 64];
    const Q z(a);
    const int pair = blockIdx.y * Q::GROUPS + threadIdx.x / TPG, which = pair & 1, head = pair >> 1;
    int share = blockIdx.x;
    const int b = find_share(share, a.g.batch, [&](int i) { return touched_pages(a.g, i); });
    if (b < 0 || head >= a.kv_heads) return;  // (a workgroup of one group has one head)
    const PageShare p(a.g, b, share);
    if (p.page_no < 0) return;
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

template <typename T, int TPG>
__global__ void __launch_bounds__((Quads<T, TPG>::THREADS)) kv_read_quads_k(KvArgs a) {
    typedef Quads<T, TPG> Q;
    extern __shared__ __align__(16) char lds[];
    const Q z(a);
    const int pair = blockIdx.y * Q::GROUPS + threadIdx.x / TPG, which = pair & 1, head = pair >> 1;
    int share = blockIdx.x;
    const int b = find_share(share, a.g.batch, [&](int i) { return touched_pages(a.g, i); });
    if (b < 0 || head >= a.kv_heads) return;
    const PageShare p(a.g, b, share);
    if (p.page_no < 0) return;
    const int64_t at = (int64_t)p.page_no * a.kv_heads + head, ld = which ? a.v_ld : a.k_ld;
    T* rows = (T*)(which ? a.v_rows : a.k_rows) + (which ? a.v_col : a.k_col) + head * z.dim;
    const int8_t* held = (which ? a.v : a.k) + at * z.page * z.dim;
    const float unit = (which ? a.v_scale : a.k_scale)[at];
    const int lo = p.fresh - p.begin, hi = p.stop - p.begin;
    char* mine = lds + threadIdx.x / TPG * z.dim * z.stride();
    if (which)
        for (int o = z.thread * 16; o < z.dim * z.page; o += TPG * 16) {
            const nt_u32x4 v = *(const nt_u32x4*)(held + o);
            uint32_t* w = (uint32_t*)(mine + o / z.page * z.stride() + o % z.page);
            w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
        }
    Q::sync();
    for (int e = z.thread; e < z.count; e += TPG) {
        const int t4 = e / z.chunks * 4, d = e % z.chunks * Q::V;
        if (t4 + 3 < lo || t4 >= hi) continue;
        uint32_t word[Q::V];
        if (which)
#pragma unroll
            for (int i = 0; i < Q::V; ++i) word[i] = *(const uint32_t*)(mine + (d + i) * z.stride() + t4);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (t4 + u < lo || t4 + u >= hi) continue;
            typename Q::Held w;
            if (which) {
#pragma unroll
                for (int i = 0; i < Q::V; ++i) w.v[i] = (int8_t)(word[i] >> 8 * u);
            } else {
                w = *(const typename Q::Held*)(held + (t4 + u) * z.dim + d);
            }
            typename Q::Row v;
#pragma unroll
            for (int i = 0; i < Q::V; ++i) v.v[i] = (T)((float)w.v[i] * unit);
            *(typename Q::Row*)(rows + (int64_t)p.span.row(p.begin + t4 + u) * ld + d) = v;
        }
    }
}

// Rows that start on no 16 bytes: one workgroup per page and head, element by
// element.
template <typename T>
__global__ void __launch_bounds__(256) kv_write_k(KvArgs a) {
    const int head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float part[4];
    int share = blockIdx.x;
    const int b = find_share(share, a.g.batch, [&](int i) { return touched_pages(a.g, i); });
    if (b < 0) return;
    const PageShare p(a.g, b, share);
    if (p.page_no < 0) return;
    const int page = a.g.page, n = (p.stop - p.fresh) * a.dim;
    const int64_t at = (int64_t)p.page_no * a.kv_heads + head;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const T* rows = (const T*)(which ? a.v_rows : a.k_rows) + (which ? a.v_col : a.k_col) + head * a.dim;
        const int64_t ld = which ? a.v_ld : a.k_ld;
        int8_t* held = (which ? a.v : a.k) + at * page * a.dim;
        float* scale = (which ? a.v_scale : a.k_scale) + at;
        float top = 0.f;
        for (int i = threadIdx.x; i < n; i += 256)
            top = max_nan(top, fabsf((float)rows[(int64_t)p.span.row(p.fresh + i / a.dim) * ld + i % a.dim]));
        top = wave_max_nan(top);
        if (lane == 0) part[wave] = top;
        __syncthreads();
        float unit = unit8(max_nan(max_nan(part[0], part[1]), max_nan(part[2], part[3])));
        const float before = *scale;
        __syncthreads();  // everybody has read the scale
        const int kept = p.fresh - p.begin;
        if (kept > 0) unit = max_nan(before, unit);
        if (threadIdx.x == 0) *scale = unit;
        if (kept > 0 && !(unit == before)) {
            for (int i = threadIdx.x; i < kept * a.dim; i += 256) {
                const int t = i / a.dim, d = i % a.dim;
                int8_t* q = held + (which ? d * page + t : i);
                *q = unit > 0.f ? (int8_t)rint((double)*q * (double)before / (double)unit) : 0;
            }
        }
        const float inverse = inverse8(unit);
        for (int i = threadIdx.x; i < n; i += 256) {
            const int t = i / a.dim, d = i % a.dim, at_t = p.fresh - p.begin + t;
            const float x = (float)rows[(int64_t)p.span.row(p.fresh + t) * ld + d];
            held[which ? d * page + at_t : at_t * a.dim + d] = (int8_t)whole8(x, unit, inverse);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_k(KvArgs a) {
    const int head = blockIdx.y;
    int share = blockIdx.x;
    const int b = find_share(share, a.g.batch, [&](int i) { return touched_pages(a.g, i); });
    if (b < 0) return;
    const PageShare p(a.g, b, share);
    if (p.page_no < 0) return;
    const int page = a.g.page, n = (p.stop - p.fresh) * a.dim;
    const int64_t at = (int64_t)p.page_no * a.kv_heads + head;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        T* rows = (T*)(which ? a.v_rows : a.k_rows) + (which ? a.v_col : a.k_col) + head * a.dim;
        const int64_t ld = which ? a.v_ld : a.k_ld;
        const int8_t* held = (which ? a.v : a.k) + at * page * a.dim;
        const float unit = (which ? a.v_scale : a.k_scale)[at];
        for (int i = threadIdx.x; i < n; i += 256) {
            const int t = i / a.dim, d = i % a.dim, at_t = p.fresh - p.begin + t;
            rows[(int64_t)p.span.row(p.fresh + t) * ld + d] =
                (T)((float)held[which ? d * page + at_t : at_t * a.dim + d] * unit);
        }
    }
}

template <typename T>
static bool quads(const KvArgs& a) {
    for (auto [p, col, ld] : {std::tuple(a.k_rows, a.k_col, a.k_ld), std::tuple(a.v_rows, a.v_col, a.v_ld)})
        if (!aligned16(p) || col * sizeof(T) % 16 != 0 || ld * (int64_t)sizeof(T) % 16 != 0) return false;
    return true;
}

template <typename T, int TPG, void (*kernel)(KvArgs)>
static void launch_quads(const char* name, const KvArgs& a) {
    typedef Quads<T, TPG> Q;
    const size_t lds = (size_t)Q::GROUPS * a.dim * (a.g.page + 4);
    if constexpr (TPG == 1024) {  // the largest pages: 66560 bytes, allowed once for each kernel
        static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 256 * 260) == hipSuccess;
        if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    }
    launch(name, kernel, dim3((unsigned)touched_bound(a.g.rows, a.g.batch, a.g.page), (unsigned)ceil_div(2 * a.kv_heads, Q::GROUPS)),
           dim3(Q::THREADS), lds, a);
}

// A wave to a page's K or V of a head while that is one quad a lane (16
// positions by 128 in f16), else a workgroup: 8 prompts of 1024 in fp32, 16
// heads of 64 in pages of 64, 15.5 us with a wave and four quads a lane, 11.7
// with a workgroup and one (read 12.2 and 10.6). The bytes alone are 7.2 us each
// way at a copy's rate, the rest is the chain of lengths, table, scale and rows
// that each page waits for, about 5 us, as for one new token in each of 32
// sequences (5.5 us). Bytes one by one took 32 us each. Pages of more than 1024
// quads (256 positions by 128 in fp32) get workgroups of 1024, whose lanes hold
// no more than others'.
template <typename T>
static void launch_write(const char* name, const KvArgs& a) {
    const int n = a.g.page * a.dim * (int)sizeof(T) / 64;
    if (!quads<T>(a))
        return launch(name, kv_write_k<T>, dim3((unsigned)touched_bound(a.g.rows, a.g.batch, a.g.page), (unsigned)a.kv_heads), dim3(256), 0, a);
    if (n <= 64) return launch_quads<T, 64, kv_write_quads_k<T, 64, 1>>(name, a);
    if (n <= 256) return launch_quads<T, 256, kv_write_quads_k<T, 256, 1>>(name, a);
    if (n <= 512) return launch_quads<T, 256, kv_write_quads_k<T, 256, 2>>(name, a);
    if (n <= 1024) return launch_quads<T, 256, kv_write_quads_k<T, 256, 4>>(name, a);
    if constexpr (sizeof(T) == 4) {
        if (n > 2048) return launch_quads<T, 1024, kv_write_quads_k<T, 1024, 4>>(name, a);
    }
    launch_quads<T, 1024, kv_write_quads_k<T, 1024, 2>>(name, a);
}

template <typename T>
static void launch_read(const char* name, const KvArgs& a) {
    const int n = a.g.page * a.dim * (int)sizeof(T) / 64;
    if (!quads<T>(a))
        return launch(name, kv_read_k<T>, dim3((unsigned)touched_bound(a.g.rows, a.g.batch, a.g.page), (unsigned)a.kv_heads), dim3(256), 0, a);
    if (n <= 64) return launch_quads<T, 64, kv_read_quads_k<T, 64>>(name, a);
    if (n <= 1024) return launch_quads<T, 256, kv_read_quads_k<T, 256>>(name, a);
    launch_quads<T, 1024, kv_read_quads_k<T, 1024>>(name, a);
}

static bool kv_args(const char* name, Tensor* k, Tensor* v, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale,
                    Tensor* v_scale, Tensor* table, Tensor* starts, Tensor* lengths, int k_col, int v_col, KvArgs* a) {
    CacheArgs c;
    int64_t rows = 0, v_rows = 0;
    if (!cache_args(name, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, 0, &c)) return false;
    const int64_t width = (int64_t)c.kv_heads * c.dim;
    if (!rows_arg(name, "k", k, k_col, width, &rows, &a->k_ld) || !rows_arg(name, "v", v, v_col, width, &v_rows, &a->v_ld))
        return false;
    if (rows != v_rows || k->dtype != v->dtype) return fail(NNC_HIP_EINVAL, name, "k and v differ in rows or type"), false;
    a->g = c.ragged;
    a->g.rows = (int)rows;
    a->k = c.k, a->v = c.v, a->k_scale = c.k_scale, a->v_scale = c.v_scale;
    a->k_rows = k->data, a->v_rows = v->data;
    a->k_col = k_col, a->v_col = v_col, a->kv_heads = c.kv_heads, a->dim = c.dim;
    return true;
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_kv_write(Tensor* k, Tensor* v, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale,
                      Tensor* table, Tensor* starts, Tensor* lengths, int k_col, int v_col) {
    const char* name = "nnc_hip_kv_write";
    KvArgs a;
    if (!kv_args(name, k, v, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, k_col, v_col, &a)) return;
    if (a.g.rows == 0 || a.g.batch == 0 || a.g.width == 0) return;
    if (!ready(name)) return;
    const double n = 2.0 * a.g.rows * a.kv_heads * a.dim;
    set_work(6.0 * n, n * (activation_bytes(k) + 1));
    if (k->dtype == NNC_DTYPE_FLOAT16)
        launch_write<half_t>(name, a);
    else
        launch_write<float>(name, a);
}

void nnc_hip_kv_read(Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table, Tensor* starts,
                     Tensor* lengths, Tensor* k, Tensor* v, int k_col, int v_col) {
    const char* name = "nnc_hip_kv_read";
    KvArgs a;
    if (!kv_args(name, k, v, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, k_col, v_col, &a)) return;
    if (a.g.rows == 0 || a.g.batch == 0 || a.g.width == 0) return;
    if (!ready(name)) return;
    const double n = 2.0 * a.g.rows * a.kv_heads * a.dim;
    set_work(n, n * (activation_bytes(k) + 1));
    if (k->dtype == NNC_DTYPE_FLOAT16)
        launch_read<half_t>(name, a);
    else
        launch_read<float>(name, a);
}

}  // extern "C"
