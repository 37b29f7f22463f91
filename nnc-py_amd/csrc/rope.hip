// Rotary positions: norms of query and key heads and their rotation by position
// (nnc_hip_rope), and the same on the way into the paged 8-bit cache
// (nnc_hip_rope_kv_write). No reference counterpart.
//
//   y = x w / sqrt(mean(x^2) + eps)           over a head's dim values, if there are weights
//   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)   for the rot / 2 pairs of its first rot dims
//
// with the pair's cosine c and sine s from the row of the angle table that the
// position names. All of it in float64 and rounded to float32 and the
// activations' type at the end: keys are then cut to whole numbers, and a
// result that depended on the order of a sum would be another whole number now
// and then. A float64 operation takes no longer than a float32 one here.
#include "kvcache.h"
#include "lanes.h"

#include "heads.h"

namespace nnc {

struct RopeArgs {
    const void* in;
    void* out;
    const void* weight;   // [dim], or [heads][dim]; null: no norm
    const float* angles;  // [places][rot]; null: no rotation
    const int* positions;  // [rows]; null: places in the sequences of g
    Ragged g;             // batch 0: every row is taken
    int64_t in_ld, out_ld;
    int64_t rows, places;
    int col, out_col, heads, dim, rot;
    bool interleaved, weight_each;
    double eps, inverse_dim;
};

// The sequence that a row belongs to, -1 if it is none's: the first whose rows
// end behind it. All lanes of a wave ask for the same row; 64 sequences are
// compared at a time. What starts holds only decides which of 0 .. batch - 1.
__device__ __forceinline__ int owner_of(const Ragged& g, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = g.batch;  // the answer is one of lo .. hi
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t past = __ballot(at < hi && g.starts[min(at, g.batch - 1) + 1] > row);
        const int probes = (hi - lo + step - 1) / step;
        const int f = past ? __ffsll((unsigned long long)past) - 1 : probes;
        if (f < probes) hi = lo + f * step;
        if (f > 0) lo += (f - 1) * step + 1;
    }
    if (lo >= g.batch) return -1;
    const Span s = span_of(g, lo);
    return row >= s.end - s.rows && row < s.end ? lo : -1;
}

// The row of the angle table for a row of the activations; -1 if the row is to
// be left alone.
__device__ __forceinline__ int64_t rope_place(const RopeArgs& a, int64_t row) {
    int64_t at = 0;
    if (a.g.batch > 0) {
        const int b = owner_of(a.g, (int)row);
        if (b < 0) return -1;
        const Span s = span_of(a.g, b);
        at = row - s.end + s.length;
    }
    if (a.positions) at = a.positions[row];
    return at < 0 ? 0 : at < a.places ? at : a.places - 1;
}

__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// 1 / sqrt(m) by the hardware's approximation (2^-26 and better) and two of
// Newton's steps
__device__ __forceinline__ double inverse_root(double m) {
    double y = __builtin_amdgcn_rsq(m);
#pragma unroll
    for (int i = 0; i < 2; ++i) y *= fma(-0.5 * m * y, y, 1.5);
    return m == INFINITY ? 0.0 : y;
}

// Any sizes: a wave to a head of a row, a pair or an unpaired dim a lane, single
// values read three times (from the cache). [4096, 20 heads of 80] f16, 20 dims
// turned, with weights, 36 us, where its bytes take 5.
template <typename T>
__global__ void __launch_bounds__(256) rope_k(RopeArgs a) {
    const int lane = threadIdx.x & 63, half = a.rot / 2;
    const int64_t items = a.rows * a.heads, step = (int64_t)gridDim.x * 4;
    for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += step) {
        const int64_t row = item / a.heads;
        const int head = (int)(item - row * a.heads);
        const int64_t place = rope_place(a, row);
        if (place < 0) continue;
        const T* x = (const T*)a.in + row * a.in_ld + a.col + (int64_t)head * a.dim;
        T* y = (T*)a.out + row * a.out_ld + a.out_col + (int64_t)head * a.dim;
        const T* w = (const T*)a.weight + (a.weight_each ? (int64_t)head * a.dim : 0);
        double r = 1.0;
        if (a.weight) {
            double sum = 0.0;
            for (int d = lane; d < a.dim; d += 64) sum += (double)(float)x[d] * (double)(float)x[d];
            r = inverse_root(wave_add(sum) * a.inverse_dim + a.eps);
        }
        auto normed = [&](int d) { return a.weight ? (double)(float)x[d] * r * (double)(float)w[d] : (double)(float)x[d]; };
        for (int u = lane; u < a.dim - half; u += 64) {
            if (u >= half) {
                y[u + half] = (T)Words<T>::narrow(normed(u + half));
                continue;
            }
            const int one = a.interleaved ? 2 * u : u, other = a.interleaved ? 2 * u + 1 : u + half;
            const double c = a.angles[place * a.rot + u], s = a.angles[place * a.rot + half + u];
            const double p = normed(one), q = normed(other);
            y[one] = (T)Words<T>::narrow(p * c - q * s);
            y[other] = (T)Words<T>::narrow(q * c + p * s);
        }
    }
}

// A unit's cosines and sines: its V pairs are the same rows' V in both layouts.
template <int V>
__device__ __forceinline__ void angles_of(const RopeArgs& a, int64_t place, int unit, float (&cs)[V], float (&sn)[V]) {
    const float* t = a.angles + place * a.rot + V * unit;
#pragma unroll
    for (int u = 0; u < V; u += 4) {
        *(float4*)(cs + u) = *(const float4*)(t + u);
        *(float4*)(sn + u) = *(const float4*)(t + a.rot / 2 + u);
    }
}
// The pairs of a unit's two packs: neighbours, or each other's values.
template <bool INTER, int V>
__device__ __forceinline__ void turn(double (&f)[V], double (&g)[V], const float (&cs)[V], const float (&sn)[V]) {
    auto pair = [](double& p, double& q, double c, double s) {
        const double t = p;
        p = t * c - q * s, q = q * c + t * s;
    };
    if constexpr (INTER) {
#pragma unroll
        for (int u = 0; u < V / 2; ++u) pair(f[2 * u], f[2 * u + 1], cs[u], sn[u]), pair(g[2 * u], g[2 * u + 1], cs[V / 2 + u], sn[V / 2 + u]);
    } else {
#pragma unroll
        for (int u = 0; u < V; ++u) pair(f[u], g[u], cs[u], sn[u]);
    }
}
// The sum over the 2^bits lanes of a head
__device__ __forceinline__ double over_head(double sum, int bits) {
    if (bits > 0) sum += lane_xor<1>(sum);
    if (bits > 1) sum += lane_xor<2>(sum);
    if (bits > 2) sum += lane_xor<4>(sum);
    if (bits > 3) sum += lane_xor<8>(sum);
    if (bits > 4) sum += lane_xor<16>(sum);
    if (bits > 5) sum += lane_xor<32>(sum);
    return sum;
}

// Heads of whole packs of 16 bytes: a lane takes two, whose values are each
// other's pairs - dims i .. and i + rot / 2 .., or 2 V neighbours - or two packs
// that stay; 2^bits lanes side by side are a head, and a wave goes through `per`
// heads of a row for each of them with the row's angles in registers, the next
// head's values on their way. Bound by the bytes: [16384, 32 + 8 heads of 128] f16
// 67 us for its 336 MB, a copy's 5.0 TB/s; a decoding step's [16, 40 x 128] is a
// launch, 3.1 us. The pairing is the kernel's, not a register's: the
// selection of partners takes a fourth of the instructions otherwise (72 us).
template <typename T, bool NORM, bool INTER>
__device__ __forceinline__ void rope_heads(const RopeArgs& a, RopeWaves shape, uint32_t item) {
    typedef Words<T> W;
    constexpr int V = W::V;
    const int bits = shape.bits;
    const int lane = threadIdx.x & 63, unit = lane & ((1 << bits) - 1), groups = shape.groups(), half = a.rot / 2;
    const uint32_t row = item / (uint32_t)shape.chunks, chunk = item - row * (uint32_t)shape.chunks;
    if (row >= a.rows) return;
    const bool turned = 2 * V * unit < a.rot, mine = 2 * V * unit < a.dim;
    const int one = turned && !INTER ? V * unit : 2 * V * unit;
    const int other = turned && !INTER ? one + half : one + V;
    const T* x = (const T*)a.in + row * a.in_ld + a.col;
    T* y = (T*)a.out + row * a.out_ld + a.out_col;
    int head = shape.begin(chunk) + (lane >> bits);
    const int end = shape.end(chunk, a.heads);
    nt_u32x4 p{}, q{}, wp{}, wq{};
    auto load = [&](int h) {
        if (mine && h < end) {
            p = *(const nt_u32x4*)(x + (int64_t)h * a.dim + one), q = *(const nt_u32x4*)(x + (int64_t)h * a.dim + other);
            if (NORM && a.weight_each) {
                const T* w = (const T*)a.weight + (int64_t)h * a.dim;
                wp = *(const nt_u32x4*)(w + one), wq = *(const nt_u32x4*)(w + other);
            }
        }
    };
    const bool all_rows = a.g.batch == 0;  // else a row may be no sequence's, and those are not read
    if (all_rows) load(head);
    if (NORM && !a.weight_each && mine) wp = *(const nt_u32x4*)((const T*)a.weight + one), wq = *(const nt_u32x4*)((const T*)a.weight + other);
    const int64_t place = rope_place(a, row);
    if (place < 0) return;
    if (!all_rows) load(head);
    float cs[V], sn[V];
    if (turned) angles_of<V>(a, place, unit, cs, sn);
    for (int first = shape.begin(chunk); first < end; first += groups, head += groups) {
        const nt_u32x4 xp = p, xq = q, vp = wp, vq = wq;
        const bool live = mine && head < end;
        const int h = head;
        load(head + groups);
        double f[V], g[V];
#pragma unroll
        for (int u = 0; u < V; ++u) f[u] = W::at(xp, u), g[u] = W::at(xq, u);
        if (NORM) {
            double sum = 0.0;
#pragma unroll
            for (int u = 0; u < V; ++u) sum = fma(f[u], f[u], sum), sum = fma(g[u], g[u], sum);
            sum = over_head(live ? sum : 0.0, bits);
            const double r = inverse_root(sum * a.inverse_dim + a.eps);
#pragma unroll
            for (int u = 0; u < V; ++u) f[u] *= r * (double)W::at(vp, u), g[u] *= r * (double)W::at(vq, u);
        }
        if (turned) turn<INTER>(f, g, cs, sn);
        if (live) {
            *(nt_u32x4*)(y + (int64_t)h * a.dim + one) = W::of(f);
            *(nt_u32x4*)(y + (int64_t)h * a.dim + other) = W::of(g);
        }
    }
}

template <typename T, bool NORM, bool INTER>
__global__ void __launch_bounds__(256) rope_packs_k(RopeArgs a, RopeWaves shape) {
    rope_heads<T, NORM, INTER>(a, shape, blockIdx.x * 4 + (threadIdx.x >> 6));
}

template <typename T>
static bool in_packs(const RopeArgs& a) {
    constexpr int V = 16 / (int)sizeof(T);
    return a.dim % (2 * V) == 0 && a.dim <= 128 * V && a.rot % (2 * V) == 0 && aligned16(a.in) && aligned16(a.out) && aligned16(a.angles) &&
           aligned16(a.weight) && a.in_ld % V == 0 && a.out_ld % V == 0 && a.col % V == 0 && a.out_col % V == 0;
}

template <typename T>
static void launch_rope_type(const char* name, const RopeArgs& a) {
    if (in_packs<T>(a)) {
        constexpr int V = 16 / (int)sizeof(T);
        const RopeWaves shape = rope_waves(a.rows, a.heads, a.dim, V, cu_count());
        const int64_t blocks = ceil_div(a.rows * shape.chunks, 4);
        if (blocks * 256 <= UINT32_MAX) {
            const dim3 grid((unsigned)blocks);
            auto kernel = a.weight ? (a.interleaved ? rope_packs_k<T, true, true> : rope_packs_k<T, true, false>)
                                   : (a.interleaved ? rope_packs_k<T, false, true> : rope_packs_k<T, false, false>);
            return launch(name, kernel, grid, dim3(256), 0, a, shape);
        }
    }
    const int64_t blocks = ceil_div(a.rows * a.heads, 4), most = (int64_t)cu_count() * 32;
    launch(name, rope_k<T>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, a);
}

static void launch_rope(const char* name, bool f16, const RopeArgs& a) {
    if (f16)
        launch_rope_type<half_t>(name, a);
    else
        launch_rope_type<float>(name, a);
}

// ---------------------------------------------------------------------------
// Into the cache: a group of TPG threads takes a page's V of a head in quads
// (kvcache.h), or its K in units of two packs, 2 QPER of them a thread, which
// are turned in registers, rounded to the rows' type, and then scaled and cut as
// nnc_hip_kv_write does. The workgroups behind those of the pages turn the queries,
// a wave for a row's heads.
//
// One launch in place of three, and the rotated keys do not go through memory: one
// token of 32 sequences, 32 heads over 8 of 128, written and read back, 18 -> 10
// us; 8 prompts of 2048 90 us for the write, 403 MB: the queries alone, 268 MB, take
// 53, keys and values 40, whose 12 float64 operations a value keep the vector units
// as busy as the memory.
// ---------------------------------------------------------------------------
struct RopeKvArgs {
    KvArgs w;
    RopeArgs q, k;
    RopeWaves shape;     // of the queries
    uint32_t shares, kv_blocks;  // pages that can be touched; workgroups of pages
};

template <typename T, int TPG, int QPER, bool INTER>
__device__ __forceinline__ void rope_page(const KvArgs& w, const RopeArgs& a, const Quads<T, TPG>& z, const PageShare& p, int head, float* part) {
    typedef Words<T> W;
    typedef Quads<T, TPG> Q;
    constexpr int V = W::V, PER = 2 * QPER;
    int bits = 0;
    while ((2 * V << bits) < z.dim) ++bits;
    const int unit = z.thread & ((1 << bits) - 1), half = a.rot / 2;
    const bool turned = 2 * V * unit < a.rot;
    const int one = turned && !INTER ? V * unit : 2 * V * unit;
    const int other = turned && !INTER ? one + half : one + V;
    const int64_t at = (int64_t)p.page_no * w.kv_heads + head;
    const T* rows = (const T*)w.k_rows + w.k_col + head * z.dim;
    int8_t* held = w.k + at * z.page * z.dim;
    float* scale = w.k_scale + at;
    const float before = *scale;
    const int lo = p.fresh - p.begin, hi = p.stop - p.begin;
    nt_u32x4 x[PER][2];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int t = (z.thread + TPG * i) >> bits;
        const bool in = t >= lo && t < hi;
        const T* row = rows + (int64_t)p.span.row(in ? p.begin + t : p.fresh) * w.k_ld;
        x[i][0] = in ? *(const nt_u32x4*)(row + one) : nt_u32x4{0, 0, 0, 0};
        x[i][1] = in ? *(const nt_u32x4*)(row + other) : nt_u32x4{0, 0, 0, 0};
    }
    nt_u32x4 wp{}, wq{};
    if (a.weight) {
        const T* weight = (const T*)a.weight + (a.weight_each ? head * z.dim : 0);
        wp = *(const nt_u32x4*)(weight + one), wq = *(const nt_u32x4*)(weight + other);
    }
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int t = (z.thread + TPG * i) >> bits;
        const bool in = t >= lo && t < hi;
        if (!__any(in)) continue;
        double f[V], g[V];
#pragma unroll
        for (int u = 0; u < V; ++u) f[u] = W::at(x[i][0], u), g[u] = W::at(x[i][1], u);
        if (a.weight) {
            double sum = 0.0;
#pragma unroll
            for (int u = 0; u < V; ++u) sum = fma(f[u], f[u], sum), sum = fma(g[u], g[u], sum);
            const double r = inverse_root(over_head(sum, bits) * a.inverse_dim + a.eps);
#pragma unroll
            for (int u = 0; u < V; ++u) f[u] *= r * (double)W::at(wp, u), g[u] *= r * (double)W::at(wq, u);
        }
        if (turned && in) {
            int64_t place = p.begin + t;
            if (a.positions) place = a.positions[p.span.row(p.begin + t)];
            float cs[V], sn[V];
            angles_of<V>(a, place < 0 ? 0 : place < a.places ? place : a.places - 1, unit, cs, sn);
            turn<INTER>(f, g, cs, sn);
        }
        x[i][0] = W::of(f), x[i][1] = W::of(g);
        if (in)
#pragma unroll
            for (int u = 0; u < V; ++u) big = max(big, max(abs_bits(W::at(x[i][0], u)), abs_bits(W::at(x[i][1], u))));
    }
    float top = __uint_as_float(over_lanes(big, [](uint32_t s, uint32_t t) { return max(s, t); }));
    if constexpr (TPG > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();  // everybody has read the scale, too
        top = part[0];
#pragma unroll
        for (int i = 1; i < TPG / 64; ++i) top = max_nan(top, part[i]);
    }
    float step = unit8(top);
    if (lo > 0) step = max_nan(before, step);
    if (z.thread == 0) *scale = step;
    if (lo > 0 && !(step == before)) {
        for (int i = z.thread; i < lo * z.dim; i += TPG) held[i] = step > 0.f ? (int8_t)rint((double)held[i] * (double)before / (double)step) : 0;
    }
    const float inverse = inverse8(step);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int t = (z.thread + TPG * i) >> bits;
        if (!(t >= lo && t < hi)) continue;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float y[V];
            typename Q::Held whole;
#pragma unroll
            for (int u = 0; u < V; ++u) y[u] = W::at(x[i][s], u);
            whole8_run<V>(y, step, inverse, whole.v);
            *(typename Q::Held*)(held + t * z.dim + (s ? other : one)) = whole;
        }
    }
}

template <typename T, int TPG, int QPER, bool INTER>
__global__ void __launch_bounds__((Quads<T, TPG>::THREADS)) rope_kv_write_k(RopeKvArgs a) {
    typedef Quads<T, TPG> Q;
    extern __shared__ __align__(16) char rope_lds[];
    __shared__ float part[Q::THREADS / 64];
    if (blockIdx.x >= a.kv_blocks) {
        const uint32_t item = (blockIdx.x - a.kv_blocks) * (Q::THREADS / 64) + (threadIdx.x >> 6);
        if (a.q.weight)
            rope_heads<T, true, INTER>(a.q, a.shape, item);
        else
            rope_heads<T, false, INTER>(a.q, a.shape, item);
        return;
    }
    const Q z(a.w);
    const uint32_t block = blockIdx.x / a.shares;
    const int pair = block * Q::GROUPS + threadIdx.x / TPG, which = pair & 1, head = pair >> 1;
    int share = blockIdx.x - block * a.shares;
    const int b = find_share(share, a.w.g.batch, [&](int i) { return touched_pages(a.w.g, i); });
    if (b < 0 || head >= a.w.kv_heads) return;  // (a workgroup of one group has one head)
    const PageShare p(a.w.g, b, share);
    if (p.page_no < 0) return;
    if (which)
        write_quads<T, TPG, QPER>(a.w, z, p, 1, head, rope_lds, part);
    else
        rope_page<T, TPG, QPER, INTER>(a.w, a.k, z, p, head, part);
}

template <typename T, int TPG, int QPER, bool INTER>
static bool launch_rope_pairs(const char* name, RopeKvArgs& a) {
    typedef Quads<T, TPG> Q;
    auto kernel = rope_kv_write_k<T, TPG, QPER, INTER>;
    const size_t lds = (size_t)Q::GROUPS * a.w.dim * (a.w.g.page + 4);
    if constexpr (TPG == 1024) {  // the largest pages: 66560 bytes
        static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 256 * 260) == hipSuccess;
        if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed"), true;
    }
    const int64_t shares = touched_bound(a.w.g.rows, a.w.g.batch, a.w.g.page), pairs = ceil_div(2 * a.w.kv_heads, Q::GROUPS);
    const int64_t q_blocks = a.q.in ? ceil_div(a.q.rows * a.shape.chunks, Q::THREADS / 64) : 0;
    if ((shares * pairs + q_blocks) * Q::THREADS > UINT32_MAX) return false;
    a.shares = (uint32_t)shares, a.kv_blocks = (uint32_t)(shares * pairs);
    launch(name, kernel, dim3((unsigned)(shares * pairs + q_blocks)), dim3(Q::THREADS), lds, a);
    return true;
}

template <typename T, int TPG, int QPER>
static bool launch_rope_quads(const char* name, RopeKvArgs& a) {
    return a.k.interleaved ? launch_rope_pairs<T, TPG, QPER, true>(name, a) : launch_rope_pairs<T, TPG, QPER, false>(name, a);
}

// In one launch, if rows, angles and weights lie in packs; false if not
template <typename T>
static bool launch_rope_kv(const char* name, RopeKvArgs& a) {
    constexpr int V = 16 / (int)sizeof(T);
    RopeArgs k = a.k;
    k.out = a.w.k, k.out_ld = 0, k.out_col = 0;  // (the cache is aligned)
    if (!quads<T>(a.w) || !in_packs<T>(k) || (a.q.in && !in_packs<T>(a.q))) return false;
    if (a.q.in) a.shape = rope_waves(a.q.rows, a.q.heads, a.q.dim, V, cu_count());
    const int n = a.w.g.page * a.w.dim * (int)sizeof(T) / 64;
    if (n <= 64) return launch_rope_quads<T, 64, 1>(name, a);
    if (n <= 256) return launch_rope_quads<T, 256, 1>(name, a);
    if (n <= 512) return launch_rope_quads<T, 256, 2>(name, a);
    if (n <= 1024) return launch_rope_quads<T, 256, 4>(name, a);
    if constexpr (sizeof(T) == 4) {
        if (n > 2048) return launch_rope_quads<T, 1024, 4>(name, a);
    }
    return launch_rope_quads<T, 1024, 2>(name, a);
}

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------

// Columns of a matrix as memory: rows of `width` bytes, ld bytes apart.
struct Columns {
    uintptr_t at;
    int64_t rows, ld, width;
};
static Columns columns(const Tensor* t, int64_t rows, int64_t ld, int64_t col, int64_t width) {
    const int64_t e = activation_bytes(t);
    return Columns{(uintptr_t)t->data + (uintptr_t)(col * e), rows, ld * e, width * e};
}
// Whether two may have a byte in common.
static bool share_bytes(const Columns& a, const Columns& b) {
    if (a.rows < 1 || b.rows < 1) return false;
    if (a.at + (uintptr_t)((a.rows - 1) * a.ld + a.width) <= b.at || b.at + (uintptr_t)((b.rows - 1) * b.ld + b.width) <= a.at) return false;
    if (a.ld != b.ld) return true;
    int64_t d = ((int64_t)b.at - (int64_t)a.at) % a.ld;
    if (d < 0) d += a.ld;
    return d < a.width || d + b.width > a.ld;
}

static bool rope_weight(const char* name, const char* what, const Tensor* in, Tensor* weight, int heads, int dim, float eps, RopeArgs* a) {
    a->weight = nullptr, a->weight_each = false, a->eps = eps;
    if (!weight) return true;
    if (!has_data(weight) || !good_shape(weight)) return fail(NNC_HIP_EINVAL, name, "%s: NULL data or bad shape", what), false;
    if (weight->dtype != in->dtype) return fail(NNC_HIP_EUNSUPP, name, "%s: of another type than the rows", what), false;
    const int64_t n = numel(weight);
    if (n != dim && n != (int64_t)heads * dim) return fail(NNC_HIP_EINVAL, name, "%s must be [dim] or [heads][dim]", what), false;
    if (!(eps >= 0.f) || !(eps < INFINITY)) return fail(NNC_HIP_EINVAL, name, "eps must not be negative"), false;
    a->weight = weight->data, a->weight_each = n != dim;
    return true;
}

static bool rope_angles(const char* name, Tensor* angles, Tensor* positions, int64_t rows, int dim, bool needs_positions, RopeArgs* a) {
    a->angles = nullptr, a->positions = nullptr, a->places = 1, a->rot = 0;
    if (!angles) {
        if (positions) return fail(NNC_HIP_EINVAL, name, "positions without angles"), false;
        return true;
    }
    if (!has_data(angles) || !good_shape(angles) || angles->ndim != 2 || angles->shape[0] < 1)
        return fail(NNC_HIP_EINVAL, name, "angles must be [positions][rot]"), false;
    if (angles->dtype != NNC_DTYPE_FLOAT32) return fail(NNC_HIP_EUNSUPP, name, "float32 angles only"), false;
    const int64_t rot = angles->shape[1];
    if (rot < 2 || rot % 2 != 0 || rot > dim) return fail(NNC_HIP_EINVAL, name, "%lld of %d dims turned", (long long)rot, dim), false;
    if (angles->shape[0] > INT32_MAX) return fail(NNC_HIP_EUNSUPP, name, "too many angles"), false;
    if (!positions && needs_positions) return fail(NNC_HIP_EINVAL, name, "angles without positions"), false;
    if (positions) {
        if (!has_data(positions) || !good_shape(positions) || numel(positions) != rows)
            return fail(NNC_HIP_EINVAL, name, "positions must be one for each row"), false;
        if (positions->dtype != NNC_DTYPE_INT32) return fail(NNC_HIP_EUNSUPP, name, "int32 positions only"), false;
        a->positions = (const int*)positions->data;
    }
    a->angles = (const float*)angles->data, a->places = angles->shape[0], a->rot = (int)rot;
    return true;
}

// Where the rotated rows go: out's columns, apart from the rows' own or the same.
static bool rope_out(const char* name, const Tensor* in, Tensor* out, int col, int out_col, int64_t width, int64_t rows, int64_t ld, RopeArgs* a) {
    int64_t out_rows = 0, out_ld = 0;
    if (!rows_arg(name, "out", out, out_col, width, &out_rows, &out_ld)) return false;
    if (out->dtype != in->dtype || out_rows != rows) return fail(NNC_HIP_EINVAL, name, "out differs from the input in rows or type"), false;
    const Columns from = columns(in, rows, ld, col, width), to = columns(out, rows, out_ld, out_col, width);
    if (!(from.at == to.at && from.ld == to.ld) && share_bytes(from, to))
        return fail(NNC_HIP_EINVAL, name, "out overlaps the input without being the same columns"), false;
    a->out = out->data, a->out_ld = out_ld, a->out_col = out_col;
    return true;
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_rope(Tensor* in, Tensor* weight, Tensor* angles, Tensor* positions, Tensor* out, int col, int out_col, int heads,
                  int dim, int interleaved, float eps) {
    const char* name = "nnc_hip_rope";
    RopeArgs a{};
    if (heads < 1 || dim < 1 || heads > 65535 || dim > 65536) return fail(NNC_HIP_EINVAL, name, "%d heads of %d", heads, dim);
    const int64_t width = (int64_t)heads * dim;
    if (!rows_arg(name, "in", in, col, width, &a.rows, &a.in_ld)) return;
    if (!rope_weight(name, "weight", in, weight, heads, dim, eps, &a) || !rope_angles(name, angles, positions, a.rows, dim, true, &a) ||
        !rope_out(name, in, out, col, out_col, width, a.rows, a.in_ld, &a))
        return;
    a.in = in->data, a.col = col, a.heads = heads, a.dim = dim, a.inverse_dim = 1.0 / dim, a.interleaved = interleaved != 0;
    if (a.rows == 0) return;
    if (!ready(name)) return;
    const double n = (double)a.rows * (double)width;
    set_work(8.0 * n, 2.0 * n * activation_bytes(in) + 4.0 * (double)a.rows * a.rot);
    launch_rope(name, in->dtype == NNC_DTYPE_FLOAT16, a);
}

void nnc_hip_rope_kv_write(Tensor* q, Tensor* k, Tensor* v, Tensor* q_weight, Tensor* k_weight, Tensor* angles, Tensor* positions,
                           Tensor* q_out, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                           Tensor* starts, Tensor* lengths, int q_col, int heads, int k_col, int v_col, int interleaved, float eps) {
    const char* name = "nnc_hip_rope_kv_write";
    KvArgs w;
    if (!kv_args(name, k, v, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, k_col, v_col, &w)) return;
    const int64_t rows = w.g.rows, kv_width = (int64_t)w.kv_heads * w.dim;
    RopeArgs ka{}, qa{};
    if (!rope_weight(name, "k_weight", k, k_weight, w.kv_heads, w.dim, eps, &ka) || !rope_angles(name, angles, positions, rows, w.dim, false, &ka)) return;
    ka.in = k->data, ka.in_ld = w.k_ld, ka.col = k_col, ka.heads = w.kv_heads;
    ka.rows = rows, ka.dim = w.dim, ka.inverse_dim = 1.0 / w.dim, ka.interleaved = interleaved != 0, ka.g = w.g;
    if (q) {
        qa = ka;
        if (heads < 1 || heads > 65535) return fail(NNC_HIP_EINVAL, name, "%d heads", heads);
        const int64_t width = (int64_t)heads * w.dim;
        int64_t q_rows = 0;
        if (!rows_arg(name, "q", q, q_col, width, &q_rows, &qa.in_ld)) return;
        if (q_rows != rows || q->dtype != k->dtype) return fail(NNC_HIP_EINVAL, name, "q and k differ in rows or type");
        if (!rope_weight(name, "q_weight", q, q_weight, heads, w.dim, eps, &qa)) return;
        qa.in = q->data, qa.col = q_col, qa.heads = heads;
        Tensor* out = q_out ? q_out : q;
        if (!rope_out(name, q, out, q_col, q_out ? 0 : q_col, width, rows, qa.in_ld, &qa)) return;
        const Columns to = columns(out, rows, qa.out_ld, qa.out_col, width);
        if (share_bytes(to, columns(k, rows, w.k_ld, k_col, kv_width)) || share_bytes(to, columns(v, rows, w.v_ld, v_col, kv_width)))
            return fail(NNC_HIP_EINVAL, name, "the rotated queries would lie over keys or values");
    } else if (q_weight || q_out) {
        return fail(NNC_HIP_EINVAL, name, "q_weight or q_out without q");
    }
    if (rows == 0 || w.g.batch == 0 || (w.g.width == 0 && !q)) return;
    if (!ready(name)) return;
    const bool f16 = k->dtype == NNC_DTYPE_FLOAT16;
    const double n = (double)rows * activation_bytes(k);
    RopeKvArgs all{};
    all.w = w, all.q = qa, all.k = ka;
    if (w.g.width == 0) {  // no pages to write to
        set_work(8.0 * rows * heads * w.dim, 2.0 * n * heads * w.dim);
        return launch_rope("nnc_hip_rope_kv_write_q", f16, qa);
    }
    set_work(8.0 * rows * (q ? heads * w.dim : 0) + 20.0 * rows * kv_width, 2.0 * n * (q ? heads * w.dim : 0) + 2.0 * (n + rows) * kv_width);
    if (f16 ? launch_rope_kv<half_t>(name, all) : launch_rope_kv<float>(name, all)) return;
    // the rotated keys pass through scratch
    const size_t bytes = (size_t)rows * kv_width * activation_bytes(k);
    ka.out = workspace(bytes);
    if (!ka.out) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes of rotated keys", bytes);
    ka.out_ld = kv_width, ka.out_col = 0;
    w.k_rows = ka.out, w.k_ld = kv_width, w.k_col = 0;
    if (q) {
        set_work(8.0 * rows * heads * w.dim, 2.0 * n * heads * w.dim);
        launch_rope("nnc_hip_rope_kv_write_q", f16, qa);
    }
    set_work(8.0 * rows * kv_width, 2.0 * n * kv_width);
    launch_rope("nnc_hip_rope_kv_write_k", f16, ka);
    set_work(12.0 * rows * kv_width, 2.0 * (n + rows) * kv_width);
    launch_write(name, f16, w);
}

}  // extern "C"
