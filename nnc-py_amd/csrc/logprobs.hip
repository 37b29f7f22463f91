// What a model answers with: log probabilities of given tokens, the entropy and
// the likeliest tokens of rows of logits (nnc_hip_token_logprobs). No reference
// counterpart.
//
//   m = max_i x_i,  S = sum_i e^(t (x_i - m));  log p_i = t (x_i - m) - log S
//   entropy = log S - sum_i t (x_i - m) e^(t (x_i - m)) / S
//
// A workgroup has a segment of a row in registers, so it is read once: maximum,
// then the sums against it, then the likeliest. A row's largest term is 1, and
// where it leaves 2^-24 and less to all others, entropy and the largest token's
// log probability are made of those: so terms that are 1 are counted, the others
// summed for themselves, two packs of them in float32 and these sums in float64.
//
// The likeliest tokens: n values at least reach the n-th largest of a wave's lane
// maxima, and the least of the waves' (n / waves)-th largest; the highest of these
// bars is what few more than n reach. Those gather in LDS, are sorted, 64 to a
// wave, as whole numbers that compare as (value, earlier index) do, and merged.
// If more than 256 reach it, or 64 where a wave has whole rows (equal values, rows
// of -infinity), each wave keeps a list of its best 64, one a lane, and merges 64 at
// a time into it. The last segment to arrive joins a row's segments.
#include "lanes.h"
#include "mfma_tile.h"

namespace nnc {

struct LogprobArgs {
    const void* logits;
    const int* tokens;
    float *logprob, *entropy;
    int* top_index;
    float* top_logprob;
    float* part;    // [row][segment][SLOT]: a segment's sums and tokens
    int* counters;  // [row], zero
    int64_t rows, vocab;
    int top, segments, each;  // packs of a segment
    int64_t row0;   // of the launch
    float scale;
};

// Whole numbers ordered as the values are, the earlier of equal ones first: a
// value's bits, negative ones turned round, before the index's complement. 0 is
// below all of them.
__device__ __forceinline__ u64 rank_of(float x, uint32_t index) {
    const uint32_t bits = __float_as_uint(x + 0.f);  // (-0 becomes 0)
    return (u64)(bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(u64 rank) {
    const uint32_t u = (uint32_t)(rank >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int index_of(u64 rank) { return (int)(0xffffffffu - (uint32_t)rank); }

template <typename K>
__device__ __forceinline__ K larger(K a, K b) { return a > b ? a : b; }
template <typename K>
__device__ __forceinline__ K smaller(K a, K b) { return a > b ? b : a; }

// 64 keys, one a lane, in rising order
template <int RUN, int J, typename K>
__device__ __forceinline__ K sort_step(K key) {
    const int lane = threadIdx.x & 63;
    const K other = lane_xor<J>(key);
    key = ((lane & RUN) == 0) == ((lane & J) == 0) ? smaller(key, other) : larger(key, other);
    if constexpr (J > 1) return sort_step<RUN, J / 2>(key);
    return key;
}
template <typename K>
__device__ __forceinline__ K sort_rising(K key) {
    key = sort_step<2, 1>(key);
    key = sort_step<4, 2>(key);
    key = sort_step<8, 4>(key);
    key = sort_step<16, 8>(key);
    key = sort_step<32, 16>(key);
    return sort_step<64, 32>(key);
}
// The 64 largest of a falling and a rising sequence, falling
template <int J>
__device__ __forceinline__ u64 merge_step(u64 key) {
    const u64 other = lane_xor<J>(key);
    key = (threadIdx.x & J) == 0 ? larger(key, other) : smaller(key, other);
    if constexpr (J > 1) return merge_step<J / 2>(key);
    return key;
}
__device__ __forceinline__ u64 merge_falling(u64 falling, u64 rising) { return merge_step<32>(larger(falling, rising)); }

// Sums of a part of a row: the terms e^(t (x - m)) that are less than 1, how
// many are 1, and all of them times their exponents, in powers of two.
struct RowSums {
    float m;  // -infinity: nothing yet
    double rest, ones, weighted;
};
// what an exponent that stands for no weight is set to
static constexpr float kFar = -1000.f;
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void rebase(RowSums& s, float m, float c) {
    const float d = fmaxf((s.m - base_of(m)) * c, kFar);
    if (m > s.m) {
        const double a = __builtin_amdgcn_exp2f(d);
        s.weighted = a * (s.weighted + d * (s.rest + s.ones));
        s.rest = a * (s.rest + s.ones);
        s.ones = 0.0;
        s.m = m;
    }
}
__device__ __forceinline__ void add_sums(RowSums& s, RowSums t, float c) {
    const float m = fmaxf(s.m, t.m);
    rebase(s, m, c), rebase(t, m, c);
    s.rest += t.rest, s.ones += t.ones, s.weighted += t.weighted;
}

// A pack's largest value
template <typename T>
__device__ __forceinline__ float largest_of(nt_u32x4 pack) {
    uint32_t most = pack[0];
#pragma unroll
    for (int u = 1; u < 4; ++u) most = Words<T>::max_of(most, pack[u]);
    const nt_u32x4 both = {most, most, most, most};
    return sizeof(T) == 4 ? Words<T>::at(both, 0) : fmaxf(Words<T>::at(both, 0), Words<T>::at(both, 1));
}

// Takes the values that are the maximum out of a lane's packs; how many. (Few of
// a wave's packs have one: the others are passed over together.)
template <typename T, int PACKS>
__device__ __forceinline__ float take_out(nt_u32x4 (&raw)[PACKS], float m) {
    float ones = 0.f;
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
        if (!__any(largest_of<T>(raw[p]) == m)) continue;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t w = raw[p][u];
            if constexpr (sizeof(T) == 4) {
                const bool one = __uint_as_float(w) == m;
                raw[p][u] = one ? Words<T>::NONE : w;
                ones += one ? 1.f : 0.f;
            } else {
                const f16x2 v = __builtin_bit_cast(f16x2, w);
                const bool one = (float)v[0] == m, other = (float)v[1] == m;
                raw[p][u] = (one ? 0xfc00u : w & 0xffffu) | (other ? 0xfc000000u : w & 0xffff0000u);
                ones += (one ? 1.f : 0.f) + (other ? 1.f : 0.f);
            }
            asm volatile("" : "+v"(ones));  // (one after the other: the comparisons of all of them are more than the registers hold)
        }
    }
    return ones;
}

// A lane's packs, without the maximum m, against it: terms 2^t, t = c (x - m). As
// c x - (c m), one operation, whose second part's rounding is the same for all and
// put right in the sums; FAR: where that would overflow. (A NaN stays in `rest`.)
template <typename T, bool FAR, int PACKS>
__device__ __forceinline__ void sum_packs(nt_u32x4 (&raw)[PACKS], float m, float c, RowSums& s) {
    constexpr int V = Words<T>::V;
    const float base = base_of(m), shift = base * c, off = FAR ? 0.f : fmaf(base, c, -shift);
#pragma unroll
    for (int p = 0; p < PACKS; p += 2) {
        float r[4], w[4];
#pragma unroll
        for (int u = 0; u < 2 * V; ++u) {
            const float x = Words<T>::at(raw[p + u / V], u % V);
            const float t = FAR ? (x - base) * c : fmaf(x, c, -shift), e = __builtin_amdgcn_exp2f(t), far = fmaxf(t, kFar);
            r[u % 4] = u < 4 ? e : r[u % 4] + e;
            w[u % 4] = u < 4 ? e * far : fmaf(e, far, w[u % 4]);
        }
        s.rest += (r[0] + r[1]) + (r[2] + r[3]);
        s.weighted += (w[0] + w[1]) + (w[2] + w[3]);
    }
    if (!FAR) {
        const double a = 1.0 - 0.69314718055994530942 * (double)off;  // 2^-off, which is 2^-24 of the shift at most
        s.weighted = a * (s.weighted - off * s.rest);
        s.rest *= a;
    }
}

// A wave's likeliest tokens
struct Likeliest {
    u64 list;   // falling
    u64 bar;    // the n-th, 0 while there are fewer
    u64* room;  // [64] LDS
    int held;
    __device__ __forceinline__ void init(u64* lds) { list = bar = 0, room = lds, held = 0; }
    __device__ __forceinline__ void merge(u64 rising, int n) {
        list = merge_falling(list, rising);
        bar = __shfl(list, n - 1);
    }
    __device__ __forceinline__ void flush(int n) {
        if (held == 0) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int lane = threadIdx.x & 63;
        const u64 key = lane < held ? room[lane] : 0;
        held = 0;
        merge(sort_rising(key), n);
        __builtin_amdgcn_wave_barrier();
    }
    // the lanes' tokens where `is`
    __device__ __forceinline__ void put(bool is, float x, int64_t index, int n) {
        const u64 key = rank_of(x, (uint32_t)index);
        u64 mask = __ballot(is && key > bar);
        if (!mask) return;
        if (held + __popcll(mask) > 64) {
            flush(n);
            mask = __ballot(is && key > bar);
            if (!mask) return;
        }
        const int lane = threadIdx.x & 63;
        if (mask >> lane & 1) room[held + __popcll(mask & ((1ull << lane) - 1))] = key;
        held += __popcll(mask);
    }
};

// Floats of a segment's slot: rest, ones, weighted (8 bytes each), m, then the
// tokens.
static constexpr int kSlotHead = 8;
__host__ __device__ constexpr int slot_floats(int top) { return kSlotHead + 2 * top; }

// NW waves to a segment of a row, PACKS packs of 16 bytes a lane as they lie in
// memory: a row's first and last pack may hold others' values.
template <typename T, int NW, int PACKS, bool TOP>
__global__ void __launch_bounds__(64 * NW) logprobs_k(LogprobArgs a) {
    constexpr int V = Words<T>::V;
    __shared__ RowSums sums[NW];
    __shared__ float tops[NW], bars[NW], parts[NW];
    __shared__ int gathered;
    __shared__ u64 room[NW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float c = a.scale * 1.44269504088896340736f;
    const uint32_t line = blockIdx.x / (uint32_t)a.segments, segment = blockIdx.x - line * (uint32_t)a.segments;
    const int64_t row = a.row0 + line;
    const T* x = (const T*)a.logits + row * a.vocab;
    const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
    const int64_t first = (int64_t)segment * a.each, rest = (off + a.vocab + V - 1) / V - first;
    const int n = (int)(rest < a.each ? rest : a.each), at = wave * 64 + lane;
    const int64_t index0 = first * V - off;  // of the segment's first value, as if its pack were the row's own
    // packs that are the row's own: [own, own_end) of the segment's
    const int own = first == 0 && off > 0 ? 1 : 0, own_end = rest <= a.each && (off + a.vocab) % V ? n - 1 : n;
    const nt_u32x4* packs = (const nt_u32x4*)(x - off) + first;
    nt_u32x4 raw[PACKS];
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
        const int j = at + NW * 64 * p;
        raw[p] = nt_u32x4{Words<T>::NONE, Words<T>::NONE, Words<T>::NONE, Words<T>::NONE};
        if (j >= own && j < own_end) raw[p] = packs[j];
    }
    for (int edge = 0; edge < 2; ++edge) {
        const int e = edge ? n - 1 : 0;
        if (edge ? own_end == n || e < own : own == 0) continue;
        Pack<T, V> part;
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const int64_t i = index0 + (int64_t)e * V + u;
            part.v[u] = i >= 0 && i < a.vocab ? x[i] : (T)-INFINITY;
        }
        const nt_u32x4 words = __builtin_bit_cast(nt_u32x4, part);
#pragma unroll
        for (int p = 0; p < PACKS; ++p) raw[p] = at + NW * 64 * p == e ? words : raw[p];
    }
    nt_u32x4 best = raw[0];
#pragma unroll
    for (int p = 1; p < PACKS; ++p)
#pragma unroll
        for (int u = 0; u < 4; ++u) best[u] = Words<T>::max_of(best[u], raw[p][u]);
    float mine = -INFINITY;
#pragma unroll
    for (int u = 0; u < V; ++u) mine = fmaxf(mine, Words<T>::at(best, u));
    float top = mine, bar = -INFINITY;
    if (TOP) {
        const float order = sort_rising(mine);
        top = __shfl(order, 63), bar = __shfl(order, 64 - a.top);
        const float part = __shfl(order, 64 - (a.top + NW - 1) / NW);
        if (NW > 1) {
            if (lane == 0) tops[wave] = top, bars[wave] = bar, parts[wave] = part;
            if (threadIdx.x == 0) gathered = 0;
            __syncthreads();
            float least = INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, tops[w]), bar = fmaxf(bar, bars[w]), least = fminf(least, parts[w]);
            bar = fmaxf(bar, least);
        } else {
            if (threadIdx.x == 0) gathered = 0;
            __syncthreads();
        }
    } else {
        top = over_lanes(mine, [](float p, float q) { return fmaxf(p, q); });
        if (NW > 1) {
            if (lane == 0) tops[wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, tops[w]);
        }
    }
    Likeliest likeliest;
    likeliest.init(room[wave]);
    if (TOP) {
        uint32_t reach = 0;  // packs that reach the bar
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const bool hit = largest_of<T>(raw[p]) >= bar;
            reach |= hit ? 1u << p : 0u;
        }
        auto pack_of = [&](int which) {
            nt_u32x4 pack = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < PACKS; ++p) pack |= raw[p] & (which == p ? 0xffffffffu : 0u);
            return pack;
        };
        constexpr int ROOM = NW * 64 < 256 ? NW * 64 : 256;
        u64* all = room[0];
        for (uint32_t hits = reach; hits; hits &= hits - 1) {
            const int which = __ffs(hits) - 1;
            const nt_u32x4 pack = pack_of(which);
            const int64_t i = index0 + (int64_t)(at + NW * 64 * which) * V;
            uint32_t values = 0;
#pragma unroll
            for (int u = 0; u < V; ++u) values |= Words<T>::at(pack, u) >= bar ? 1u << u : 0u;
            if (bar == -INFINITY) {  // what is not the row's own reaches it, too
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if (at + NW * 64 * which >= n || i + u < 0 || i + u >= a.vocab) values &= ~(1u << u);
            }
            int place = atomicAdd(&gathered, __popc(values));
            for (; values; values &= values - 1, ++place) {
                const int u = __ffs(values) - 1;
                const uint32_t w = (u * (int)sizeof(T) & 8 ? (u * (int)sizeof(T) & 4 ? pack[3] : pack[2]) : u * (int)sizeof(T) & 4 ? pack[1] : pack[0]);
                const nt_u32x4 first_of = {sizeof(T) == 2 && (u & 1) ? w >> 16 : w, 0, 0, 0};
                if (place < ROOM) all[place] = rank_of(Words<T>::at(first_of, 0), (uint32_t)(i + u));
            }
        }
        __syncthreads();
        const int total = gathered;
        if (total <= ROOM) {
            u64 key = 0;
            if (wave * 64 < total) {
                key = sort_rising(threadIdx.x < total ? all[threadIdx.x] : 0);
                if (wave > 0) all[threadIdx.x] = key;
            }
            if (wave == 0) likeliest.merge(key, a.top);
            if (NW > 1 && total > 64) {
                __syncthreads();
                if (wave == 0)
                    for (int w = 1; w * 64 < total; ++w) likeliest.merge(room[w][lane], a.top);
            }
        } else {
            __syncthreads();
            for (uint32_t hits = reach; __any(hits); hits &= hits - 1) {
                const int which = hits ? __ffs(hits) - 1 : 0;
                nt_u32x4 pack = pack_of(which);
#pragma unroll 1
                for (int u = 0; u < V; ++u) {
                    const float y = Words<T>::at(pack, 0);
                    const int64_t i = index0 + (int64_t)(at + NW * 64 * which) * V + u;
                    const bool is = hits && y >= bar && at + NW * 64 * which < n && i >= 0 && i < a.vocab;
                    if (__any(is)) likeliest.put(is, y, i, a.top);
                    pack = Words<T>::next(pack);
                }
            }
            likeliest.flush(a.top);
            if (NW > 1) {
                room[wave][63 - lane] = likeliest.list;
                __syncthreads();
                if (wave == 0)
                    for (int w = 1; w < NW; ++w) likeliest.merge(room[w][lane], a.top);
            }
        }
    }
    RowSums s{top, 0.0, 0.0, 0.0};
    if (top > -INFINITY && __any(mine == top)) s.ones = take_out<T>(raw, top);
    if (fabsf(base_of(top) * c) < 4096.f)  // what `off` neglects, its square, is below 2^-25
        sum_packs<T, false>(raw, top, c, s);
    else
        sum_packs<T, true>(raw, top, c, s);
    // join the lanes, the waves, the segments
    auto add = [](double p, double q) { return p + q; };
    s.rest = over_lanes(s.rest, add), s.ones = over_lanes(s.ones, add), s.weighted = over_lanes(s.weighted, add);
    if (NW > 1) {
        if (lane == 0) sums[wave] = s;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int w = 1; w < NW; ++w) {
                s.rest += sums[w].rest, s.ones += sums[w].ones, s.weighted += sums[w].weighted;
            }
        }
    }
    if (NW > 1 && a.segments > 1) {  // (a wave has whole rows)
        const int slot = slot_floats(a.top);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(a.part);
        auto put8 = [&](uint32_t at, u64 x) {
            store_partial(r, at * 4u, __uint_as_float((uint32_t)x));
            store_partial(r, at * 4u + 4u, __uint_as_float((uint32_t)(x >> 32)));
        };
        auto get8 = [&](uint32_t at) {
            return (u64)__float_as_uint(load_partial(r, at * 4u)) | (u64)__float_as_uint(load_partial(r, at * 4u + 4u)) << 32;
        };
        if (wave == 0) {
            const uint32_t at = blockIdx.x * (uint32_t)slot;
            if (lane == 0) {
                put8(at, __double_as_longlong(s.rest));
                put8(at + 2, __double_as_longlong(s.ones));
                put8(at + 4, __double_as_longlong(s.weighted));
                store_partial(r, at * 4u + 24u, s.m);
            }
            if (TOP && lane < a.top) put8(at + kSlotHead + 2 * lane, likeliest.list);
        }
        if (!finish_arrive(a.counters + line, a.segments - 1)) return;
        if (wave == 0) {
            s = RowSums{-INFINITY, 0.0, 0.0, 0.0};
            for (int g = lane; g < a.segments; g += 64) {
                const uint32_t at = (uint32_t)(line * a.segments + g) * slot;
                add_sums(s, RowSums{load_partial(r, at * 4u + 24u), __longlong_as_double(get8(at)), __longlong_as_double(get8(at + 2)),
                                    __longlong_as_double(get8(at + 4))}, c);
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1)
                add_sums(s, RowSums{__shfl_xor(s.m, o), __shfl_xor(s.rest, o), __shfl_xor(s.ones, o), __shfl_xor(s.weighted, o)}, c);
        }
        if (TOP) {
            likeliest.init(room[wave]);
            for (int g = wave; g < a.segments; g += NW) {
                const uint32_t at = (uint32_t)(line * a.segments + g) * slot + kSlotHead;
                likeliest.merge(63 - lane < a.top ? get8(at + 2 * (63 - lane)) : 0, a.top);
            }
            room[wave][63 - lane] = likeliest.list;
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int w = 1; w < NW; ++w) likeliest.merge(room[w][lane], a.top);
        }
    }
    if (wave == 0) {
        const double sum = s.rest + s.ones;
        const bool ok = fabsf(s.m) < INFINITY && sum == sum;
        const double log_sum = s.ones == 1.0 ? log1p(s.rest) : log(sum);
        auto log_p = [&](float y) { return (float)((double)a.scale * ((double)y - (double)s.m) - log_sum); };
        if (lane == 0) {
            if (a.entropy) a.entropy[row] = ok ? (float)(log_sum - s.weighted / sum * 0.69314718055994530942) : NAN;
            if (a.logprob) {
                const int t = a.tokens[row];
                a.logprob[row] = ok && t >= 0 && t < a.vocab ? log_p((float)x[t]) : NAN;
            }
        }
        if (TOP && lane < a.top) {
            const u64 key = likeliest.list;
            a.top_index[row * a.top + lane] = ok && key ? index_of(key) : -1;
            a.top_logprob[row * a.top + lane] = !ok ? NAN : key ? log_p(value_of(key)) : -INFINITY;
        }
    }
}

template <typename T, int NW, int PACKS, bool TOP>
static void launch_packs(const char* name, LogprobArgs a, int64_t packs) {
    a.segments = (int)ceil_div(packs, NW * 64 * PACKS);
    a.each = (int)ceil_div(packs, a.segments);
    // rows at a time: their segments' slots and counters
    const int64_t all = a.rows, slots = (int64_t)a.segments * slot_floats(a.top) * sizeof(float);
    const int64_t most = a.segments > 1 ? ((int64_t)64 << 20) / slots : (int64_t)1 << 22;
    a.rows = most < 1 ? 1 : most < all ? most : all;
    if (a.segments > 1) {
        a.part = workspace((size_t)(a.rows * slots));
        a.counters = tile_counters((size_t)a.rows);
        if (!a.part || !a.counters) return fail(NNC_HIP_ENOMEM, name, "no workspace for %lld bytes of partial sums", (long long)(a.rows * slots));
    }
    for (const int64_t each = a.rows; a.row0 < all; a.row0 += each) {
        a.rows = each < all - a.row0 ? each : all - a.row0;
        const dim3 grid((unsigned)(a.rows * a.segments));
        const double n = (double)a.rows * (double)a.vocab;
        set_work(6.0 * n, n * sizeof(T) + 8.0 * (double)a.rows * (1 + a.top));
        launch(name, logprobs_k<T, NW, PACKS, TOP>, grid, dim3(64 * NW), 0, a);
    }
}

// A wave to a row that fits into its registers, else four to a segment: of 4
// packs a lane while that makes few workgroups, else of 16, or 8 where no tokens
// are asked for. 16 and 8 packs, us: [512, 128256] f16, 20 tokens 50 and 56, none
// 37 and 33; [2048, 32000] f16, 1 token 37 and 49; [301, 50257] fp32, none 18 and
// 16. (12 packs with 20 tokens 53; eight waves with 8 packs were slower by a
// tenth.) A copy's rate leaves 26 us for the first two. With tokens a third of the
// time is the sorting of candidates, and 150 registers leave 3 waves a SIMD to cover
// it; without, the sums keep the vector units busy for 82% of the time. 8 rows of
// 32000 in fp32 take 9.7 us with 5 tokens, 6.0 without: load, bar, candidates, sort,
// join are one chain.
template <typename T, bool TOP>
static void launch_logprobs(const char* name, const LogprobArgs& a) {
    const int64_t packs = a.vocab * (int64_t)sizeof(T) / 16 + 2;
    if (packs <= 256) return launch_packs<T, 1, 4, TOP>(name, a, packs);
    if (packs <= 512 && a.rows >= cu_count()) return launch_packs<T, 1, 8, TOP>(name, a, packs);
    if (ceil_div(packs, 1024) * a.rows <= 4 * (int64_t)cu_count()) return launch_packs<T, 4, 4, TOP>(name, a, packs);
    launch_packs<T, 4, TOP ? 16 : 8, TOP>(name, a, packs);
}

static bool row_output(const char* name, const char* what, Tensor* t, int dtype, int64_t n) {
    if (!t) return true;
    if (!has_data(t) || !good_shape(t)) return fail(NNC_HIP_EINVAL, name, "%s: NULL data or bad shape", what), false;
    if ((int)t->dtype != dtype) return fail(NNC_HIP_EUNSUPP, name, "%s: wrong type", what), false;
    if (n >= 0 && numel(t) != n) return fail(NNC_HIP_EINVAL, name, "%s: wrong size", what), false;
    return true;
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_token_logprobs(Tensor* logits, Tensor* tokens, Tensor* logprob, Tensor* entropy, Tensor* top_index, Tensor* top_logprob,
                            float scale) {
    const char* name = "nnc_hip_token_logprobs";
    LogprobArgs a{};
    int64_t ld = 0;
    if (!rows_arg(name, "logits", logits, 0, 1, &a.rows, &ld)) return;
    a.vocab = ld;
    if (!tokens != !logprob || !top_index != !top_logprob)
        return fail(NNC_HIP_EINVAL, name, "tokens go with logprob, top_index with top_logprob");
    if (!row_output(name, "tokens", tokens, NNC_DTYPE_INT32, a.rows) || !row_output(name, "logprob", logprob, NNC_DTYPE_FLOAT32, a.rows) ||
        !row_output(name, "entropy", entropy, NNC_DTYPE_FLOAT32, a.rows) || !row_output(name, "top_index", top_index, NNC_DTYPE_INT32, -1) ||
        !row_output(name, "top_logprob", top_logprob, NNC_DTYPE_FLOAT32, -1))
        return;
    if (top_index) {
        const int64_t n = top_index->shape[top_index->ndim - 1];
        if (n < 1 || n > 64) return fail(NNC_HIP_EUNSUPP, name, "%lld alternatives (1 to 64)", (long long)n);
        if (numel(top_index) != a.rows * n || numel(top_logprob) != a.rows * n || top_logprob->shape[top_logprob->ndim - 1] != n)
            return fail(NNC_HIP_EINVAL, name, "top_index and top_logprob must be [rows][n]");
        a.top = (int)n;
    }
    if (!(scale > 0.f) || !(scale < INFINITY)) return fail(NNC_HIP_EINVAL, name, "scale must be positive");
    if (a.rows == 0 || (!logprob && !entropy && !top_index)) return;
    if (!ready(name)) return;
    a.logits = logits->data, a.scale = scale;
    if (logprob) a.tokens = (const int*)tokens->data, a.logprob = (float*)logprob->data;
    if (entropy) a.entropy = (float*)entropy->data;
    if (top_index) a.top_index = (int*)top_index->data, a.top_logprob = (float*)top_logprob->data;
    if (logits->dtype == NNC_DTYPE_FLOAT16)
        a.top ? launch_logprobs<half_t, true>(name, a) : launch_logprobs<half_t, false>(name, a);
    else
        a.top ? launch_logprobs<float, true>(name, a) : launch_logprobs<float, false>(name, a);
}

}  // extern "C"
