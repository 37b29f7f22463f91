// What a model answers with: log probabilities of given tokens, the entropy and
// the likeliest tokens of rows of logits (nnc_hip_token_logprobs). No reference
// counterpart.
//
//   m = max_i x_i,  S = sum_i e^(t (x_i - m));  log p_i = t (x_i - m) - log S
//   entropy = log S - sum_i t (x_i - m) e^(t (x_i - m)) / S
//
// in one pass with a running maximum for each lane. A row's largest term is 1,
// and where it leaves 2^-24 and less to all others, entropy and the largest
// token's log probability are made of those: so terms of the lane's maximum are
// counted, the others summed for themselves, 16 or 32 of them in float32 and
// these sums in float64.
//
// The likeliest tokens: a wave keeps 64 of them in order, one a lane, as whole
// numbers that compare as (value, earlier index) do. A batch of a few packs a
// lane only looks for tokens if one is above the n-th that the wave has; they
// gather in LDS, and 64 at a time are sorted and merged, which a row needs about
// n log(vocab / n) / 64 times for each wave. The first bar is the n-th largest of
// the lanes' maxima in the first batch.
//
// Rows are cut into segments while there are fewer than the GPU has room for;
// the last to arrive joins them.
#include "mfma_tile.h"
#include "quant8.h"

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
    int top, segments;
    float scale;
};

// Whole numbers ordered as the values are, the earlier of equal ones first: a
// value's bits, negative ones turned round, before the index's complement. 0 is
// below all of them.
typedef unsigned long long u64;
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
template <typename K>
__device__ __forceinline__ K sort_rising(K key) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const K other = __shfl_xor(key, j);
            const bool up = (lane & k) == 0, low = (lane & j) == 0;
            key = up == low ? smaller(key, other) : larger(key, other);
        }
    return key;
}
// The 64 largest of a falling and a rising sequence, falling
__device__ __forceinline__ u64 merge_falling(u64 falling, u64 rising) {
    const int lane = threadIdx.x & 63;
    u64 key = larger(falling, rising);
#pragma unroll
    for (int j = 32; j > 0; j >>= 1) {
        const u64 other = __shfl_xor(key, j);
        key = (lane & j) == 0 ? larger(key, other) : smaller(key, other);
    }
    return key;
}

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
__device__ __forceinline__ RowSums shuffled(const RowSums& s, int o) {
    return RowSums{__shfl_xor(s.m, o), __shfl_xor(s.rest, o), __shfl_xor(s.ones, o), __shfl_xor(s.weighted, o)};
}

// A wave's likeliest tokens
struct Likeliest {
    u64 list;   // falling
    u64 bar;    // the n-th, 0 while there are fewer
    float over;  // its value
    u64* room;  // [64] LDS
    int held;
    __device__ __forceinline__ void init(u64* lds) { list = bar = 0, over = -INFINITY, room = lds, held = 0; }
    __device__ __forceinline__ void merge(u64 rising, int n) {
        list = merge_falling(list, rising);
        bar = __shfl(list, n - 1);
        over = bar ? value_of(bar) : -INFINITY;
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

// NW waves to a segment of a row. A row is read in packs of 16 bytes as they
// lie in memory: its first and last pack may hold others' values.
template <typename T, int NW, bool TOP>
__global__ void __launch_bounds__(64 * NW) logprobs_k(LogprobArgs a) {
    constexpr int V = 16 / (int)sizeof(T), PACKS = 4;
    typedef Pack<T, V> P;
    __shared__ RowSums sums[NW];
    __shared__ u64 room[NW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float c = a.scale * 1.44269504088896340736f;
    const int64_t units = a.rows * a.segments;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t row = unit / a.segments;
        const int segment = (int)(unit - row * a.segments);
        const T* x = (const T*)a.logits + row * a.vocab;
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const P* packs = (const P*)(x - off);
        const int64_t count = (off + a.vocab + V - 1) / V;  // of packs
        const int64_t first = segment * count / a.segments, last = (segment + 1) * count / a.segments;
        RowSums s{-INFINITY, 0.0, 0.0, 0.0};
        Likeliest likeliest;
        likeliest.init(room[wave]);
        bool begun = false;
        for (int64_t at = first + wave * 64 * PACKS; at < last; at += NW * 64 * PACKS) {
            float v[PACKS][V];
            P raw[PACKS];
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                const int64_t k = at + 64 * p + lane;
                if (k < last && k * V >= off && (k + 1) * V <= off + a.vocab) {
                    raw[p] = packs[k];
                } else {
#pragma unroll
                    for (int u = 0; u < V; ++u) {
                        const int64_t i = k * V + u - off;
                        raw[p].v[u] = k < last && i >= 0 && i < a.vocab ? x[i] : (T)-INFINITY;
                    }
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int p = 0; p < PACKS; ++p)
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    v[p][u] = (float)raw[p].v[u];
                    top = fmaxf(top, v[p][u]);
                }
            if (__any(top > s.m)) rebase(s, fmaxf(s.m, top), c);
            const float base = base_of(s.m);
            float rest[PACKS], weighted[PACKS], ones = 0.f;
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                float r[V], w[V];
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    const float t = (v[p][u] - base) * c, e = __builtin_amdgcn_exp2f(t);  // (a NaN stays in the sum)
                    const bool one = v[p][u] == s.m;
                    ones += one ? 1.f : 0.f;
                    r[u] = one ? 0.f : e;
                    w[u] = e * fmaxf(t, kFar);
                }
#pragma unroll
                for (int n = V / 2; n > 0; n /= 2)
#pragma unroll
                    for (int u = 0; u < n; ++u) r[u] += r[u + n], w[u] += w[u + n];
                rest[p] = r[0], weighted[p] = w[0];
            }
            static_assert(PACKS == 4, "pairs of pairs");
            s.rest += (rest[0] + rest[1]) + (rest[2] + rest[3]);
            s.weighted += (weighted[0] + weighted[1]) + (weighted[2] + weighted[3]);
            if (s.m > -INFINITY) s.ones += ones;
            if (TOP) {
                // from the second batch on equal ones come after those that the wave has
                float over = likeliest.over;
                bool look = __any(top > over);
                if (!begun) {
                    over = __shfl(sort_rising(top), 64 - a.top);
                    look = true;
                }
                const bool equal = !begun || !likeliest.bar;
                begun = true;
                if (look || equal) {
#pragma unroll
                    for (int p = 0; p < PACKS; ++p)
#pragma unroll
                        for (int u = 0; u < V; ++u) {
                            const int64_t i = (at + 64 * p + lane) * V + u - off;
                            const bool is = (equal ? v[p][u] >= over : v[p][u] > over) && at + 64 * p + lane < last && i >= 0 && i < a.vocab;
                            if (__any(is)) likeliest.put(is, v[p][u], i, a.top);
                        }
                    if (!likeliest.bar) likeliest.flush(a.top);
                }
            }
        }
        if (TOP) likeliest.flush(a.top);
        // join the lanes, the waves, the segments
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) add_sums(s, shuffled(s, o), c);
        if (NW > 1) {
            if (lane == 0) sums[wave] = s;
            if (TOP) room[wave][63 - lane] = likeliest.list;
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int w = 1; w < NW; ++w) {
                    add_sums(s, sums[w], c);
                    if (TOP) likeliest.merge(room[w][lane], a.top);
                }
            }
        }
        if (a.segments > 1) {
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
                const uint32_t at = (uint32_t)unit * slot;
                if (lane == 0) {
                    put8(at, __double_as_longlong(s.rest));
                    put8(at + 2, __double_as_longlong(s.ones));
                    put8(at + 4, __double_as_longlong(s.weighted));
                    store_partial(r, at * 4u + 24u, s.m);
                }
                if (TOP && lane < a.top) put8(at + kSlotHead + 2 * lane, likeliest.list);
            }
            if (!finish_arrive(a.counters + row, a.segments - 1)) {
                __syncthreads();
                continue;
            }
            if (wave == 0) {
                s = RowSums{-INFINITY, 0.0, 0.0, 0.0};
                for (int g = lane; g < a.segments; g += 64) {
                    const uint32_t at = (uint32_t)(row * a.segments + g) * slot;
                    add_sums(s, RowSums{load_partial(r, at * 4u + 24u), __longlong_as_double(get8(at)), __longlong_as_double(get8(at + 2)),
                                        __longlong_as_double(get8(at + 4))}, c);
                }
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) add_sums(s, shuffled(s, o), c);
            }
            if (TOP) {
                likeliest.init(room[wave]);
                for (int g = wave; g < a.segments; g += NW) {
                    const uint32_t at = (uint32_t)(row * a.segments + g) * slot + kSlotHead;
                    likeliest.merge(63 - lane < a.top ? get8(at + 2 * (63 - lane)) : 0, a.top);
                }
                if (NW > 1) {
                    room[wave][63 - lane] = likeliest.list;
                    __syncthreads();
                    if (wave == 0)
#pragma unroll
                        for (int w = 1; w < NW; ++w) likeliest.merge(room[w][lane], a.top);
                }
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
        if (NW > 1) __syncthreads();  // the LDS is the next unit's
    }
}

template <typename T, int NW>
static void launch_waves(const char* name, const LogprobArgs& a) {
    const int64_t units = a.rows * a.segments, most = (int64_t)cu_count() * 64;
    const dim3 grid((unsigned)(units < most ? units : most));
    if (a.top > 0)
        launch(name, logprobs_k<T, NW, true>, grid, dim3(64 * NW), 0, a);
    else
        launch(name, logprobs_k<T, NW, false>, grid, dim3(64 * NW), 0, a);
}

// A wave to a row of up to 2048 values, else four
template <typename T>
static void launch_logprobs(const char* name, const LogprobArgs& a) {
    if (a.vocab <= 2048) return launch_waves<T, 1>(name, a);
    launch_waves<T, 4>(name, a);
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
    const double n = (double)a.rows * (double)a.vocab;
    set_work(6.0 * n, n * activation_bytes(logits) + 8.0 * (double)a.rows * (1 + a.top));
    // Segments of 4096 values or more, up to 6 workgroups a CU of them
    const int64_t room = 6 * (int64_t)cu_count(), longest = a.vocab / 4096;
    a.segments = (int)(a.rows >= room ? 1 : room / a.rows < longest ? room / a.rows : longest);
    if (a.segments < 1) a.segments = 1;
    if (a.segments > 1) {
        const size_t bytes = (size_t)a.rows * a.segments * slot_floats(a.top) * sizeof(float);
        a.part = workspace(bytes);
        a.counters = tile_counters((size_t)a.rows);
        if (!a.part || !a.counters) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes of partial sums", bytes);
    }
    if (logits->dtype == NNC_DTYPE_FLOAT16)
        launch_logprobs<half_t>(name, a);
    else
        launch_logprobs<float>(name, a);
}

}  // extern "C"
