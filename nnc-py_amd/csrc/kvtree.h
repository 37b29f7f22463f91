// What the kernels of nnc_hip_kv_tree_attention share (kvtree.hip,
// kvtree_rows.hip): how the keys of all sequences and heads are cut into runs, and
// how the shares of a tile are joined.
#pragma once

#include <limits.h>

#include "kvattn.h"
#include "lanes.h"

namespace nnc {

struct TreeArgs {
    Ragged g;
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    const int* tree;  // [rows][words]
    const void* q;
    void* out;
    float* part;    // [run][2][row of the tile][dim + 4]: sums, m, l, e
    int* counters;  // [cached head][tile], zero
    int64_t ld;
    int64_t tiles;  // for each cached head, at most
    int q_col, heads, kv_heads, group, window, words, least;
    int runs;       // workgroups, at most
    uint32_t slot_magic;
    bool q_vec;   // query rows start on 16 bytes
    float scale;  // with log2(e)
};

// The keys that rows of a sequence see, [lo, hi), and the tiles and units that
// they make for each cached head.
struct TreeSpan {
    Span span;
    int lo, tiles, units;
    __device__ __forceinline__ void set(const TreeArgs& a, int tile, int stride) {
        tiles = query_tiles(span, a.group, tile);
        lo = tree_low(span.first(), a.window);
        units = max(1, (span.length - lo + stride - 1) / stride);
    }
};

// Unit u of one cached head's: its sequence and tile, its place among the tile's
// units, and the tiles of the sequences before.
struct TreePlace {
    TreeSpan s;
    int b, tile, unit;
    int64_t tiles;
};

// The units of one cached head, found by 64 sequences at a time. The first 64
// stay in registers, a sequence a lane.
template <int TILE, int STRIDE>
struct TreeIndex {
    const TreeArgs& a;
    TreeSpan mine;       // the lane's sequence
    int tiles, upto_t;   // its tiles, with those of the lanes before
    int64_t upto;        // units likewise
    __device__ __forceinline__ void load(int base, int64_t tiles_before) {
        const int lane = threadIdx.x & 63;
        mine = TreeSpan{};
        tiles = 0;
        if (base + lane < a.g.batch) {
            mine.span = span_of(a.g, base + lane);
            mine.set(a, TILE, STRIDE);
            tiles = mine.tiles;
        }
        // (starts that decrease would make more tiles than there are counters for)
        upto_t = sum_before(tiles);
        const int64_t room = a.tiles - tiles_before - (upto_t - tiles);
        if (room < tiles) tiles = room > 0 ? (int)room : 0;
        upto = (int64_t)sum_before((u64)tiles * (u64)mine.units);
    }
    __device__ __forceinline__ explicit TreeIndex(const TreeArgs& args) : a(args) { load(0, 0); }
    __device__ __forceinline__ int64_t total() {
        int64_t units = 0, before = 0;
        for (int base = 0;;) {
            units += last(upto), before += last(upto_t);
            base += 64;
            if (base >= a.g.batch || before >= a.tiles) break;
            load(base, before);
        }
        if (a.g.batch > 64) load(0, 0);
        return units;
    }
    __device__ __forceinline__ static int64_t last(int64_t x) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, 63));
    }
    __device__ __forceinline__ static int last(int x) { return __builtin_amdgcn_readlane(x, 63); }
    // u below total()
    __device__ __forceinline__ TreePlace find(int64_t u) {
        TreePlace p;
        p.tiles = 0;
        bool moved = false;
        for (int base = 0;; base += 64, moved = true) {
            if (base > 0) load(base, p.tiles);
            const uint64_t past = __ballot(upto > u);
            if (past || base + 64 >= a.g.batch) {
                const int at = past ? __ffsll((unsigned long long)past) - 1 : 63;
                auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
                p.b = base + at;
                p.s.span.end = of(mine.span.end), p.s.span.length = of(mine.span.length), p.s.span.rows = of(mine.span.rows);
                p.s.lo = of(mine.lo), p.s.tiles = of(tiles), p.s.units = of(mine.units);
                const int64_t whole = (int64_t)((uint64_t)(uint32_t)of((int)(upto >> 32)) << 32 | (uint32_t)of((int)upto));
                u -= whole - (int64_t)p.s.tiles * p.s.units;
                p.tiles += of(upto_t) - of(mine.tiles);
                break;
            }
            u -= last(upto), p.tiles += last(upto_t);
        }
        if (moved) load(0, 0);
        if (u < p.s.units) {
            p.tile = 0, p.unit = (int)u;
        } else {
            p.tile = (int)(u / p.s.units), p.unit = (int)(u - (int64_t)p.tile * p.s.units);
        }
        return p;
    }
    // The sequence that has tile t, and the units before the tile; none: b -1
    __device__ __forceinline__ TreePlace find_tile(int64_t t, int64_t& before) {
        TreePlace p;
        p.b = -1, p.tiles = 0, p.unit = 0, before = 0;
        for (int base = 0;; base += 64) {
            if (base > 0) load(base, p.tiles);
            const uint64_t past = __ballot(p.tiles + upto_t > t);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
                p.b = base + at;
                p.s.span.end = of(mine.span.end), p.s.span.length = of(mine.span.length), p.s.span.rows = of(mine.span.rows);
                p.s.lo = of(mine.lo), p.s.tiles = of(tiles), p.s.units = of(mine.units);
                p.tiles += of(upto_t) - of(mine.tiles);
                p.tile = (int)(t - p.tiles);
                if (p.tile >= p.s.tiles) p.b = -1;
                const int64_t whole = (int64_t)((uint64_t)(uint32_t)of((int)(upto >> 32)) << 32 | (uint32_t)of((int)upto));
                before += whole - (int64_t)(p.s.tiles - p.tile) * p.s.units;
                return p;
            }
            if (base + 64 >= a.g.batch) return p;
            before += last(upto), p.tiles += last(upto_t);
        }
    }
};

// Runs that so many units are cut into: of `least` units or more.
__device__ __forceinline__ int tree_runs(const TreeArgs& a, int64_t total) {
    const int64_t useful = (total + a.least - 1) / a.least;
    return __builtin_amdgcn_readfirstlane((int)(useful < a.runs ? useful : a.runs));
}

// Tiles whose keys a workgroup goes through in less time than storing and joining
// two shares takes are left whole: up to so many keys.
static constexpr int kShortKeys = 1024;

// A run's share of an item: units [unit, unit + n) of a tile and cached head.
struct TreeShare {
    Span span;
    int b, tile, head_kv, lo, unit, n, rows;  // rows: of the tile
    bool whole;
};

template <int D, int R>
struct TreePlaces {
    static constexpr int ROW = D + 4;
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ explicit TreePlaces(const TreeArgs& a) : r(make_rsrc(a.part)) {}
    __device__ __forceinline__ uint32_t at(int place, int row, int col) const { return (uint32_t)((place * R + row) * ROW + col) * 4u; }
    __device__ __forceinline__ void put4(int place, int row, int col, float x, float y, float z, float w) const {
        typedef unsigned ux4 __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b128(ux4{__float_as_uint(x), __float_as_uint(y), __float_as_uint(z), __float_as_uint(w)}, r,
                                               (int)at(place, row, col), 0, kDeviceScope);
    }
};

// The shares of an item, `rows` (1 .. R) of its rows from row0 on: kJoin shares at
// a time, each row's maxima and divisors first, then 4 dims of a row a
// thread. place(s) is where share s is; out(row) the row's output.
static constexpr int kJoin = 32;
template <typename T, int D, int TILE, int R, int THREADS, class Place, class Out>
__device__ __forceinline__ void join_shares(const TreePlaces<D, TILE>& from, int row0, int rows, int shares, Place place, Out out, float* lds) {
    constexpr int QUADS = D / 4, PER = (R * QUADS + THREADS - 1) / THREADS, AHEAD = 8;
    static_assert(R <= THREADS && kJoin <= THREADS, "a thread each");
    float (*ms)[R] = reinterpret_cast<float (*)[R]>(lds);             // [kJoin][R]
    float (*ls)[R] = reinterpret_cast<float (*)[R]>(lds + kJoin * R), (*es)[R] = reinterpret_cast<float (*)[R]>(lds + 2 * kJoin * R);
    float* scale = lds + 3 * kJoin * R;  // [R]
    float* exps = scale + R;             // [R]
    int* places = reinterpret_cast<int*>(exps + R);  // [kJoin]
    const int tid = threadIdx.x;
    auto row_of = [&](int q) { return min((tid + THREADS * q) / QUADS, R - 1); };
    float top = kNone, e = kUnseen, sum = 0.f;  // of row tid
    f32x4 o[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) o[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < shares; s0 += kJoin) {
        const int n = min(kJoin, shares - s0);
        __syncthreads();
        if (tid < n) places[tid] = place(s0 + tid);
        __syncthreads();
        for (int k = tid; k < n * R; k += THREADS) {
            const int sh = k / R, row = k % R;
            const f32x4 x = load_partial4(from.r, from.at(places[sh], row0 + min(row, rows - 1), D));
            ms[sh][row] = x[0], ls[sh][row] = x[1], es[sh][row] = x[2];
        }
        __syncthreads();
        if (tid < R) {
            float m = top, far = reference(top, e);
            for (int sh = 0; sh < n; ++sh) m = fmaxf(m, ms[sh][tid]), far = fmaxf(far, reference(ms[sh][tid], es[sh][tid]));
            const float en = exponent(m, far);
            sum *= rescale(top, e, m, en);
            for (int sh = 0; sh < n; ++sh) {
                sum = fmaf(rescale(ms[sh][tid], es[sh][tid], m, en), ls[sh][tid], sum);
                ms[sh][tid] = __builtin_amdgcn_exp2f(ms[sh][tid] - m);
            }
            scale[tid] = __builtin_amdgcn_exp2f(top - m);
            top = m, e = en;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; ++q) o[q] *= scale[row_of(q)];
        for (int t = 0; t < n; t += AHEAD) {
            f32x4 v[AHEAD][PER];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int q = 0; q < PER; ++q)
                    v[u][q] = load_partial4(from.r, from.at(places[min(t + u, n - 1)], row0 + min(row_of(q), rows - 1), (tid + THREADS * q) % QUADS * 4));
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int q = 0; q < PER; ++q) {
                    const float w = t + u < n ? ms[min(t + u, n - 1)][row_of(q)] : 0.f;
                    o[q] += v[u][q] * w;
                }
        }
    }
    __syncthreads();
    if (tid < R) scale[tid] = sum == 0.f ? 0.f : 1.0f / sum, exps[tid] = e;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int row = row_of(q), d = (tid + THREADS * q) % QUADS * 4;
        if (row >= rows || tid + THREADS * q >= R * QUADS) continue;
        T v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float y = o[q][r];
            v[r] = (T)ldexpf(y * scale[row], (int)exps[row]);
        }
        __builtin_memcpy(__builtin_assume_aligned(out(row0 + row) + d, 4 * sizeof(T)), v, sizeof v);
    }
}

// Walks the workgroup's run: share(w, its place) for each range of units of a tile
// and cached head, then, where others have a part of it, cut(w, the tile's number,
// shares, the place of each). Tiles of SHORT units or fewer are left whole.
template <int TILE, int STRIDE, int SHORT, class Share, class Cut>
__device__ __forceinline__ void walk_run(const TreeArgs& a, Share share, Cut cut) {
    TreeIndex<TILE, STRIDE> index(a);
    const int64_t each = index.total(), total = each * a.kv_heads;
    const int runs = tree_runs(a, total);
    if ((int)blockIdx.x >= runs) return;
    const int run = xcd_remap(blockIdx.x, runs);
    auto find = [&](int64_t u, int& head_kv) {
        head_kv = u < each ? 0 : (int)(u / each);
        return index.find(u - head_kv * each);
    };
    // a short item is not cut, but its first run's
    auto begin_of = [&](int r) {
        const int64_t u = run_begin(r, total, runs);
        int head_kv;
        if (u == 0 || u == total) return u;
        const TreePlace p = find(u, head_kv);
        return p.s.units <= SHORT ? u - p.unit : u;
    };
    const int64_t end = begin_of(run + 1);
    for (int64_t at = begin_of(run); at < end;) {
        TreeShare w;
        const TreePlace p = find(at, w.head_kv);
        w.span = p.s.span, w.b = p.b, w.lo = p.s.lo, w.tile = p.tile, w.unit = p.unit;
        w.n = (int)(end - at < p.s.units - w.unit ? end - at : p.s.units - w.unit);
        w.whole = w.n == p.s.units;
        const int64_t left = (int64_t)w.span.rows * a.group - (int64_t)w.tile * TILE;
        w.rows = left < TILE ? (int)left : TILE;
        const int64_t begin = at - w.unit;  // of the item
        share(w, share_place(run, begin, total, runs));
        if (!w.whole) {
            const int run0 = run_of(begin, total, runs), shares = run_of(begin + p.s.units - 1, total, runs) - run0 + 1;
            cut(w, p.tiles + w.tile, shares, [&](int sh) { return share_place(run0 + sh, begin, total, runs); });
        }
        at += w.n;
        __syncthreads();  // the LDS is the next share's
    }
}

// Where row r of a tile goes.
template <typename T, int D, int R>
__device__ __forceinline__ T* tree_row(const TreeArgs& a, const TreeShare& w, int r) {
    const int64_t f = (int64_t)w.tile * R + r;
    const int t = (int)(f / a.group), head = w.head_kv * a.group + (int)(f - (int64_t)t * a.group);
    return (T*)a.out + ((int64_t)(w.span.end - w.span.rows + t) * a.heads + head) * D;
}

// Room for the shares of a.runs runs; false with an error recorded
inline bool tree_scratch(const char* name, TreeArgs& a, int64_t rows, int tile, int dim) {
    a.tiles = query_tiles_bound(rows, a.g.batch, a.group, tile);
    const size_t bytes = (size_t)a.runs * 2 * tile * (dim + 4) * sizeof(float);
    if (a.tiles * a.kv_heads > INT32_MAX) return fail(NNC_HIP_EUNSUPP, name, "%lld rows of %d heads", (long long)rows, a.heads), false;
    a.part = workspace(bytes);
    if (!a.part) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes of partial sums", bytes), false;
    return true;
}

// Many rows of long contexts (kvtree_rows.hip): false if its kernels are not for
// these; reach: the keys of a sequence, at most
bool launch_tree_rows(const char* name, bool f16, int dim, const TreeArgs& a, int64_t rows, int64_t each, int64_t reach);

}  // namespace nnc
