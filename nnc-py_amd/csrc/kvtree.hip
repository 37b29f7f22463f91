// Attention of drafted tokens over the paged 8-bit cache
// (nnc_hip_kv_tree_attention). No reference counterpart.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j
//   j < first, or j = first + m for the rows m that row i's mask names
//
// with first the position of the sequence's first new row: a tree of drafts,
// whose branches do not see each other, behind a common context. Scores, weights
// and sums as in kvattention.hip, a lane having the scores of 16 consecutive
// keys for a query row.
//
// Drafts are many rows for one cached head - tokens times the heads of a group -
// but not enough to hide that the cache has to be read, and the keys are many.
// So a wave takes 16 or 32 query rows with 64 keys at a time: a key's whole
// numbers are made f16 in registers, once for all of them, and the four waves of
// a workgroup need no barrier until their rows are joined. The keys of all
// sequences and heads, in units of 64 for each wave, are one line that is cut
// into a run for each workgroup that the CUs hold, so that ragged lengths leave
// none idle: what a run has of a sequence that others share is stored, and the
// last to arrive joins the shares in their order.
//
// Few rows are bound by the cache's bytes: 32 sequences of 4 behind 4096, 32
// heads over 8 of 128 in f16, 52 us, 5.1 TB/s, the rate of a copy. More by what
// passes L2, as each 32 rows of a head read the keys for themselves: 32 sequences of
// 16 behind up to 8192 77 us, 344 MB at 4.8 TB/s, of which the keys are 207, with the
// vector units, which widen the keys and make masks, maxima and exponentials, 49%
// busy (kvtree_rows.hip has the kernel for the longest lines of them).
#include "kvtree.h"

namespace nnc {

// NB blocks of 16 query rows of a tile of R against a share's keys: to the
// output if the share is whole, else to its place.
template <typename T, int D, int R, int NB, int NW>
__device__ __forceinline__ void tree_share(const TreeArgs& a, const TreeShare& w, int place, float* lds) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int STRIDE = 64 * NW, STEPS = D / 32, PIECES = F32 ? 2 : 1, KV = D / 16;
    f16x8* qs = reinterpret_cast<f16x8*>(lds);                    // [NB][STEPS][PIECES][lane]
    int* rows = reinterpret_cast<int*>(lds + R * D / 2 * PIECES);  // [R]: row of the activations, -1: none
    int* lows = rows + R;                                          // [R]: the last position that a window hides
    int* ups = lows + R;                                           // [R]: the power of two that the row's pieces are scaled by
    float* ml = reinterpret_cast<float*>(ups + R);                 // [3][NW][R]
    float* os = ml + 3 * NW * R;                                   // [NW / 2][R][D + 4]
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Span& span = w.span;
    const int first = span.first();
    const int64_t all = (int64_t)span.rows * a.group;
    const int to = min(span.length, w.lo + (w.unit + w.n) * STRIDE);

    const int page = a.g.page, page16 = page / 16, wide = a.g.width - 1;
    const int64_t plane = (int64_t)page * D, page_bytes = (int64_t)a.kv_heads * plane;
    const int* table = a.g.table + (int64_t)w.b * a.g.width;
    const int8_t* kbase = a.k + (int64_t)w.head_kv * plane + (int64_t)(i & 3) * D + g * (D / 4);
    const int8_t* vbase = a.v + (int64_t)w.head_kv * plane + i * page;
    int kid, vid;
    auto find = [&](int tb) {
        kid = table[min((int)slot_of(tb / 16 + (i >> 2), a.slot_magic), wide)];
        vid = table[min((int)slot_of(tb / 16 + g, a.slot_magic), wide)];
    };
    ix2 kb[4][D / 32];
    ix4 vb[KV];
    float ks, vs;
    bool have;
    auto load_k = [&](int tb) {
        const int t16 = tb / 16 + (i >> 2), off = (t16 - (int)slot_of(t16, a.slot_magic) * page16) * 16;
        const int64_t pn = kid >= 0 && kid < a.g.pages && t16 * 16 < to ? kid : 0;
        const int8_t* p = kbase + pn * page_bytes + off * D;
#pragma unroll
        for (int bl = 0; bl < 4; ++bl)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) kb[bl][c] = *reinterpret_cast<const ix2*>(p + bl * 4 * D + 8 * c);
    };
    auto load_v = [&](int tb) {
        const int t16 = tb / 16 + g, off = (t16 - (int)slot_of(t16, a.slot_magic) * page16) * 16;
        have = vid >= 0 && vid < a.g.pages && t16 * 16 < to;
        const int64_t pn = have ? vid : 0;
        const int8_t* p = vbase + pn * page_bytes + off;
#pragma unroll
        for (int c = 0; c < KV; ++c) vb[c] = *reinterpret_cast<const ix4*>(p + c * 16 * page);
        ks = a.k_scale[pn * a.kv_heads + w.head_kv];
        vs = a.v_scale[pn * a.kv_heads + w.head_kv];
    };
    int tb = w.lo + w.unit * STRIDE + 64 * wave;
    if (tb < to) find(tb);

    // the query rows' dims g * D / 4 .. + D / 4, by a wave for each block
    constexpr int QV = 16 / (int)sizeof(T);
    for (int rb = wave; rb < NB; rb += NW) {
        const int64_t fr = (int64_t)w.tile * R + 16 * rb + i;
        const bool ok = fr < all;
        const int tok = (int)((ok ? fr : 0) / a.group), gh = (int)((ok ? fr : 0) - (int64_t)tok * a.group);
        const int row = span.end - span.rows + tok;
        T qx[D / 4];
        const T* qp = (const T*)a.q + (int64_t)row * a.ld + a.q_col + (w.head_kv * a.group + gh) * D + g * (D / 4);
        if (a.q_vec) {
#pragma unroll
            for (int d = 0; d < D / 4; d += QV) *reinterpret_cast<ix4*>(qx + d) = *reinterpret_cast<const ix4*>(qp + d);
        } else {
#pragma unroll
            for (int d = 0; d < D / 4; ++d) qx[d] = qp[d];
        }
        int e = 0;
        if (F32) {
            // the row's largest value to [2^13, 2^14)
            float top = 0.f;
#pragma unroll
            for (int d = 0; d < D / 4; ++d) top = fmaxf(top, fabsf((float)qx[d]));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            (void)frexpf(top, &e);
            e = top > 0.f && top < INFINITY ? 14 - e : 0;
        }
        if (g == 0) {
            rows[16 * rb + i] = ok ? row : -1;
            ups[16 * rb + i] = e;
            lows[16 * rb + i] = a.window > 0 ? first + tree_depth(a.tree + (int64_t)row * a.words, a.words, span.rows) - 1 - a.window : INT_MIN;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            f16x8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = F32 ? ldexpf((float)qx[8 * s + j], e) : (float)qx[8 * s + j];
                hi[j] = (half_t)y;
                lo[j] = (half_t)(y - (float)hi[j]);
            }
            qs[((rb * STEPS + s) * PIECES) * 64 + lane] = hi;
            if (F32) qs[((rb * STEPS + s) * PIECES + 1) * 64 + lane] = lo;
        }
    }
    if (tb < to) {
        load_k(tb);
        load_v(tb);
        find(tb + STRIDE);
    }
    __syncthreads();
    float m[NB], l[NB], ex[NB];  // m and ex the row's, l the lane's
    fx4 o[NB][KV];
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) {
        m[rb] = kNone, l[rb] = 0.f, ex[rb] = kUnseen;
#pragma unroll
        for (int c = 0; c < KV; ++c) o[rb][c] = fx4{0.f, 0.f, 0.f, 0.f};
    }

    for (; tb < to; tb += STRIDE) {
        // scores of keys tb + 16 g + 4 b + r
        fx4 x[NB][4];
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            f16x8 qf[NB][PIECES];
#pragma unroll
            for (int rb = 0; rb < NB; ++rb)
#pragma unroll
                for (int pc = 0; pc < PIECES; ++pc) qf[rb][pc] = qs[((rb * STEPS + st) * PIECES + pc) * 64 + lane];
#pragma unroll
            for (int bl = 0; bl < 4; ++bl) {
                const f16x8 kf = widen8((uint32_t)kb[bl][st][0], (uint32_t)kb[bl][st][1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc)
#pragma unroll
                    for (int rb = 0; rb < NB; ++rb)
                        x[rb][bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rb][pc], st == 0 && pc == PIECES - 1 ? fx4{} : x[rb][bl], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(tb + STRIDE);
        __builtin_amdgcn_sched_barrier(0);
        const float u = ks * a.scale, log_v = scale_log(vs), inv_v = 1.0f / vs;
        const bool clear = tb + 64 <= first && a.window <= 0 && __all(have);
        float ku[NB], lv[NB], iv[NB], top[NB], mx[NB], factor[NB];
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            ku[rb] = F32 ? ldexpf(u, -ups[16 * rb + i]) : u, lv[rb] = log_v, iv[rb] = inv_v;
            ku[rb] = ku[rb] == 0.f ? 0x1p-126f : ku[rb];  // for the product with -inf
        }
        if (!clear) {
#pragma unroll
            for (int rb = 0; rb < NB; ++rb) {
                const int j = tb + 16 * g, row = rows[16 * rb + i];
                uint32_t bits = have && row >= 0 ? tree_bits(a.tree + (int64_t)row * a.words, a.words, first, span.length, j) : 0u;
                if (a.window > 0) {  // of the context, up to low
                    const int n = min(min(lows[16 * rb + i] + 1, first) - j, 16);
                    if (n > 0) bits &= 0xffffffffu << n;
                }
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float y = x[rb][c / 4][c % 4];
                    x[rb][c / 4][c % 4] = bits >> c & 1 ? y : -INFINITY;
                }
                // a row that sees none of the 16: their scales are not its own
                if (!bits) ku[rb] = 1.f, lv[rb] = 0.f, iv[rb] = 0.f;
            }
        }
        bool move = false;
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            top[rb] = -INFINITY;
#pragma unroll
            for (int c = 0; c < 16; ++c) top[rb] = fmaxf(top[rb], x[rb][c / 4][c % 4]);
            mx[rb] = fmaf(top[rb], ku[rb], lv[rb]);
        }
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) mx[rb] = fmaxf(mx[rb], __shfl_xor(mx[rb], 16));
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            mx[rb] = fmaxf(mx[rb], __shfl_xor(mx[rb], 32));
            factor[rb] = ldexpf(iv[rb], (int)ex[rb]);
            move |= mx[rb] > m[rb] + kSlack || factor[rb] > kMostFactor;
        }
        if (__any(move)) {
#pragma unroll
            for (int rb = 0; rb < NB; ++rb) {
                const float mn = fmaxf(m[rb], mx[rb]), alpha = __builtin_amdgcn_exp2f(m[rb] - mn);
                float far = fmaxf(reference(m[rb], ex[rb]), top[rb] * ku[rb]);
                far = fmaxf(far, __shfl_xor(far, 16));
                far = fmaxf(far, __shfl_xor(far, 32));
                const float en = exponent(mn, far);
                l[rb] *= rescale(m[rb], ex[rb], mn, en);
                m[rb] = mn, ex[rb] = en;
#pragma unroll
                for (int c = 0; c < KV; ++c) o[rb][c] *= alpha;
                factor[rb] = ldexpf(iv[rb], (int)en);
                if (__any(factor[rb] > kMostFactor)) {
                    const float base = reference(m[rb], en);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float y = x[rb][c / 4][c % 4];
                        l[rb] += __builtin_amdgcn_exp2f(fmaf(y, ku[rb], -base));
                    }
                    factor[rb] = 0.f;
                }
            }
        }
        f16x8 pf[NB][PIECES][2];
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            const float shift = lv[rb] - (m[rb] - kPLog);
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float s0 = x[rb][2 * n + j / 4][j % 4], s1 = x[rb][2 * n + j / 4][j % 4 + 1];
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s0, ku[rb], shift)), p1 = __builtin_amdgcn_exp2f(fmaf(s1, ku[rb], shift));
                    sum += p0;
                    sum += p1;
                    const f16x2 hi = __builtin_convertvector((fx2{p0, p1}), f16x2);
                    pf[rb][0][n][j] = hi[0], pf[rb][0][n][j + 1] = hi[1];
                    if (F32) {
                        const f16x2 lo = __builtin_convertvector((fx2{p0 - (float)hi[0], p1 - (float)hi[1]}), f16x2);
                        pf[rb][PIECES - 1][n][j] = lo[0], pf[rb][PIECES - 1][n][j + 1] = lo[1];
                    }
                }
            l[rb] = fmaf(sum, factor[rb], l[rb]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int c = 0; c < KV; ++c) {
                const f16x8 vf = widen8((uint32_t)vb[c][2 * n], (uint32_t)vb[c][2 * n + 1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc)
#pragma unroll
                    for (int rb = 0; rb < NB; ++rb) o[rb][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rb][pc][n], o[rb][c], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        load_v(tb + STRIDE);
        find(tb + 2 * STRIDE);
    }

    // join the waves: each row's maximum, divisor and exponent, then the upper
    // half of the waves hands its sums to the lower, until one has all
    float inv[NB];
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) {
        l[rb] += __shfl_xor(l[rb], 16);
        l[rb] += __shfl_xor(l[rb], 32);
        if (g == 0) {
            float* mine = ml + wave * R + 16 * rb + i;
            mine[0] = m[rb], mine[NW * R] = l[rb], mine[2 * NW * R] = ex[rb];
        }
    }
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) {
        const float* r = ml + 16 * rb + i;
        float top = kNone, far = kNone, sum = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) top = fmaxf(top, r[v * R]), far = fmaxf(far, reference(r[v * R], r[(2 * NW + v) * R]));
        ex[rb] = exponent(top, far);
#pragma unroll
        for (int v = 0; v < NW; ++v) sum += r[(NW + v) * R] * rescale(r[v * R], r[(2 * NW + v) * R], top, ex[rb]);
        const float f = __builtin_amdgcn_exp2f(m[rb] - top);
#pragma unroll
        for (int c = 0; c < KV; ++c) o[rb][c] *= f;
        m[rb] = top, l[rb] = sum;
        inv[rb] = sum == 0.f ? 0.f : 1.0f / sum;
    }
#pragma unroll
    for (int n = NW / 2; n > 0; n /= 2) {
        if (wave >= n && wave < 2 * n)
#pragma unroll
            for (int rb = 0; rb < NB; ++rb)
#pragma unroll
                for (int c = 0; c < KV; ++c) *reinterpret_cast<fx4*>(os + ((wave - n) * R + 16 * rb + i) * (D + 4) + 16 * c + 4 * g) = o[rb][c];
        __syncthreads();
        if (wave < n)
#pragma unroll
            for (int rb = 0; rb < NB; ++rb)
#pragma unroll
                for (int c = 0; c < KV; ++c) o[rb][c] += *reinterpret_cast<const fx4*>(os + (wave * R + 16 * rb + i) * (D + 4) + 16 * c + 4 * g);
        __syncthreads();
    }
    if (wave > 0) return;
    const TreePlaces<D, R> places(a);
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) {
        const int row = rows[16 * rb + i];
        if (row < 0) continue;
        if (w.whole) {
            const int tok = row - (span.end - span.rows), gh = (int)((int64_t)w.tile * R + 16 * rb + i - (int64_t)tok * a.group);
            T* op = (T*)a.out + ((int64_t)row * a.heads + w.head_kv * a.group + gh) * D + 4 * g;
#pragma unroll
            for (int c = 0; c < KV; ++c) {
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = (T)ldexpf(o[rb][c][r] * inv[rb], (int)ex[rb]);
                __builtin_memcpy(__builtin_assume_aligned(op + 16 * c, 4 * sizeof(T)), v, sizeof v);
            }
        } else {
#pragma unroll
            for (int c = 0; c < KV; ++c) {
                const float p = o[rb][c][0], q = o[rb][c][1], r = o[rb][c][2], s = o[rb][c][3];
                places.put4(place, 16 * rb + i, 16 * c + 4 * g, p, q, r, s);
            }
            if (g == 0) places.put4(place, 16 * rb + i, D, m[rb], l[rb], ex[rb], 0.f);
        }
    }
}

template <typename T, int D, int RB, int NW, int OCC>
__global__ void __launch_bounds__(64 * NW, OCC) kv_tree_k(TreeArgs a) {
    constexpr int STRIDE = 64 * NW, R = 16 * RB;
    extern __shared__ __align__(16) float tree_lds[];
    walk_run<R, STRIDE, kShortKeys / STRIDE>(
        a,
        [&](const TreeShare& w, int place) {
            if (RB > 1 && w.rows > 16)
                tree_share<T, D, R, RB, NW>(a, w, place, tree_lds);
            else
                tree_share<T, D, R, 1, NW>(a, w, place, tree_lds);
        },
        [&](const TreeShare& w, int64_t tile, int shares, auto place) {
            if (!finish_arrive(a.counters + w.head_kv * a.tiles + tile, shares - 1)) return;
            join_shares<T, D, R, R, 64 * NW>(TreePlaces<D, R>(a), 0, w.rows, shares, place, [&](int r) { return tree_row<T, D, R>(a, w, r); }, tree_lds);
        });
}

template <typename T, int D, int RB, int NW>
constexpr int tree_lds_bytes() {
    constexpr int share = 4 * 16 * RB * (D / 2 * (sizeof(T) == 4 ? 2 : 1) + 3 + 3 * NW + NW / 2 * (D + 4)), join = 4 * (16 * RB * (3 * kJoin + 2) + kJoin);
    return share > join ? share : join;
}

template <typename T, int D, int RB, int NW, int OCC>
static void launch_blocks(const char* name, TreeArgs& a, int64_t rows) {
    auto kernel = kv_tree_k<T, D, RB, NW, OCC>;
    constexpr int lds = tree_lds_bytes<T, D, RB, NW>();
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    // (whole items on 16 rows, two workgroups a CU: 64 trees of 4 behind up to 1024 30 -> 26 us, 256 of 2 behind up to
    // 500 87 -> 62)
    a.runs = cu_count() * (OCC > 1 || (RB == 1 && D <= 128 && a.least == 1) ? 2 : 1);
    if (!tree_scratch(name, a, rows, 16 * RB, D)) return;
    a.counters = tile_counters((size_t)(a.tiles * a.kv_heads));
    if (!a.counters) return fail(NNC_HIP_ENOMEM, name, "no workspace for counters");
    launch(name, kernel, dim3((unsigned)a.runs), dim3(64 * NW), lds, a);
}

// Query rows of a tile: 16 while a sequence has no more for a cached head; 32 with
// the registers of a SIMD for one wave while it has no more, else for two, of
// which one has its exponentials while the other has its products. 32 rows, one
// and two waves, us, of 32 heads over 8 of 128: 32 sequences of 8 behind 4096 56 and
// 67, of 16 behind up to 8192 101 and 77, one of 64 behind 65536 147 and 122. (64
// rows, whose sums leave no second wave: 93 and 148 for the last two.) Of dim 256,
// 16 heads over 4, 16 rows and 32, us: 8 sequences of 16 behind 4096 40 and 44, of
// 8 30 and 41, one of 64 behind 16384 61 and 60: 16 there.
template <typename T, int D>
static void launch_tree(const char* name, TreeArgs& a, int64_t rows, int64_t each) {
    if constexpr (D <= 128) {
        if (each > 32) return launch_blocks<T, D, 2, 4, 2>(name, a, rows);
        if (each > 16) return launch_blocks<T, D, 2, 4, 1>(name, a, rows);
    }
    launch_blocks<T, D, 1, 4, 1>(name, a, rows);
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_kv_tree_attention(Tensor* q, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                               Tensor* starts, Tensor* lengths, Tensor* tree, Tensor* out, int q_col, int heads, float scale,
                               int window, int max_length) {
    const char* name = "nnc_hip_kv_tree_attention";
    CacheArgs c;
    int64_t rows = 0, ld = 0;
    if (!cache_args(name, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, 0, &c)) return;
    if (heads < 1 || heads % c.kv_heads != 0 || heads > 65535)
        return fail(NNC_HIP_EINVAL, name, "%d heads over %d cached ones", heads, c.kv_heads);
    const int64_t width = (int64_t)heads * c.dim;
    if (!rows_arg(name, "q", q, q_col, width, &rows, &ld)) return;
    if (!has_data(tree) || !good_shape(tree) || tree->ndim != 2 || tree->shape[0] != rows || tree->shape[1] < 1)
        return fail(NNC_HIP_EINVAL, name, "tree must be [rows][words]");
    if (tree->dtype != NNC_DTYPE_INT32) return fail(NNC_HIP_EUNSUPP, name, "an int32 tree only");
    if (!has_data(out) || !good_shape(out) || out->dtype != q->dtype || numel(out) != rows * width ||
        out->shape[out->ndim - 1] != width)
        return fail(NNC_HIP_EINVAL, name, "out must be [rows][heads * dim] of q's type");
    if (window < 0 || max_length < 0) return fail(NNC_HIP_EINVAL, name, "negative window or max_length");
    if (!(scale > 0.f) || !(scale < INFINITY)) return fail(NNC_HIP_EINVAL, name, "scale must be positive");
    if (!aligned16(out->data)) return fail(NNC_HIP_EUNSUPP, name, "out must be 16-byte aligned");
    if (tree->shape[1] > INT32_MAX / 32) return fail(NNC_HIP_EUNSUPP, name, "masks of %lld words", (long long)tree->shape[1]);
    if (rows == 0 || c.ragged.batch == 0) return;
    const int group = heads / c.kv_heads;
    if (rows * group > (1 << 27) || rows > UINT32_MAX / 256)
        return fail(NNC_HIP_EUNSUPP, name, "%lld rows of %d heads", (long long)rows, heads);
    if (!ready(name)) return;
    const int capacity = c.ragged.width * c.page;
    const int longest = max_length > 0 && max_length < capacity ? max_length : capacity, seen = window_of(window, capacity);
    const int64_t holders = rows < c.ragged.batch ? rows : c.ragged.batch, each = ceil_div(rows * group, holders);
    const int64_t reach = tree_reach(seen, ceil_div(rows, holders), longest);
    TreeArgs a{c.ragged, c.k, c.v, c.k_scale, c.v_scale, (const int*)tree->data, q->data, out->data, nullptr, nullptr, ld, 0, q_col, heads,
               c.kv_heads, group, seen, (int)tree->shape[1], reach <= kShortKeys ? 1 : 2, 0, slot_magic(c.page / 16),
               aligned16(q->data) && ld * activation_bytes(q) % 16 == 0 && q_col * activation_bytes(q) % 16 == 0,
               scale * 1.44269504088896340736f};
    a.g.rows = (int)rows;
    const int64_t once = seen > 0 ? (int64_t)seen - 1 + ceil_div(rows, holders) : longest;  // the keys of a sequence that a row sees
    set_work(0.0, 2.0 * c.kv_heads * c.dim * (double)(once < longest ? once : longest) * c.ragged.batch);
    const bool f16 = q->dtype == NNC_DTYPE_FLOAT16;
    if (launch_tree_rows(name, f16, c.dim, a, rows, each, reach)) return;
    switch (c.dim) {
        case 32: return f16 ? launch_tree<half_t, 32>(name, a, rows, each) : launch_tree<float, 32>(name, a, rows, each);
        case 64: return f16 ? launch_tree<half_t, 64>(name, a, rows, each) : launch_tree<float, 64>(name, a, rows, each);
        case 128: return f16 ? launch_tree<half_t, 128>(name, a, rows, each) : launch_tree<float, 128>(name, a, rows, each);
        default: return f16 ? launch_tree<half_t, 256>(name, a, rows, each) : launch_tree<float, 256>(name, a, rows, each);
    }
}

}  // extern "C"
