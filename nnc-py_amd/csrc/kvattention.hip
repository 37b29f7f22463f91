// Attention over the paged 8-bit cache (nnc_hip_kv_attention). No reference
// counterpart.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j
//   j <= pos_i, j > pos_i - window;  k_j = K_j u_k(page), v_j = V_j u_v(page)
//
// with K, V whole numbers and one scale for each page and head. One pass over
// the keys: in units of powers of two, s_j = scale log2(e) u_k (q . K_j) and
// x_j = s_j + log2(u_v); m a running maximum of x, p_j = 2^(x_j - m); then
//
//   out = 2^e (sum_j p_j V_j) / l,   l = sum_j 2^(s_j - m + e) = sum_j p_j 2^e / u_v
//
// so that the pages' value scales cost nothing in the second product, and p
// has the size of what it contributes. e is a whole number that keeps l near 1:
// m - e is about the largest s. The factor 2^e / u_v of a page serves as long as
// p did not lose what l needs: where it is over 2^60 (a page of values far below
// another's, or of zeros) l takes its own exponentials.
//
// v_mfma_f32_16x16x32_f16, keys as the first operand's rows and query rows as
// the second's columns (S^T = K Q^T, then O^T = V^T P^T): lane (i = lane % 16,
// g = lane / 16) then holds query row i's scores of keys 4g + r, which is
// the layout in which the second product takes its P operand, without moving
// anything between lanes. A wave takes 64 keys at a time; row i of its block b
// is key 16 (i / 4) + 4b + i % 4, so that lane group g ends up with the 16
// consecutive keys 16g .. 16g + 15: one scale each, and 16 consecutive bytes
// of V. Whole numbers of 8 bits are exact in f16. Query rows are f16 as they
// are; fp32 ones are scaled by a power of two and cut into two f16 pieces (22
// bits), and so is p then. For f16 outputs p is rounded to f16 once, which moves a
// weight by 2^-11 of it at most, as the output's own rounding moves the result.
//
// A workgroup takes 16 query rows - heads of one cached head, then tokens -
// and a share of the keys, its waves 64 keys each in turn; the waves' sums are
// joined through LDS, the shares' through the workspace. The cache's bytes
// bound it: 64 sequences of up to 8192 positions (32 heads over 8 of 128) 105 us,
// 552 MB at 5.2 TB/s, as a large copy (in the batch's own order, whose longest
// ended last, 130); one of 131072 54.6 us, 4.9 TB/s. A short call is a chain of
// dependent loads (lengths, table, page) and joins, 7.4 us for four of 333.
#include <limits.h>

#include "kvattn.h"

namespace nnc {

struct KvAttnArgs {
    Ragged g;
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    const void* q;
    void* out;
    float* part;    // [tile][cached head][split][row of the tile][dim + 4]: sums, m, l, e
    int* counters;  // [tile][cached head], zero
    int64_t ld;
    int q_col, heads, kv_heads, group, window, splits, chunk, tiles;
    uint32_t slot_magic;
    bool q_vec;  // query rows start on 16 bytes
    bool by_length;  // long sequences' workgroups first
    float scale;  // with log2(e)
};

// ---------------------------------------------------------------------------
// Shares of the keys: every workgroup of a tile and head stores its rows' sums,
// maximum and divisor (device scope, mfma_tile.h), and the last to arrive joins
// them in the shares' order and writes the rows. Against a launch of its own
// for that: 4 to 5 us less.
// ---------------------------------------------------------------------------
template <int D>
struct Shares {
    static constexpr int ROW = D + 4;
    __amdgpu_buffer_rsrc_t r;
    int tile;  // rows of a share
    __device__ __forceinline__ Shares(const KvAttnArgs& a, int item, int tile_) : tile(tile_) {
        r = make_rsrc(a.part + (int64_t)item * a.splits * tile_ * ROW);
    }
    __device__ __forceinline__ uint32_t at(int share, int row, int col) const {
        return (uint32_t)((share * tile + row) * ROW + col) * 4u;
    }
    __device__ __forceinline__ void put4(int share, int row, int col, float x, float y, float z, float w) const {
        typedef unsigned ux4 __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b128(ux4{__float_as_uint(x), __float_as_uint(y), __float_as_uint(z), __float_as_uint(w)}, r,
                                               (int)at(share, row, col), 0, kDeviceScope);
    }
    // one wave: row `row` of the tile to `out`
    template <typename T>
    __device__ __forceinline__ void join(int shares, int row, T* out) const {
        constexpr int PER = D >= 64 ? D / 64 : 1;
        const int lane = threadIdx.x & 63, dim = lane % (D / PER) * PER;
        float top = kNone, far = kNone;
        for (int s = lane; s < shares; s += 64) {
            const float m = load_partial(r, at(s, row, D));
            top = fmaxf(top, m);
            far = fmaxf(far, reference(m, load_partial(r, at(s, row, D + 2))));
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o)), far = fmaxf(far, __shfl_xor(far, o));
        const float e = exponent(top, far);
        float sum = 0.f, o[PER];
#pragma unroll
        for (int q = 0; q < PER; ++q) o[q] = 0.f;
        for (int s0 = 0; s0 < shares; s0 += 64) {
            float w = 0.f;
            if (s0 + lane < shares) {
                const float m = load_partial(r, at(s0 + lane, row, D));
                w = __builtin_amdgcn_exp2f(m - top);
                sum = fmaf(rescale(m, load_partial(r, at(s0 + lane, row, D + 2)), top, e), load_partial(r, at(s0 + lane, row, D + 1)), sum);
            }
            const int n = min(64, shares - s0);
            for (int t = 0; t < n; t += 8) {
                float v[8][PER];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const uint32_t from = at(min(s0 + t + u, shares - 1), row, dim);
                    if constexpr (PER == 4) {
                        const f32x4 x = load_partial4(r, from);
                        v[u][0] = x[0], v[u][1] = x[1], v[u][2] = x[2], v[u][3] = x[3];
                    } else {
#pragma unroll
                        for (int q = 0; q < PER; ++q) v[u][q] = load_partial(r, from + 4 * q);
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const float wt = __shfl(w, t + u);  // 0 behind the last share
#pragma unroll
                    for (int q = 0; q < PER; ++q) o[q] = fmaf(v[u][q], wt, o[q]);
                }
            }
        }
        sum = wave_add(sum);
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        if (lane < D / PER) {
#pragma unroll
            for (int q = 0; q < PER; ++q) out[dim + q] = (T)ldexpf(o[q] * inv, (int)e);
        }
    }
};

// Where workgroups come in several rounds, those of long sequences go first, in
// eighths of the longest: the `tile`-th sequence in that order, -1 behind the
// last, -2 if a sequence has more than one tile.
static constexpr int kOrdered = 256;  // sequences
__device__ __forceinline__ int longest_first(const Ragged& g, int group, int tile) {
    const int lane = threadIdx.x & 63, passes = (g.batch + 63) / 64;
    float length[kOrdered / 64], most = 0.f;
    bool one = true;
#pragma unroll
    for (int u = 0; u < kOrdered / 64; ++u) {
        length[u] = -1.f;
        if (u < passes && 64 * u + lane < g.batch) {
            const Span span = span_of(g, 64 * u + lane);
            const int tiles = query_tiles(span, group, 16);
            if (tiles > 0) length[u] = (float)span.length;
            one &= tiles <= 1;
            most = fmaxf(most, length[u]);
        }
    }
    if (!__all(one)) return -2;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
    const float eighths = 8.f / (most + 1.f);
    for (int c = 7; c >= 0; --c)
#pragma unroll
        for (int u = 0; u < kOrdered / 64; ++u) {
            if (u >= passes) continue;
            const uint64_t in = __ballot(length[u] >= 0.f && min((int)(length[u] * eighths), 7) == c);
            const int n = __popcll(in);
            if (tile < n) return 64 * u + __ffsll(__ballot((in >> lane & 1) && __popcll(in & ((1ull << lane) - 1)) == tile)) - 1;
            tile -= n;
        }
    return -1;
}

// most waves of a workgroup for few query rows (dim 256: one wave's registers)
constexpr int token_waves(int dim) { return dim <= 128 ? 8 : 4; }

// (dim 32: four waves a SIMD; three, where the compiler takes a few registers
// more, are 29 us and not 25 for 512 sequences of up to 300, 8 heads, fp32)
template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, D == 32 ? 4 : 1) kv_attention_k(KvAttnArgs a) {
    constexpr int STRIDE = 64 * NW;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int STEPS = D / 32, PIECES = F32 ? 2 : 1, KV = D / 16;  // KV: 16-dim blocks of the output
    __shared__ float ml[3][NW][16];
    __shared__ __align__(16) float os[NW / 2][16][D + 4];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.z;
    int head_kv = blockIdx.y, tile = blockIdx.x, b = -2;
    if (a.by_length) {  // all heads of a sequence, then the next one's
        const int lin = blockIdx.y * a.tiles + blockIdx.x;
        tile = lin / a.kv_heads, head_kv = lin - tile * a.kv_heads;
        b = longest_first(a.g, a.group, tile);
        if (b >= 0) tile = 0;
    }
    if (b == -2) b = find_share(tile, a.g.batch, [&](int s) { return query_tiles(span_of(a.g, s), a.group, 16); });
    if (b < 0) return;
    const Span span = span_of(a.g, b);
    const int64_t all = (int64_t)span.rows * a.group, fr = (int64_t)tile * 16 + i;
    const bool row_ok = fr < all;
    const int tok = (int)((row_ok ? fr : 0) / a.group), gh = (int)((row_ok ? fr : 0) - (int64_t)tok * a.group);
    const int pos = row_ok ? span.first() + tok : -1;
    const int64_t row = span.end - span.rows + tok;
    const int head = head_kv * a.group + gh;
    const int first_pos = span.first() + (int)((int64_t)tile * 16 / a.group);
    const int64_t last = (int64_t)tile * 16 + 15 < all ? (int64_t)tile * 16 + 15 : all - 1;
    const int last_pos = span.first() + (int)(last / a.group);
    const KeyRange range(first_pos, last_pos, a.window, a.splits, a.chunk, STRIDE);
    const int shares = range.shares();
    if (split >= shares) return;
    const int from = range.lo + split * range.chunk;
    const int to = min(range.hi, from + range.chunk);

    // K: the lane's row in the four blocks is in 16-key group i / 4. V: the
    // lane's 16 keys are group g. A chunk's table entries are read one chunk
    // before its keys and values; those into the registers of the chunk before
    // as soon as these are used.
    const int page = a.g.page, page16 = page / 16, wide = a.g.width - 1;
    const int64_t plane = (int64_t)page * D, page_bytes = (int64_t)a.kv_heads * plane;
    const int* table = a.g.table + (int64_t)b * a.g.width;
    const int8_t* kbase = a.k + (int64_t)head_kv * plane + (int64_t)(i & 3) * D + g * (D / 4);
    const int8_t* vbase = a.v + (int64_t)head_kv * plane + i * page;
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
        ks = a.k_scale[pn * a.kv_heads + head_kv];
        vs = a.v_scale[pn * a.kv_heads + head_kv];
    };
    // the query row's dims g * D / 4 .. + D / 4, read before the first keys
    int tb = from + 64 * wave;
    if (tb < to) find(tb);
    constexpr int QV = 16 / (int)sizeof(T);
    T qx[D / 4];
    {
        const T* qp = (const T*)a.q + row * a.ld + a.q_col + head * D + g * (D / 4);
        if (a.q_vec) {
#pragma unroll
            for (int d = 0; d < D / 4; d += QV) *reinterpret_cast<ix4*>(qx + d) = *reinterpret_cast<const ix4*>(qp + d);
        } else {
#pragma unroll
            for (int d = 0; d < D / 4; ++d) qx[d] = qp[d];
        }
    }
    if (tb < to) {
        load_k(tb);
        load_v(tb);
        find(tb + STRIDE);
    }
    f16x8 qf[PIECES][STEPS];
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
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = F32 ? ldexpf((float)qx[8 * s + j], e) : (float)qx[8 * s + j];
            const half_t hi = (half_t)y;
            qf[0][s][j] = hi;
            if (F32) qf[PIECES - 1][s][j] = (half_t)(y - (float)hi);
        }
    float m = kNone, l = 0.f;  // m and ex the row's, l the lane's
    float ex = kUnseen;
    fx4 o[KV];
#pragma unroll
    for (int c = 0; c < KV; ++c) o[c] = fx4{0.f, 0.f, 0.f, 0.f};

    for (; tb < to; tb += STRIDE) {
        // scores of keys tb + 16 g + 4 b + r
        float x[16];
        float top = -INFINITY;
#pragma unroll
        for (int bl = 0; bl < 4; ++bl) {
            fx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const f16x8 kf = widen8((uint32_t)kb[bl][st][0], (uint32_t)kb[bl][st][1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[pc][st], s, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * bl + r] = s[r];
        }
        load_k(tb + STRIDE);
        float ku = F32 ? ldexpf(ks * a.scale, -e) : ks * a.scale, lv = scale_log(vs), iv = 1.0f / vs;
        ku = ku == 0.f ? 0x1p-126f : ku;  // for the product with -inf
        if (!(tb + 63 <= first_pos && (a.window <= 0 || tb > last_pos - a.window) && __all(have))) {
            const int j = tb + 16 * g, low = a.window > 0 ? pos - a.window : INT_MIN, up = have ? pos : INT_MIN;
#pragma unroll
            for (int c = 0; c < 16; ++c) x[c] = j + c <= up && j + c > low ? x[c] : -INFINITY;
            // a row that sees none of the 16: their scales are not its own
            if (!(j <= up && j + 15 > low)) ku = 1.f, lv = 0.f, iv = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) top = fmaxf(top, x[c]);
        float mx = fmaf(top, ku, lv);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        float factor = ldexpf(iv, (int)ex), sum = 0.f;
        if (__any(mx > m + kSlack || factor > kMostFactor)) {
            const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - mn);
            float far = fmaxf(reference(m, ex), top * ku);
            far = fmaxf(far, __shfl_xor(far, 16));
            far = fmaxf(far, __shfl_xor(far, 32));
            const float en = exponent(mn, far);
            l *= rescale(m, ex, mn, en);
            m = mn, ex = en;
#pragma unroll
            for (int c = 0; c < KV; ++c) o[c] *= alpha;
            factor = ldexpf(iv, (int)ex);
            if (__any(factor > kMostFactor)) {
                const float base = reference(m, ex);
#pragma unroll
                for (int c = 0; c < 16; ++c) l += __builtin_amdgcn_exp2f(fmaf(x[c], ku, -base));
                factor = 0.f;
            }
        }
        const float shift = lv - (m - kPLog);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            x[c] = __builtin_amdgcn_exp2f(fmaf(x[c], ku, shift));
            sum += x[c];
        }
        l = fmaf(sum, factor, l);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f16x8 pf[PIECES];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float p0 = x[8 * n + j], p1 = x[8 * n + j + 1];
                const f16x2 hi = __builtin_convertvector((fx2{p0, p1}), f16x2);
                pf[0][j] = hi[0], pf[0][j + 1] = hi[1];
                if (F32) {
                    const f16x2 lo = __builtin_convertvector((fx2{p0 - (float)hi[0], p1 - (float)hi[1]}), f16x2);
                    pf[PIECES - 1][j] = lo[0], pf[PIECES - 1][j + 1] = lo[1];
                }
            }
#pragma unroll
            for (int c = 0; c < KV; ++c) {
                const f16x8 vf = widen8((uint32_t)vb[c][2 * n], (uint32_t)vb[c][2 * n + 1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc) o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[pc], o[c], 0, 0, 0);
            }
        }
        load_v(tb + STRIDE);
        find(tb + 2 * STRIDE);
    }
    // join the waves
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) ml[0][wave][i] = m, ml[1][wave][i] = l, ml[2][wave][i] = ex;
    __syncthreads();
    float top = kNone, far = kNone, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[0][w][i]), far = fmaxf(far, reference(ml[0][w][i], ml[2][w][i]));
    ex = exponent(top, far);
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += ml[1][w][i] * rescale(ml[0][w][i], ml[2][w][i], top, ex);
    const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int c = 0; c < KV; ++c) o[c] *= f;
    // the upper half of the waves hands its sums to the lower, until one has all
#pragma unroll
    for (int n = NW / 2; n > 0; n /= 2) {
        if (wave >= n && wave < 2 * n)
#pragma unroll
            for (int c = 0; c < KV; ++c) *reinterpret_cast<fx4*>(&os[wave - n][i][16 * c + 4 * g]) = o[c];
        __syncthreads();
        if (wave < n)
#pragma unroll
            for (int c = 0; c < KV; ++c) o[c] += *reinterpret_cast<const fx4*>(&os[wave][i][16 * c + 4 * g]);
        if (n > 1) __syncthreads();
    }
    if (shares == 1) {
        if (wave > 0 || !row_ok) return;
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        T* op = (T*)a.out + (row * a.heads + head) * D + 4 * g;
#pragma unroll
        for (int c = 0; c < KV; ++c) {
            T v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (T)ldexpf(o[c][r] * inv, (int)ex);
            __builtin_memcpy(__builtin_assume_aligned(op + 16 * c, 4 * sizeof(T)), v, sizeof v);
        }
        return;
    }
    const int item = blockIdx.x * a.kv_heads + head_kv;
    const Shares<D> part(a, item, 16);
    if (wave == 0 && row_ok) {
#pragma unroll
        for (int c = 0; c < KV; ++c) {
            const float x = o[c][0], y = o[c][1], z = o[c][2], w = o[c][3];
            part.put4(split, i, 16 * c + 4 * g, x, y, z, w);
        }
        if (g == 0) part.put4(split, i, D, top, sum, ex, 0.f);
    }
    if (!finish_arrive(a.counters + item, shares - 1)) return;
    for (int r = wave; r < 16 && (int64_t)tile * 16 + r < all; r += NW) {
        const int64_t f = (int64_t)tile * 16 + r;
        const int t = (int)(f / a.group), hd = head_kv * a.group + (int)(f - (int64_t)t * a.group);
        part.join(shares, r, (T*)a.out + ((int64_t)(span.end - span.rows + t) * a.heads + hd) * D);
    }
}

// ---------------------------------------------------------------------------
// Many query rows (prompts): 32 rows per wave, 4 or 8 waves, the keys 64 at a
// time through LDS, where they are kept as f16: widened once for all waves.
// Two prompts of 2048 rows behind 2048 positions, 32 heads over 8 of 128: 240
// us, 860 TFLOP/s of the 1334 that a large f16 product reaches. The matrix units
// are busy for 40% of the cycles and the vector units, with masks, exponentials
// and conversions, for 59%; the two overlap only in part.
// v_mfma_f32_32x32x16_f16 as above; query row i = lane % 32, lane half h. Row 8q + 4h + u of a block of 32 keys is key 16h + 4q + u: lane half h
// has the scores of 16 consecutive keys, which one page's scales serve.
//
// LDS rows: K's in that order, 2 dim bytes each; V's one per dim, 128 bytes.
// Their 16-byte chunks are permuted so that 16 lanes reading a chunk of 16
// rows hit all 64 banks. Two stages: chunk t + 1 is widened and stored, and
// the loads of t + 2 go out, before t is used, with one barrier for each.
// ---------------------------------------------------------------------------
template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, D <= 128 || NW == 8 ? 2 : 1) kv_prompt_k(KvAttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int STEPS = D / 16, PIECES = F32 ? 2 : 1, DB = D / 32, KRB = 2 * D;
    constexpr int ROWS = 32 * NW, THREADS = 64 * NW, STAGE = 64 * KRB + D * 128, LOADS = (4 * D + THREADS - 1) / THREADS;  // 16-byte pieces per thread and operand
    extern __shared__ __align__(16) char lds[];
    // [stage]: of 4 groups of 16 keys, K's scale, V's scale's logarithm and
    // inverse, 1 if they can be read; then the four last again
    float* units = (float*)(lds + 2 * STAGE);
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // one XCD after the other, so that the tiles of a head share its L2; the
    // tiles with most keys first
    const int lin = xcd_remap(blockIdx.x, a.tiles * a.kv_heads), head_kv = lin / a.tiles;
    int tile = a.tiles - 1 - lin % a.tiles;
    const int b = __builtin_amdgcn_readfirstlane(
        find_share(tile, a.g.batch, [&](int s) { return query_tiles(span_of(a.g, s), a.group, ROWS); }));
    if (b < 0) return;
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Span span = span_of(a.g, b);
    const int64_t all = (int64_t)span.rows * a.group, row0 = (int64_t)tile * ROWS;
    const int64_t last = row0 + ROWS - 1 < all ? row0 + ROWS - 1 : all - 1;
    const int first_pos = span.first() + (int)(row0 / a.group), last_pos = span.first() + (int)(last / a.group);
    const KeyRange range(first_pos, last_pos, a.window, 1, 64, 64);
    const int from = range.lo, to = range.hi;
    const int64_t fr = row0 + 32 * wave + i;
    const bool row_ok = fr < all;
    const int tok = (int)((row_ok ? fr : last) / a.group), gh = (int)((row_ok ? fr : last) - (int64_t)tok * a.group);
    const int posh = span.first() + tok - 16 * h;  // the row's position, against keys numbered without 16 h
    const int row = span.end - span.rows + tok, head = head_kv * a.group + gh;

    // staging: this thread's pieces. The table entries of a chunk are read one
    // chunk before its keys and values, those two before they are used.
    const int page = a.g.page, page16 = page / 16;
    const int64_t plane = (int64_t)page * D, page_bytes = (int64_t)a.kv_heads * plane;
    const int8_t* kbase = a.k + (int64_t)head_kv * plane;
    const int8_t* vbase = a.v + (int64_t)head_kv * plane;
    const int* table = a.g.table + (int64_t)b * a.g.width;
    auto key_group = [&](int p) { return (threadIdx.x + THREADS * p) / D; };  // 16 keys of D / 16 pieces each
    int kid[LOADS], vid;
    auto entry = [&](int t16) { return table[min((int)slot_of(t16, a.slot_magic), a.g.width - 1)]; };
    auto find = [&](int tb) {
#pragma unroll
        for (int p = 0; p < LOADS; ++p) kid[p] = entry(tb / 16 + key_group(p));
        vid = entry(tb / 16 + (threadIdx.x & 3));
    };
    ix4 kr[LOADS], vr[LOADS];
    float su[2];
    bool can_read = false;
    auto load = [&](int tb) {
        const int gv = tb / 16 + (threadIdx.x & 3);
        const bool have = vid >= 0 && vid < a.g.pages && gv * 16 < to;
        const int64_t pv = have ? vid : 0;
        const int offv = (gv - (int)slot_of(gv, a.slot_magic) * page16) * 16;
#pragma unroll
        for (int p = 0; p < LOADS; ++p) {
            const int e = threadIdx.x + THREADS * p;
            if (4 * D < THREADS && e >= 4 * D) break;
            const int gk = tb / 16 + key_group(p), off = (gk - (int)slot_of(gk, a.slot_magic) * page16) * 16;
            const int64_t pk = kid[p] >= 0 && kid[p] < a.g.pages && gk * 16 < to ? kid[p] : 0;
            kr[p] = *reinterpret_cast<const ix4*>(kbase + pk * page_bytes + off * D + e % D * 16);
            vr[p] = *reinterpret_cast<const ix4*>(vbase + pv * page_bytes + (e >> 2) * page + offv);
        }
        if (threadIdx.x < 4) {
            su[0] = a.k_scale[pv * a.kv_heads + head_kv];
            su[1] = a.v_scale[pv * a.kv_heads + head_kv];
            can_read = have;
        }
    };
    // LDS offsets: a chunk's number only changes address bits that an exclusive
    // or reaches, so one base each (with the stage in it) is all that is kept
    const int kt = threadIdx.x % (4 * D) / (D / 16), ktr = (kt & 32) | (kt & 12) << 1 | (kt & 16) >> 2 | (kt & 3);
    const int kput = lds_chunk<KRB>(ktr, threadIdx.x % (D / 16) * 2);
    const int vput = 64 * KRB + lds_chunk<128>(threadIdx.x % (4 * D) >> 2, (threadIdx.x & 3) * 2);
    const int kget = lds_chunk<KRB>(i, h), vget = 64 * KRB + lds_chunk<128>(i, 2 * h);
    auto store = [&](int stage) {
        const int kp = kput + stage * STAGE, vp = vput + stage * STAGE;
#pragma unroll
        for (int p = 0; p < LOADS; ++p) {
            if (4 * D < THREADS && threadIdx.x >= 4 * D) break;
            // THREADS pieces further: 32 keys, or 16 (key 16 is row 4)
            constexpr bool HALF = THREADS * 16 / D == 16;
            const int k0 = HALF ? (kp ^ (p & 1) * 64) + (p & 1) * 4 * KRB + (p >> 1) * 32 * KRB : kp + p * 32 * KRB;
            *reinterpret_cast<f16x8*>(lds + k0) = widen8((uint32_t)kr[p][0], (uint32_t)kr[p][1]);
            *reinterpret_cast<f16x8*>(lds + (k0 ^ 16)) = widen8((uint32_t)kr[p][2], (uint32_t)kr[p][3]);
            *reinterpret_cast<f16x8*>(lds + vp + p * THREADS * 32) = widen8((uint32_t)vr[p][0], (uint32_t)vr[p][1]);
            *reinterpret_cast<f16x8*>(lds + (vp ^ 16) + p * THREADS * 32) = widen8((uint32_t)vr[p][2], (uint32_t)vr[p][3]);
        }
        if (threadIdx.x < 4) {
            const float vu = can_read ? su[1] : 1.f, ok = can_read ? 1.f : 0.f;
            *reinterpret_cast<fx4*>(units + stage * 20 + threadIdx.x * 4) =
                fx4{can_read ? su[0] * a.scale : 0.f, scale_log(vu), 1.0f / vu, ok};
            units[stage * 20 + 16 + threadIdx.x] = ok;
        }
    };

    // the query row
    f16x8 qf[PIECES][STEPS];
    int e = 0;
    {
        const T* qp = (const T*)a.q + (int64_t)row * a.ld + a.q_col + head * D + 8 * h;
        if (F32) {
            float top = 0.f;
            for (int s = 0; s < STEPS; ++s)
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)qp[16 * s + j]));
            top = fmaxf(top, __shfl_xor(top, 32));
            (void)frexpf(top, &e);
            e = top > 0.f && top < INFINITY ? 14 - e : 0;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = F32 ? ldexpf((float)qp[16 * s + j], e) : (float)qp[16 * s + j];
                const half_t hi = (half_t)y;
                qf[0][s][j] = hi;
                if (F32) qf[PIECES - 1][s][j] = (half_t)(y - (float)hi);
            }
    }
    float m = kNone, l = 0.f;  // m and ex the row's, l the lane's
    float ex = kUnseen;
    fx16 o[DB];
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

    auto attend = [&](int tb, int stage, bool masked) {
        const int ka = kget + stage * STAGE, va = vget + stage * STAGE;
        fx16 x[2];
        float ku[2], lv[2], iv[2], top[2], mx = -INFINITY;
        // operands are read in groups, one group ahead of its MFMAs
        constexpr int GK = STEPS < 4 || D > 128 || (D == 128 && F32) ? 2 : 4, GV = GK, GROUPS = 2 * STEPS / GK;
        f16x8 kf[2][GK], vf[2][GV];
        auto read_k = [&](int n) {
#pragma unroll
            for (int u = 0; u < GK; ++u) {
                const int st = n * GK + u;
                kf[n & 1][u] = *reinterpret_cast<const f16x8*>(lds + (ka ^ st % STEPS * 32) + st / STEPS * 32 * KRB);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto read_v = [&](int n) {
#pragma unroll
            for (int w = 0; w < GV; ++w) {
                const int u = (n * GV + w) % 4, c = (n * GV + w) / 4;
                vf[n & 1][w] = *reinterpret_cast<const f16x8*>(lds + (va ^ ((u >> 1) * 64 + (u & 1) * 16)) + c * 32 * 128);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        read_k(0);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int n = kb * GROUPS / 2; n < (kb + 1) * GROUPS / 2; ++n) {
                if (n + 1 < GROUPS)
                    read_k(n + 1);
                else
                    read_v(0);
#pragma unroll
                for (int u = 0; u < GK; ++u)
#pragma unroll
                    for (int pc = PIECES - 1; pc >= 0; --pc) {
                        const bool first = n == kb * GROUPS / 2 && u == 0 && pc == PIECES - 1;
                        x[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n & 1][u], qf[pc][n * GK % STEPS + u], first ? fx16{} : x[kb], 0, 0, 0);
                    }
            }
            const fx4 un = *reinterpret_cast<const fx4*>(units + stage * 20 + (2 * kb + h) * 4);
            ku[kb] = F32 ? ldexpf(un[0], -e) : un[0], lv[kb] = un[1], iv[kb] = un[2];
            ku[kb] = ku[kb] == 0.f ? 0x1p-126f : ku[kb];  // for the product with -inf
            // key tb + 32 kb + 16 h + r is in x[kb][r]
            if (masked) {
                const int j = tb + 32 * kb, low = a.window > 0 ? posh - a.window : INT_MIN;
                const int up = un[3] != 0.f ? posh : INT_MIN;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = x[kb][r];
                    x[kb][r] = j + r <= up && j + r > low ? y : -INFINITY;
                }
                // a row that sees none of the 16: their scales are not its own
                if (!(j <= up && j + 15 > low)) ku[kb] = 1.f, lv[kb] = 0.f, iv[kb] = 0.f;
            }
            top[kb] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top[kb] = fmaxf(top[kb], x[kb][r]);
            mx = fmaxf(mx, fmaf(top[kb], ku[kb], lv[kb]));
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        float factor[2] = {ldexpf(iv[0], (int)ex), ldexpf(iv[1], (int)ex)};
        if (__any(mx > m + kSlack || fmaxf(factor[0], factor[1]) > kMostFactor)) {
            const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - mn);
            float far = fmaxf(reference(m, ex), fmaxf(top[0] * ku[0], top[1] * ku[1]));
            far = fmaxf(far, __shfl_xor(far, 32));
            const float en = exponent(mn, far);
            l *= rescale(m, ex, mn, en);
            m = mn, ex = en;
#pragma unroll
            for (int c = 0; c < DB; ++c) o[c] *= alpha;
            factor[0] = ldexpf(iv[0], (int)ex), factor[1] = ldexpf(iv[1], (int)ex);
            if (__any(fmaxf(factor[0], factor[1]) > kMostFactor)) {
                const float base = reference(m, ex);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float s = x[kb][r];
                        l += __builtin_amdgcn_exp2f(fmaf(s, ku[kb], -base));
                    }
                    factor[kb] = 0.f;
                }
            }
        }
        const float base = m - kPLog;
        f16x8 pf[PIECES][2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const float shift = lv[kb] - base;  // base: m - 12, of p's 2^12
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float s = x[kb][r], p = __builtin_amdgcn_exp2f(fmaf(s, ku[kb], shift));
                sum += p;
                x[kb][r] = p;
            }
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = x[kb][r], p1 = x[kb][r + 1];
                const f16x2 hi = __builtin_convertvector((fx2{p0, p1}), f16x2);
                pf[0][kb][r / 8][r % 8] = hi[0], pf[0][kb][r / 8][r % 8 + 1] = hi[1];
                if (F32) {
                    const f16x2 lo = __builtin_convertvector((fx2{p0 - (float)hi[0], p1 - (float)hi[1]}), f16x2);
                    pf[PIECES - 1][kb][r / 8][r % 8] = lo[0], pf[PIECES - 1][kb][r / 8][r % 8 + 1] = lo[1];
                }
            }
            l = fmaf(sum, factor[kb], l);
        }
#pragma unroll
        for (int n = 0; n < DB * 4 / GV; ++n) {
            if (n + 1 < DB * 4 / GV) read_v(n + 1);
#pragma unroll
            for (int w = 0; w < GV; ++w) {
                const int u = (n * GV + w) % 4, c = (n * GV + w) / 4;
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc)
                    o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n & 1][w], pf[pc][u >> 1][u & 1], o[c], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (from < to) {
        find(from);
        load(from);
        find(from + 64);
        store(0);
        load(from + 64);
        find(from + 128);
    }
    int stage = 0;
    for (int tb = from; tb < to; tb += 64, stage ^= 1) {
        dma_barrier<63>();  // this chunk is stored, the other stage is no longer read; loads stay in flight
        store(stage ^ 1);
        load(tb + 128);
        find(tb + 192);
        const bool whole = tb + 63 <= first_pos && (a.window <= 0 || tb > last_pos - a.window);
        const fx4 ok = *reinterpret_cast<const fx4*>(units + stage * 20 + 16);
        attend(tb, stage, !whole || !__all(ok[0] * ok[1] * ok[2] * ok[3] != 0.f));
    }

    l += __shfl_xor(l, 32);
    if (!row_ok) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T* op = (T*)a.out + ((int64_t)row * a.heads + head) * D + 4 * h;
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            T v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (T)ldexpf(o[c][4 * q + r] * inv, (int)ex);
            __builtin_memcpy(__builtin_assume_aligned(op + 32 * c + 8 * q, 4 * sizeof(T)), v, sizeof v);
        }
}

template <typename T, int D, int NW>
static void launch_prompt(const char* name, const KvAttnArgs& a) {
    auto kernel = kv_prompt_k<T, D, NW>;
    constexpr int lds = 2 * (64 * 2 * D + D * 128) + 2 * 20 * 4;
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    launch(NW == 8 ? "nnc_hip_kv_attention_256" : "nnc_hip_kv_attention_128", kernel, dim3((unsigned)(a.tiles * a.kv_heads)), dim3(64 * NW), lds, a);
}

template <typename T, int D>
static void launch_kv_attention(const char* name, const KvAttnArgs& a, int tile, int waves) {
    if constexpr (D <= 128) {  // (dim 256: 512 registers a wave, and four of them)
        if (tile == 256) return launch_prompt<T, D, 8>(name, a);
    }
    if (tile == 128) return launch_prompt<T, D, 4>(name, a);
    const dim3 grid((unsigned)a.tiles, (unsigned)a.kv_heads, (unsigned)a.splits);
    if constexpr (D <= 128) {
        if (waves == 4) return launch(name, kv_attention_k<T, D, 4>, grid, dim3(256), 0, a);
        if (waves == 2) return launch(name, kv_attention_k<T, D, 2>, grid, dim3(128), 0, a);
    }
    launch(name, kv_attention_k<T, D, token_waves(D)>, grid, dim3(64 * token_waves(D)), 0, a);
}

template <typename T>
static void launch_dim(const char* name, const KvAttnArgs& a, int tile, int waves, int dim) {
    switch (dim) {
        case 32: return launch_kv_attention<T, 32>(name, a, tile, waves);
        case 64: return launch_kv_attention<T, 64>(name, a, tile, waves);
        case 128: return launch_kv_attention<T, 128>(name, a, tile, waves);
        default: return launch_kv_attention<T, 256>(name, a, tile, waves);
    }
}

// Query rows of a workgroup: 256 or 128 by the prompt kernel, 16 by the other,
// which divides the keys instead. By the time that a CU takes for 64 keys,
// dim 128, in us: 256 rows 2.5, 128 rows 1.9, two workgroups of them 3.0,
// 256 rows as 16 tiles of 16 6.1. With 256, 128 and 16 rows, us, 32 heads over 8
// of 128, f16: two prompts of 2048 behind 2048 241, 285, 592; 16 of 1024 256, 253,
// 523; four of 256 behind 1792 76, 68, 101; one of 256 behind 7936 264, 242, 92;
// one of 256 17, 15, 10; 64 of 16 behind 1008 79, 52, 85, of 4 behind 4092 298,
// 192, 99. fp32: two of 2048 375, 426, 643; 16 of 1024 374, 373, 630; four of 256
// 107, 89, 120; one of 256 behind 7936 372, 311, 106.
static int query_tile(int64_t rows, int64_t batch, int group, int kv_heads, int dim) {
    const int64_t cus = cu_count(), holders = rows < batch ? rows : batch;  // sequences that can have rows
    auto count = [&](int tile) {
        const int64_t n = ceil_div(rows * group, tile);
        return (n > holders ? n : holders) * kv_heads;
    };
    const int64_t n256 = count(256), n128 = count(128);
    const double t16 = 6.1 * (double)(rows * group) * kv_heads / (256.0 * cus);
    const double t128 = n128 <= cus ? 1.9 : 3.0 * ceil_div(n128, 2 * cus);
    const double t256 = dim <= 128 ? 2.5 * ceil_div(n256, cus) : 1e30;
    return t256 < t128 && t256 < t16 ? 256 : t128 < t16 ? 128 : 16;
}

// Waves of a workgroup of 16 query rows. All workgroups at once: as many as
// there can be. In several rounds, fewer waves leave room for other
// workgroups on the CU, whose keys arrive while one starts or joins; more
// have a long sequence done sooner. 8, 4 and 2 waves, us, 32 heads over 8 of
// 128, f16: 64 sequences of up to 8192 106, 112, 127; 64 of 4096 100, 97, 101;
// 64 of up to 1024 25, 20, 22; 128 of up to 4096 114, 102, 117; 128 of up to 512
// 38, 25, 20; 256 of up to 1024 99, 66, 53; 512 of up to 4096 448, 403, 423; 512
// of up to 300, 8 heads of 64, fp32 121, 50, 34.
static int query_waves(int64_t items, int longest) {
    const double rounds = (double)items / cu_count();
    if (rounds <= 1.0 || longest > 2048 * rounds) return 8;
    return rounds >= 4.0 && longest <= 128 * rounds ? 2 : 4;
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_kv_attention(Tensor* q, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                          Tensor* starts, Tensor* lengths, Tensor* out, int q_col, int heads, float scale, int window,
                          int max_length) {
    const char* name = "nnc_hip_kv_attention";
    CacheArgs c;
    int64_t rows = 0, ld = 0;
    if (!cache_args(name, k_cache, v_cache, k_scale, v_scale, table, starts, lengths, 0, &c)) return;
    if (heads < 1 || heads % c.kv_heads != 0 || heads > 65535)
        return fail(NNC_HIP_EINVAL, name, "%d heads over %d cached ones", heads, c.kv_heads);
    const int64_t width = (int64_t)heads * c.dim;
    if (!rows_arg(name, "q", q, q_col, width, &rows, &ld)) return;
    if (!has_data(out) || !good_shape(out) || out->dtype != q->dtype || numel(out) != rows * width ||
        out->shape[out->ndim - 1] != width)
        return fail(NNC_HIP_EINVAL, name, "out must be [rows][heads * dim] of q's type");
    if (window < 0 || max_length < 0) return fail(NNC_HIP_EINVAL, name, "negative window or max_length");
    if (!(scale > 0.f) || !(scale < INFINITY)) return fail(NNC_HIP_EINVAL, name, "scale must be positive");
    if (!aligned16(out->data)) return fail(NNC_HIP_EUNSUPP, name, "out must be 16-byte aligned");
    if (rows == 0 || c.ragged.batch == 0) return;
    const int group = heads / c.kv_heads;
    if (rows * group > (1 << 27)) return fail(NNC_HIP_EUNSUPP, name, "%lld rows of %d heads", (long long)rows, heads);
    if (!ready(name)) return;
    const int capacity = c.ragged.width * c.page;
    const int longest = max_length > 0 && max_length < capacity ? max_length : capacity;
    const int tile = query_tile(rows, c.ragged.batch, group, c.kv_heads, c.dim);
    const int64_t tiles = query_tiles_bound(rows, c.ragged.batch, group, tile), items = tiles * c.kv_heads;
    if (items * 64 * 8 > UINT32_MAX) return fail(NNC_HIP_EUNSUPP, name, "%lld rows of %d heads", (long long)rows, heads);
    KvAttnArgs a{c.ragged, c.k, c.v, c.k_scale, c.v_scale, q->data, out->data, nullptr, nullptr, ld, q_col, heads, c.kv_heads,
                 group, window_of(window, capacity), 1, 64, (int)tiles, slot_magic(c.page / 16),
                 aligned16(q->data) && ld * activation_bytes(q) % 16 == 0 && q_col * activation_bytes(q) % 16 == 0, false,
                 scale * 1.44269504088896340736f};
    a.g.rows = (int)rows;
    const int waves = query_waves(items, longest);
    a.by_length = tile == 16 && items > cu_count() && c.ragged.batch <= kOrdered && rows <= kOrdered;
    if (tile == 16) {
        // shares of the keys, 512 or more each, while all workgroups run at
        // once, one on a CU (a second round starts 6 us later: one sequence of
        // 131072 in 32 shares 48.2 us, in 64 54.9, call after call on one cache).
        // By the longest sequence: a window leaves most shares empty, and one
        // token behind 131072 takes 31 us under a window of 8192
        const int step = 64 * token_waves(c.dim);
        const int64_t want = cu_count() / items, most = ceil_div(longest, 512);
        a.splits = (int)(want < most ? want : most);
        if (a.splits < 1) a.splits = 1;
        a.chunk = (int)(ceil_div(ceil_div(longest > 0 ? longest : 1, a.splits), step) * step);
    }
    if (a.splits > 1) {
        const size_t bytes = (size_t)items * a.splits * tile * (c.dim + 4) * sizeof(float);
        a.part = workspace(bytes);
        a.counters = tile_counters((size_t)items);
        if (!a.part || !a.counters) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes of partial sums", bytes);
    }
    // every sequence taken as the longest; of it, what its rows' windows reach
    const int64_t reach = a.window > 0 ? (int64_t)a.window - 1 + ceil_div(rows, c.ragged.batch) : longest;
    set_work(0.0, 2.0 * c.kv_heads * c.dim * (double)(reach < longest ? reach : longest) * c.ragged.batch);
    if (q->dtype == NNC_DTYPE_FLOAT16)
        launch_dim<half_t>(name, a, tile, waves, c.dim);
    else
        launch_dim<float>(name, a, tile, waves, c.dim);
}

}  // extern "C"
