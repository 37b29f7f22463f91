// Attention over the paged 8-bit cache (nnc_hip_kv_attention). No reference
// counterpart.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j
//   j <= pos_i, j > pos_i - window;  k_j = K_j u_k(page), v_j = V_j u_v(page)
//
// with K, V whole numbers and one scale for each page and head. One pass over
// the keys: in units of powers of two, x_j = scale log2(e) u_k (q . K_j) +
// log2(u_v), running maximum m of x, p_j = 2^(x_j - m); then
//
//   out = (sum_j p_j V_j) / (sum_j p_j / u_v(j))
//
// so that the pages' value scales cost nothing in the second product, and p
// has the size of what it contributes.
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
// bits), and so is p then (f16 outputs: p rounded to f16 once, 2^-12 of it).
//
// A workgroup takes 16 query rows - heads of one cached head, then tokens -
// and a share of the keys, its four waves 64 keys each in turn; the waves'
// sums are joined through LDS, the shares' through the workspace.
#include <limits.h>

#include "mfma_tile.h"
#include "quant8.h"

namespace nnc {

struct KvAttnArgs {
    Ragged g;
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    const void* q;
    void* out;
    float* part;  // [row][head][split][dim + 2]: sums, maximum, divisor
    int64_t ld;
    int q_col, heads, kv_heads, group, window, splits, chunk, tile;  // tile: query rows of a workgroup
    uint32_t slot_magic;
    float scale;  // with log2(e)
};

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

// p is scaled by this before it is rounded to f16: its smallest steps are
// then 2^-36 of the row's largest
static constexpr float kPLog = 12.f, kPScale = 4096.f;
typedef float fx2 __attribute__((ext_vector_type(2)));

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_attention_k(KvAttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int STEPS = D / 32, PIECES = F32 ? 2 : 1, KV = D / 16;
    __shared__ float ml[2][4][16];
    __shared__ __align__(16) float os[3][16][D + 4];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head_kv = blockIdx.y, split = blockIdx.z;
    int tile = blockIdx.x;
    const int b = find_share(tile, a.g.batch, [&](int s) { return query_tiles(span_of(a.g, s), a.group, 16); });
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
    const KeyRange range(first_pos, span.first() + (int)(last / a.group), a.window, a.splits, a.chunk, 256);
    const int shares = range.shares();
    if (split >= shares) return;
    const int from = range.lo + split * range.chunk;
    const int to = min(range.hi, from + range.chunk);

    // the query row's dims g * D / 4 .. + D / 4
    f16x8 qf[PIECES][STEPS];
    float qs = a.scale;
    {
        const T* qp = (const T*)a.q + row * a.ld + a.q_col + head * D + g * (D / 4);
        float x[D / 4];
        float top = 0.f;
#pragma unroll
        for (int d = 0; d < D / 4; ++d) {
            x[d] = row_ok ? (float)qp[d] : 0.f;
            top = fmaxf(top, fabsf(x[d]));
        }
        if (F32) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // the row's largest value to [2^13, 2^14)
            int e = 0;
            (void)frexpf(top, &e);
            e = top > 0.f && top < INFINITY ? 14 - e : 0;
            qs = ldexpf(qs, -e);
#pragma unroll
            for (int d = 0; d < D / 4; ++d) x[d] = ldexpf(x[d], e);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[8 * s + j];
                const half_t hi = (half_t)y;
                qf[0][s][j] = hi;
                if (F32) qf[PIECES - 1][s][j] = (half_t)(y - (float)hi);
            }
    }
    float m = -INFINITY, l = 0.f;
    fx4 o[KV];
#pragma unroll
    for (int c = 0; c < KV; ++c) o[c] = fx4{0.f, 0.f, 0.f, 0.f};

    const int page = a.g.page, page16 = page / 16;
    const int64_t plane = (int64_t)page * D;
    for (int tb = from + 64 * wave; tb < to; tb += 256) {
        // K: the lane's row in the four blocks is in 16-key group i / 4
        uint32_t kb[4][D / 16];
        {
            const int t16 = tb / 16 + (i >> 2), slot = t16 / page16;
            const int pn = t16 * 16 < to ? page_at(a.g, b, slot) : -1;
            const int8_t* kp = a.k + ((int64_t)max(pn, 0) * a.kv_heads + head_kv) * plane +
                               (int64_t)((t16 - slot * page16) * 16 + (i & 3)) * D + g * (D / 4);
#pragma unroll
            for (int bl = 0; bl < 4; ++bl)
#pragma unroll
                for (int c = 0; c < D / 16; c += 2) {
                    const ix2 w = *reinterpret_cast<const ix2*>(kp + bl * 4 * D + 4 * c);
                    kb[bl][c] = w[0], kb[bl][c + 1] = w[1];
                }
        }
        // V: the lane's 16 keys are group g
        ix4 vb[KV];
        const int t16 = tb / 16 + g, slot = t16 / page16;
        const int pn = t16 * 16 < to ? page_at(a.g, b, slot) : -1;
        const int64_t at = (int64_t)max(pn, 0) * a.kv_heads + head_kv;
        {
            const int8_t* vp = a.v + at * plane + (t16 - slot * page16) * 16 + i * page;
#pragma unroll
            for (int c = 0; c < KV; ++c) vb[c] = *reinterpret_cast<const ix4*>(vp + c * 16 * page);
        }
        const float ku = pn >= 0 ? a.k_scale[at] * qs : 0.f;
        float vu = pn >= 0 ? a.v_scale[at] : 1.f;
        vu = vu == 0.f ? 1.f : vu;
        const float lv = __builtin_amdgcn_logf(vu), iv = 1.0f / vu;
        // scores of keys tb + 16 g + 4 b + r
        float x[16];
#pragma unroll
        for (int bl = 0; bl < 4; ++bl) {
            fx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const f16x8 kf = widen8(kb[bl][2 * st], kb[bl][2 * st + 1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[pc][st], s, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = tb + 16 * g + 4 * bl + r;
                const bool seen = pn >= 0 && j <= pos && (a.window <= 0 || j > pos - a.window);
                x[4 * bl + r] = seen ? fmaf(s[r], ku, lv) : -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int c = 1; c < 16; ++c) mx = fmaxf(mx, x[c]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l *= alpha;
        float p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            p[c] = __builtin_amdgcn_exp2f(x[c] - base);
            l += x[c] == -INFINITY ? 0.f : p[c] * iv;
        }
#pragma unroll
        for (int c = 0; c < KV; ++c) o[c] *= alpha;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f16x8 pf[PIECES];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = p[8 * h + j] * kPScale;
                const half_t hi = (half_t)y;
                pf[0][j] = hi;
                if (F32) pf[PIECES - 1][j] = (half_t)(y - (float)hi);
            }
#pragma unroll
            for (int c = 0; c < KV; ++c) {
                const f16x8 vf = widen8((uint32_t)vb[c][2 * h], (uint32_t)vb[c][2 * h + 1]);
#pragma unroll
                for (int pc = PIECES - 1; pc >= 0; --pc) o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[pc], o[c], 0, 0, 0);
            }
        }
    }
    // join the waves
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) ml[0][wave][i] = m, ml[1][wave][i] = l;
    __syncthreads();
    float top = ml[0][0][i];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[0][w][i]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += ml[1][w][i] * __builtin_amdgcn_exp2f(ml[0][w][i] - base);
    const float f = __builtin_amdgcn_exp2f(m - base) * (1.0f / kPScale);
#pragma unroll
    for (int c = 0; c < KV; ++c) {
        o[c] *= f;
        if (wave > 0) *reinterpret_cast<fx4*>(&os[wave - 1][i][16 * c + 4 * g]) = o[c];
    }
    __syncthreads();
    if (wave > 0 || !row_ok) return;
#pragma unroll
    for (int c = 0; c < KV; ++c)
#pragma unroll
        for (int w = 0; w < 3; ++w) o[c] += *reinterpret_cast<const fx4*>(&os[w][i][16 * c + 4 * g]);
    if (shares == 1) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        T* op = (T*)a.out + (row * a.heads + head) * D + 4 * g;
#pragma unroll
        for (int c = 0; c < KV; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) op[16 * c + r] = (T)(o[c][r] * inv);
    } else {
        float* pp = a.part + ((row * a.heads + head) * a.splits + split) * (D + 2);
#pragma unroll
        for (int c = 0; c < KV; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) pp[16 * c + 4 * g + r] = o[c][r];
        if (g == 0) pp[D] = top, pp[D + 1] = sum;
    }
}

// ---------------------------------------------------------------------------
// Many query rows (prompts): 32 rows per wave, 4 or 8 waves, the keys 64 at a
// time through LDS, where they are kept as f16: widened once for all waves. v_mfma_f32_32x32x16_f16 as above; query row i = lane % 32, lane half
// h. Row 8q + 4h + u of a block of 32 keys is key 16h + 4q + u: lane half h
// has the scores of 16 consecutive keys, which one page's scales serve.
//
// LDS rows: K's in that order, 2 dim bytes each; V's one per dim, 128 bytes.
// Their 16-byte chunks are permuted so that 16 lanes reading a chunk of 16
// rows hit all 64 banks. Two stages: chunk t + 1 is widened and stored, and
// the loads of t + 2 go out, before t is used, with one barrier for each.
//
// The accumulators are only scaled down when some row's maximum has grown by
// more than 2^3 since they last were (p is f16 and starts at 2^12).
// ---------------------------------------------------------------------------
typedef float fx16 __attribute__((ext_vector_type(16)));

template <int RB>
__device__ __forceinline__ int lds_chunk(int row, int chunk) {  // byte offset; rows of RB bytes
    const int key = RB >= 256 ? row & 15 : RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
    return row * RB + (chunk ^ key) * 16;
}

template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, D <= 128 || NW == 8 ? 2 : 1) kv_prompt_k(KvAttnArgs a, int tiles) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int STEPS = D / 16, PIECES = F32 ? 2 : 1, DB = D / 32, KRB = 2 * D;
    constexpr int ROWS = 32 * NW, THREADS = 64 * NW, STAGE = 64 * KRB + D * 128, LOADS = (4 * D + THREADS - 1) / THREADS;  // 16-byte pieces per thread and operand
    constexpr float kSlack = 3.f;
    extern __shared__ __align__(16) char lds[];
    // [stage]: of 4 groups of 16 keys, K's scale, V's scale's logarithm and
    // inverse, 1 if they can be read; then the four last again
    float* units = (float*)(lds + 2 * STAGE);
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // one XCD after the other, so that the tiles of a head share its L2; the
    // tiles with most keys first
    const int lin = xcd_remap(blockIdx.x, tiles * a.kv_heads * a.splits);
    const int split = lin / (tiles * a.kv_heads), head_kv = lin / tiles - split * a.kv_heads;
    int tile = tiles - 1 - lin % tiles;
    const int b = __builtin_amdgcn_readfirstlane(
        find_share(tile, a.g.batch, [&](int s) { return query_tiles(span_of(a.g, s), a.group, ROWS); }));
    if (b < 0) return;
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Span span = span_of(a.g, b);
    const int64_t all = (int64_t)span.rows * a.group, row0 = (int64_t)tile * ROWS;
    const int64_t last = row0 + ROWS - 1 < all ? row0 + ROWS - 1 : all - 1;
    const int first_pos = span.first() + (int)(row0 / a.group), last_pos = span.first() + (int)(last / a.group);
    const KeyRange range(first_pos, last_pos, a.window, a.splits, a.chunk, 64);
    const int shares = range.shares();
    if (split >= shares) return;
    const int from = range.lo + split * range.chunk, to = min(range.hi, from + range.chunk);
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
            const float vu = !can_read || su[1] == 0.f ? 1.f : su[1], ok = can_read ? 1.f : 0.f;
            *reinterpret_cast<fx4*>(units + stage * 20 + threadIdx.x * 4) =
                fx4{can_read ? su[0] * a.scale : 0.f, __builtin_amdgcn_logf(vu), 1.0f / vu, ok};
            units[stage * 20 + 16 + threadIdx.x] = ok;
        }
    };

    // the query row
    f16x8 qf[PIECES][STEPS];
    float qscale = 1.f;
    {
        const T* qp = (const T*)a.q + (int64_t)row * a.ld + a.q_col + head * D + 8 * h;
        int e = 0;
        if (F32) {
            float top = 0.f;
            for (int s = 0; s < STEPS; ++s)
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)qp[16 * s + j]));
            top = fmaxf(top, __shfl_xor(top, 32));
            (void)frexpf(top, &e);
            e = top > 0.f && top < INFINITY ? 14 - e : 0;
            qscale = ldexpf(1.f, -e);
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
    float m = -INFINITY, l = 0.f;
    fx16 o[DB];
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

    auto attend = [&](int tb, int stage, bool masked) {
        const int ka = kget + stage * STAGE, va = vget + stage * STAGE;
        fx16 x[2];
        float ku[2], lv[2], iv[2], mx = -INFINITY;
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
            ku[kb] = un[0] * qscale, lv[kb] = un[1], iv[kb] = un[2];
            ku[kb] = ku[kb] == 0.f ? 0x1p-126f : ku[kb];  // for the product with -inf
            // key tb + 32 kb + 16 h + r is in x[kb][r]
            if (masked) {
                const int j = tb + 32 * kb, low = a.window > 0 ? posh - a.window : INT_MIN;
                const int top = un[3] != 0.f ? posh : INT_MIN;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = x[kb][r];
                    x[kb][r] = j + r <= top && j + r > low ? y : -INFINITY;
                }
                // a row that sees none of the 16: their scales are not its own
                if (!(j <= top && j + 15 > low)) ku[kb] = 1.f, lv[kb] = 0.f, iv[kb] = 0.f;
            }
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, x[kb][r]);
            mx = fmaxf(mx, fmaf(top, ku[kb], lv[kb]));
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m + kSlack)) {
            const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int c = 0; c < DB; ++c) o[c] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m - kPLog;
        f16x8 pf[PIECES][2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const float shift = lv[kb] - base;  // base: m - 12, the 2^12 of kPScale
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
            l = fmaf(sum, iv[kb], l);
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
    if (shares == 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* op = (T*)a.out + ((int64_t)row * a.heads + head) * D + 4 * h;
#pragma unroll
        for (int c = 0; c < DB; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = (T)(o[c][4 * q + r] * inv);
                __builtin_memcpy(__builtin_assume_aligned(op + 32 * c + 8 * q, 4 * sizeof(T)), v, sizeof v);
            }
    } else {
        float* pp = a.part + (((int64_t)row * a.heads + head) * a.splits + split) * (D + 2);
#pragma unroll
        for (int c = 0; c < DB; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) pp[32 * c + 8 * (r >> 2) + 4 * h + (r & 3)] = o[c][r];
        if (h == 0) pp[D] = m, pp[D + 1] = l;
    }
}

// joins the shares of one query row and head, in their order
template <typename T, int D>
__global__ void __launch_bounds__(64) kv_attention_join_k(KvAttnArgs a) {
    int tok = blockIdx.x;
    const int b = find_share(tok, a.g.batch, [&](int s) { return span_of(a.g, s).rows; });
    if (b < 0) return;
    const Span span = span_of(a.g, b);
    const int head = blockIdx.y, gh = head % a.group;
    // the tile that the row was in
    const int64_t all = (int64_t)span.rows * a.group, tile = ((int64_t)tok * a.group + gh) / a.tile;
    const int64_t last = (tile + 1) * a.tile < all ? (tile + 1) * a.tile - 1 : all - 1;
    const KeyRange range(span.first() + (int)(tile * a.tile / a.group), span.first() + (int)(last / a.group), a.window,
                         a.splits, a.chunk, a.tile == 16 ? 256 : 64);
    const int shares = range.shares();
    if (shares == 1) return;
    const int64_t row = span.end - span.rows + tok;
    const float* pp = a.part + (row * a.heads + head) * a.splits * (D + 2);
    float top = -INFINITY;
    for (int s = 0; s < shares; ++s) top = fmaxf(top, pp[(int64_t)s * (D + 2) + D]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int s = 0; s < shares; ++s) sum += pp[(int64_t)s * (D + 2) + D + 1] * __builtin_amdgcn_exp2f(pp[(int64_t)s * (D + 2) + D] - base);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    for (int d = threadIdx.x; d < D; d += 64) {
        float o = 0.f;
        for (int s = 0; s < shares; ++s) o += pp[(int64_t)s * (D + 2) + d] * __builtin_amdgcn_exp2f(pp[(int64_t)s * (D + 2) + D] - base);
        ((T*)a.out)[(row * a.heads + head) * D + d] = (T)(o * inv);
    }
}

template <typename T, int D, int NW>
static void launch_prompt(const char* name, const KvAttnArgs& a, unsigned tiles) {
    auto kernel = kv_prompt_k<T, D, NW>;
    constexpr int lds = 2 * (64 * 2 * D + D * 128) + 2 * 20 * 4;
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    launch(name, kernel, dim3(tiles * (unsigned)(a.kv_heads * a.splits)), dim3(64 * NW), lds, a, (int)tiles);
}

template <typename T, int D>
static void launch_kv_attention(const char* name, const KvAttnArgs& a, unsigned tiles) {
    if (a.tile >= 128) {
        if constexpr (D <= 128) {  // (dim 256: 512 registers a wave, and four of them)
            if (a.tile == 256) launch_prompt<T, D, 8>(name, a, tiles);
        }
        if (a.tile == 128) launch_prompt<T, D, 4>(name, a, tiles);
    } else {
        launch(name, kv_attention_k<T, D>, dim3(tiles, (unsigned)a.kv_heads, (unsigned)a.splits), dim3(256), 0, a);
    }
    if (a.splits > 1)
        launch("nnc_hip_kv_attention_join", kv_attention_join_k<T, D>, dim3((unsigned)a.g.rows, (unsigned)a.heads), dim3(64), 0, a);
}

template <typename T>
static void launch_dim(const char* name, const KvAttnArgs& a, unsigned tiles, int dim) {
    switch (dim) {
        case 32: return launch_kv_attention<T, 32>(name, a, tiles);
        case 64: return launch_kv_attention<T, 64>(name, a, tiles);
        case 128: return launch_kv_attention<T, 128>(name, a, tiles);
        default: return launch_kv_attention<T, 256>(name, a, tiles);
    }
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
    const int64_t holders = rows < c.ragged.batch ? rows : c.ragged.batch;  // sequences that can have rows
    const int tile = c.dim <= 128 && rows * group >= 256 * holders ? 256 : rows * group >= 64 * holders ? 128 : 16, step = tile == 16 ? 256 : 64;
    const int64_t tiles = query_tiles_bound(rows, c.ragged.batch, group, tile);
    KvAttnArgs a{c.ragged, c.k, c.v, c.k_scale, c.v_scale, q->data, out->data, nullptr, ld, q_col, heads, c.kv_heads,
                 group, window, 1, 0, tile, slot_magic(c.page / 16), scale * 1.44269504088896340736f};
    a.g.rows = (int)rows;
    // enough shares of the keys to give every CU sixteen waves (eight of prompts)
    const int64_t want = ceil_div((tile == 256 ? 1 : tile == 128 ? 2 : 4) * (int64_t)cu_count(), tiles * c.kv_heads), most = ceil_div(longest, 512);
    a.splits = (int)(want < most ? want : most);
    if (a.splits < 1) a.splits = 1;
    a.chunk = (int)(ceil_div(ceil_div(longest > 0 ? longest : 1, a.splits), step) * step);
    if (a.splits > 1) {
        const size_t bytes = (size_t)rows * heads * a.splits * (c.dim + 2) * sizeof(float);
        a.part = workspace(bytes);
        if (!a.part) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes of partial sums", bytes);
    }
    set_work(0.0, 2.0 * c.kv_heads * c.dim * (double)longest * c.ragged.batch);
    if (q->dtype == NNC_DTYPE_FLOAT16)
        launch_dim<half_t>(name, a, (unsigned)tiles, c.dim);
    else
        launch_dim<float>(name, a, (unsigned)tiles, c.dim);
}

}  // extern "C"
