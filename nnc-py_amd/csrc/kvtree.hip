// Attention of drafted tokens over the paged 8-bit cache
// (nnc_hip_kv_tree_attention). No reference counterpart.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j
//   j < first, or j = first + m for the rows m that row i's mask names
//
// with first the position of the sequence's first new row: a tree of drafts,
// whose branches do not see each other, behind a common context.
#include <limits.h>

#include "quant8.h"

namespace nnc {

struct TreeArgs {
    Ragged g;
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    const int* tree;  // [rows][words]
    const void* q;
    void* out;
    int64_t ld;
    int q_col, heads, kv_heads, group, window, words;
    float scale;  // with log2(e)
};

// A workgroup to a row and head, a wave to 64 keys at a time, a key a lane for
// the scores and a dim a lane for the values. Float32 throughout.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_tree_k(TreeArgs a) {
    constexpr int PER = D / 64 ? D / 64 : 1;
    __shared__ float qs[D], ps[4][64], os[4][D], ml[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = blockIdx.y, head_kv = head / a.group;
    int at = blockIdx.x;
    const int b = find_share(at, a.g.batch, [&](int s) { return span_of(a.g, s).rows; });
    if (b < 0) return;
    const Span span = span_of(a.g, b);
    const int first = span.first();
    const int64_t row = span.end - span.rows + at;
    const int* mask = a.tree + row * a.words;
    int low = INT_MIN;
    if (a.window > 0) low = first + tree_depth(mask, a.words, span.rows) - 1 - a.window;
    const T* qp = (const T*)a.q + row * a.ld + a.q_col + (int64_t)head * D;
    for (int d = threadIdx.x; d < D; d += 256) qs[d] = (float)qp[d];
    __syncthreads();
    const int page = a.g.page;
    float m = -INFINITY, l = 0.f, o[PER] = {};
    for (int tb = 64 * wave; tb < span.length; tb += 256) {
        const int j = tb + lane;
        const uint32_t bits = tree_bits(mask, a.words, first, span.length, j & ~15);
        const int pn = j < span.length ? page_at(a.g, b, j / page) : -1;
        float s = -INFINITY, u = 0.f;
        if (pn >= 0 && (bits >> (j & 15) & 1) && (j >= first || j > low)) {
            const int64_t plane = (int64_t)pn * a.kv_heads + head_kv;
            const int8_t* k = a.k + (plane * page + j % page) * D;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot = fmaf(qs[d], (float)k[d], dot);
            s = dot * (a.k_scale[plane] * a.scale);
            u = a.v_scale[plane];
        }
        float top = s;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) top = max_nan(top, __shfl_xor(top, x));
        const float mn = max_nan(m, top), base = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2f(m - base), p = s == -INFINITY ? 0.f : exp2f(s - base);
        l = l * alpha + wave_add(p);
        m = mn;
        ps[wave][lane] = p == 0.f ? 0.f : p * u;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = lane + 64 * i;
            o[i] *= alpha;
            if (d < D)
                for (int c = 0; c < 64; c += 16) {
                    const int pc = tb + c < span.length ? page_at(a.g, b, (tb + c) / page) : -1;
                    if (pc < 0) continue;
                    const int8_t* v = a.v + (((int64_t)pc * a.kv_heads + head_kv) * D + d) * page + (tb + c) % page;
                    for (int e = 0; e < 16; ++e)
                        if (ps[wave][c + e] != 0.f) o[i] = fmaf(ps[wave][c + e], (float)v[e], o[i]);
                }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) ml[0][wave] = m, ml[1][wave] = l;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 64 * i < D) os[wave][lane + 64 * i] = o[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < 4; ++w) top = max_nan(top, ml[0][w]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < 4; ++w) sum += ml[1][w] * exp2f(ml[0][w] - base);
    T* out = (T*)a.out + (row * a.heads + head) * D;
    for (int d = threadIdx.x; d < D; d += 256) {
        float y = 0.f;
        for (int w = 0; w < 4; ++w) y += os[w][d] * exp2f(ml[0][w] - base);
        out[d] = (T)(sum == 0.f ? 0.f : y / sum);
    }
}

template <typename T>
static void launch_tree(const char* name, const TreeArgs& a, int dim) {
    const dim3 grid((unsigned)a.g.rows, (unsigned)a.heads);
    switch (dim) {
        case 32: return launch(name, kv_tree_k<T, 32>, grid, dim3(256), 0, a);
        case 64: return launch(name, kv_tree_k<T, 64>, grid, dim3(256), 0, a);
        case 128: return launch(name, kv_tree_k<T, 128>, grid, dim3(256), 0, a);
        default: return launch(name, kv_tree_k<T, 256>, grid, dim3(256), 0, a);
    }
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
    const int longest = max_length > 0 && max_length < capacity ? max_length : capacity;
    TreeArgs a{c.ragged, c.k, c.v, c.k_scale, c.v_scale, (const int*)tree->data, q->data, out->data, ld, q_col, heads, c.kv_heads,
               group, window_of(window, capacity), (int)tree->shape[1], scale * 1.44269504088896340736f};
    a.g.rows = (int)rows;
    const int64_t reach = a.window > 0 ? (int64_t)a.window - 1 + ceil_div(rows, c.ragged.batch) : longest;
    set_work(0.0, 2.0 * c.kv_heads * c.dim * (double)(reach < longest ? reach : longest) * c.ragged.batch);
    if (q->dtype == NNC_DTYPE_FLOAT16)
        launch_tree<half_t>(name, a, c.dim);
    else
        launch_tree<float>(name, a, c.dim);
}

}  // extern "C"
