// What a model answers with: log probabilities of given tokens, the entropy and
// the likeliest tokens of rows of logits (nnc_hip_token_logprobs). No reference
// counterpart.
//
//   m = max_i x_i,  S = sum_i e^(t (x_i - m));  log p_i = t (x_i - m) - log S
//   entropy = log S - sum_i t (x_i - m) e^(t (x_i - m)) / S
//
// The sums are float64: a row's largest term is 1, and where it leaves 2^-24
// and less to all others, entropy and the largest token's log probability are
// made of those.
#include "quant8.h"

namespace nnc {

struct LogprobArgs {
    const void* logits;
    const int* tokens;
    float *logprob, *entropy;
    int* top_index;
    float* top_logprob;
    int64_t rows, vocab;
    int top;
    float scale;
};

// Whole numbers ordered as the values are, the earlier of equal ones first: a
// value's bits, negative ones turned round, before the index's complement.
__device__ __forceinline__ uint64_t rank_of(float x, uint32_t index) {
    const uint32_t bits = __float_as_uint(x + 0.f);  // (-0 becomes 0)
    return (uint64_t)(bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(uint64_t rank) {
    const uint32_t u = (uint32_t)(rank >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int index_of(uint64_t rank) { return (int)(0xffffffffu - (uint32_t)rank); }

template <typename V, class Op>
__device__ __forceinline__ V block_reduce(V v, V (&part)[4], Op op) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return op(op(part[0], part[1]), op(part[2], part[3]));
}

// A workgroup to a row, which it reads for the maximum, for the sums, and once
// for each alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprobs_k(LogprobArgs a) {
    __shared__ float fpart[4];
    __shared__ double dpart[4];
    __shared__ unsigned long long upart[4];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.logits + row * a.vocab;
        float m = -INFINITY;
        for (int64_t i = threadIdx.x; i < a.vocab; i += 256) m = max_nan(m, (float)x[i]);
        m = block_reduce(m, fpart, [](float p, float q) { return max_nan(p, q); });
        const bool ok = fabsf(m) < INFINITY;
        double sum = 0.0, weighted = 0.0;
        for (int64_t i = threadIdx.x; i < a.vocab; i += 256) {
            const float d = a.scale * ((float)x[i] - m), e = expf(d);
            sum += e;
            if (e > 0.f) weighted += d * e;
        }
        auto add = [](double p, double q) { return p + q; };
        sum = block_reduce(sum, dpart, add);
        weighted = block_reduce(weighted, dpart, add);
        const double log_sum = log(sum);
        auto log_p = [&](float v) { return (float)((double)a.scale * ((double)v - (double)m) - log_sum); };
        if (threadIdx.x == 0) {
            if (a.entropy) a.entropy[row] = ok ? (float)(log_sum - weighted / sum) : NAN;
            if (a.logprob) {
                const int t = a.tokens[row];
                a.logprob[row] = ok && t >= 0 && t < a.vocab ? log_p((float)x[t]) : NAN;
            }
        }
        unsigned long long last = ~0ull;
        for (int n = 0; n < a.top; ++n) {
            unsigned long long best = 0;
            for (int64_t i = threadIdx.x; ok && i < a.vocab; i += 256) {
                const unsigned long long r = rank_of((float)x[i], (uint32_t)i);
                if (r < last && r > best) best = r;
            }
            last = block_reduce(best, upart, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
            if (threadIdx.x == 0) {
                a.top_index[row * a.top + n] = last ? index_of(last) : -1;
                a.top_logprob[row * a.top + n] = last ? log_p(value_of(last)) : ok ? -INFINITY : NAN;
            }
        }
    }
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
    const int64_t most = (int64_t)cu_count() * 8;
    const dim3 grid((unsigned)(a.rows < most ? a.rows : most));
    if (logits->dtype == NNC_DTYPE_FLOAT16)
        launch(name, logprobs_k<half_t>, grid, dim3(256), 0, a);
    else
        launch(name, logprobs_k<float>, grid, dim3(256), 0, a);
}

}  // extern "C"
