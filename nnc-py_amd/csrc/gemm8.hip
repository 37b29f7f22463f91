// Matrix product of 8-bit integers (nnc_hip_matmul_i8): activations a
// [M][K] with a scale for each row, weights w [N][K] with a scale for each
// row,
//   out[m][n] = (sum_k a[m][k] w[n][k]) * (a_scale[m] * w_scale[n]) + bias[n].
// The sum is exact (32-bit integers: K up to 131071); the scales, the bias
// and the output's rounding follow in 32 bits. No reference counterpart.
//
// v_mfma_i32_16x16x64_i8: lane (i = lane % 16, g = lane / 16) holds 16 k of
// row i of either operand; the k order is the same in both, so it does not
// matter which 16 of the 64 a lane group has. Result register r is row
// 4g + r, column i.
#include "mfma_tile.h"
#include "quant8.h"

namespace nnc {

struct Gemm8Args {
    const int8_t* a;
    const int8_t* w;
    const float* as;
    const float* ws;
    const float* bias;
    void* out;
    int64_t m, n;
    int k;
    bool vec_out;  // output rows start on 16 bytes
};

// 16 consecutive k of a row from k on, zeros behind its end; K >= 1, any
// alignment. The last chunk is read as the row's last 16 bytes and shifted,
// so that nothing behind the matrix is touched.
typedef ix4 ix4_any __attribute__((aligned(1)));
__device__ __forceinline__ ix4 row_chunk(const int8_t* row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const ix4_any*>(row + k);
    if (k >= K) return ix4{0, 0, 0, 0};
    unsigned __int128 v = 0;
    if (K >= 16) {
        const ix4 last = *reinterpret_cast<const ix4_any*>(row + K - 16);
        v = __builtin_bit_cast(unsigned __int128, last) >> (8 * (k + 16 - K));
    } else {
        for (int i = K - 1; i >= k; --i) v = v << 8 | (uint8_t)row[i];
    }
    return __builtin_bit_cast(ix4, v);
}

// ---------------------------------------------------------------------------
// Tiles: BM x BN outputs per workgroup, WM x WN waves, 128 k at a time, two LDS
// stages: the loads of slice t + 1 are in flight while slice t is used. DMA:
// straight from global memory into LDS, 16 bytes per lane. That needs K % 16
// == 0 and 16-byte aligned operands: a chunk is wholly inside or outside the
// matrix, and one outside gets an offset past the buffer (zeros). Without it
// the chunks go through registers (row_chunk).
// An LDS row is 128 k of one row of a or w, its 16-byte chunk c at position
// c ^ (row % 8), so that eight lanes reading a chunk of eight rows hit all
// banks. w's rows are the MFMA's first operand: a lane then holds four
// consecutive columns of one output row.
// ---------------------------------------------------------------------------
typedef int ix16 __attribute__((ext_vector_type(16)));

template <int BM_, int BN_, int WM_, int WN_>
struct Tile8 {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM * WN, THREADS = 64 * NW;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 blocks per wave
    static constexpr int STAGE = (BM + BN) * 128;
    static constexpr int LOADS_A = BM / (8 * NW), LOADS_W = BN / (8 * NW);  // instructions per wave and slice
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM >= 1 && TN >= 1, "rows split evenly over the waves");
    // the epilogue's 32 rows of a wave, padded to 16 bytes off a multiple of 128
    static constexpr int WAVE_N = 32 * TN;
    template <typename T>
    static constexpr int out_ld() { return WAVE_N * (int)sizeof(T) + 16; }
    static constexpr int LDS = 2 * STAGE > NW * 32 * out_ld<float>() ? 2 * STAGE : NW * 32 * out_ld<float>();
};

// the tile of a workgroup: bands of 8 tile rows, column by column, eight
// consecutive workgroups' worth of them on one XCD, so that the operands'
// slices are shared through its L2
__device__ __forceinline__ void tile8_pos(int wg, int tiles_m, int tiles_n, int& mt, int& nt) {
    const int t = xcd_remap(wg, tiles_m * tiles_n);
    const int band = t / (8 * tiles_n), in = t - band * 8 * tiles_n, rows = min(8, tiles_m - band * 8);
    nt = in / rows;
    mt = band * 8 + in - nt * rows;
}

template <class L, typename T, bool DMA>
__global__ void __launch_bounds__(L::THREADS) gemm8_tile_k(Gemm8Args p, int tiles_m, int tiles_n) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / L::WN, wn = wave % L::WN;
    int mt, nt;
    tile8_pos(blockIdx.x, tiles_m, tiles_n, mt, nt);
    const int64_t m0 = (int64_t)mt * L::BM, n0 = (int64_t)nt * L::BN;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc((const float*)(p.a + m0 * p.k)), rw = make_rsrc((const float*)(p.w + n0 * p.k));
    // this lane's rows and chunk of the loads
    const int kc = ((lane & 7) ^ (lane >> 3)) * 16;
    uint32_t va[L::LOADS_A], vw[L::LOADS_W];
#pragma unroll
    for (int i = 0; i < L::LOADS_A; ++i) {
        const int r = (wave + L::NW * i) * 8 + (lane >> 3);
        va[i] = DMA ? keep_or_oob((uint32_t)(r * p.k + kc), m0 + r < p.m) : (uint32_t)(m0 + r < p.m ? r : (int)(p.m - 1 - m0)) * p.k;
    }
#pragma unroll
    for (int i = 0; i < L::LOADS_W; ++i) {
        const int r = (wave + L::NW * i) * 8 + (lane >> 3);
        vw[i] = DMA ? keep_or_oob((uint32_t)(r * p.k + kc), n0 + r < p.n) : (uint32_t)(n0 + r < p.n ? r : (int)(p.n - 1 - n0)) * p.k;
    }
    ix4 staged[DMA ? 1 : L::LOADS_A + L::LOADS_W];
    auto issue = [&](int stage, int k0) {
        if constexpr (DMA) {
            char* s = lds + stage * L::STAGE;
            const bool in = k0 + kc < p.k;
#pragma unroll
            for (int i = 0; i < L::LOADS_A; ++i)
                dma_load16(ra, (float*)(s + (wave + L::NW * i) * 1024), in ? va[i] : kOutOfRange, (uint32_t)k0);
#pragma unroll
            for (int i = 0; i < L::LOADS_W; ++i)
                dma_load16(rw, (float*)(s + L::BM * 128 + (wave + L::NW * i) * 1024), in ? vw[i] : kOutOfRange, (uint32_t)k0);
        } else {
            (void)stage;
#pragma unroll
            for (int i = 0; i < L::LOADS_A; ++i) staged[i] = row_chunk(p.a + m0 * p.k + va[i], k0 + kc, p.k);
#pragma unroll
            for (int i = 0; i < L::LOADS_W; ++i) staged[L::LOADS_A + i] = row_chunk(p.w + n0 * p.k + vw[i], k0 + kc, p.k);
        }
    };
    auto land = [&](int stage) {
        if constexpr (!DMA) {
            char* s = lds + stage * L::STAGE;
#pragma unroll
            for (int i = 0; i < L::LOADS_A; ++i) *reinterpret_cast<ix4*>(s + (wave + L::NW * i) * 1024 + lane * 16) = staged[i];
#pragma unroll
            for (int i = 0; i < L::LOADS_W; ++i)
                *reinterpret_cast<ix4*>(s + L::BM * 128 + (wave + L::NW * i) * 1024 + lane * 16) = staged[L::LOADS_A + i];
        }
    };
    ix16 acc[L::TM][L::TN];
#pragma unroll
    for (int i = 0; i < L::TM; ++i)
#pragma unroll
        for (int j = 0; j < L::TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int ra0 = (wm * 32 * L::TM + l32) * 128, rw0 = L::BM * 128 + (wn * L::WAVE_N + l32) * 128;
    issue(0, 0);
    land(0);
    int stage = 0;
    for (int k0 = 0; k0 < p.k; k0 += 128, stage ^= 1) {
        if constexpr (DMA)
            dma_barrier<0>();  // this slice has landed, the other stage is no longer read
        else
            __syncthreads();
        if (k0 + 128 < p.k) issue(stage ^ 1, k0 + 128);
        const char* s = lds + stage * L::STAGE;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const int c = ((2 * st + half) ^ (lane & 7)) * 16;
            ix4 x[L::TM], y[L::TN];
#pragma unroll
            for (int j = 0; j < L::TN; ++j) y[j] = *reinterpret_cast<const ix4*>(s + rw0 + j * 4096 + c);
#pragma unroll
            for (int i = 0; i < L::TM; ++i) x[i] = *reinterpret_cast<const ix4*>(s + ra0 + i * 4096 + c);
#pragma unroll
            for (int i = 0; i < L::TM; ++i)
#pragma unroll
                for (int j = 0; j < L::TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(y[j], x[i], acc[i][j], 0, 0, 0);
        }
        if (k0 + 128 < p.k) land(stage ^ 1);
    }
    dma_barrier<0>();  // every wave is done with the stages
    // scaled and rounded 32 rows at a time through this wave's part of LDS, to
    // whole 16-byte stores where rows start on 16 bytes
    constexpr int LD = L::template out_ld<T>(), PER = 16 / (int)sizeof(T), LANES = L::WAVE_N / PER;
    char* mine = lds + wave * 32 * L::template out_ld<float>();
    const int64_t nw = n0 + wn * L::WAVE_N;
#pragma unroll
    for (int i = 0; i < L::TM; ++i) {
        const int64_t mb = m0 + (wm * L::TM + i) * 32;
        const float sm = mb + l32 < p.m ? p.as[mb + l32] : 0.f;
#pragma unroll
        for (int j = 0; j < L::TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 32 * j + 8 * q + 4 * half;
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t n = nw + c + r < p.n ? nw + c + r : p.n - 1;
                    const float b = p.bias ? p.bias[n] : 0.f;
                    const int sum = acc[i][j][4 * q + r];
                    v[r] = (T)fmaf((float)sum, sm * p.ws[n], b);
                }
                __builtin_memcpy(__builtin_assume_aligned(mine + l32 * LD + c * sizeof(T), 4 * sizeof(T)), v, sizeof v);
            }
        __builtin_amdgcn_wave_barrier();
        if (p.vec_out) {
#pragma unroll
            for (int e = 0; e < 32; e += 64 / LANES) {
                const int r = e + lane / LANES, c = (lane % LANES) * PER;
                const ix4 v = *reinterpret_cast<const ix4*>(mine + r * LD + c * sizeof(T));
                if (mb + r < p.m && nw + c < p.n) *reinterpret_cast<ix4*>((T*)p.out + (mb + r) * p.n + nw + c) = v;
            }
        } else {
            for (int e = lane; e < 32 * L::WAVE_N; e += 64) {
                const int r = e / L::WAVE_N, c = e % L::WAVE_N;
                if (mb + r < p.m && nw + c < p.n) ((T*)p.out)[(mb + r) * p.n + nw + c] = *reinterpret_cast<const T*>(mine + r * LD + c * sizeof(T));
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <class L, typename T, bool DMA>
static void launch_tile8(const char* name, const Gemm8Args& p) {
    auto kernel = gemm8_tile_k<L, T, DMA>;
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::LDS) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    const int64_t tm = ceil_div(p.m, L::BM), tn = ceil_div(p.n, L::BN);
    launch(name, kernel, dim3((unsigned)(tm * tn)), dim3(L::THREADS), L::LDS, p, (int)tm, (int)tn);
}

// ---------------------------------------------------------------------------
// Few rows of a: every weight is read once, straight into registers, and that
// is all the time there is. A workgroup takes 16 rows of w and up to 16 MT
// rows of a, its waves 256 k each in turn; lane (i, g) reads the 64
// consecutive k from 64 g of its row (whole cache lines per row), 16 of them
// for each MFMA. The waves' sums, whole numbers, are joined through LDS.
// ---------------------------------------------------------------------------
template <int MT, int NW, typename T, bool ALIGNED>
__global__ void __launch_bounds__(64 * NW) gemm8_rows_k(Gemm8Args p) {
    __shared__ int part[NW][MT][16][17];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
    const int8_t* w = p.w + min(n0 + i, p.n - 1) * p.k;
    const int8_t* a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = p.a + min(m0 + 16 * t + i, p.m - 1) * p.k;
    ix4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = ix4{0, 0, 0, 0};
    auto chunk = [&](const int8_t* row, int k) {
        if constexpr (ALIGNED)
            return k < p.k ? *reinterpret_cast<const ix4*>(row + k) : ix4{0, 0, 0, 0};
        else
            return row_chunk(row, k, p.k);
    };
    for (int k0 = wave * 256 + g * 64; k0 - g * 64 < p.k; k0 += NW * 256) {
        ix4 y[4], x[MT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = chunk(w, k0 + 16 * j);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[t][j] = chunk(a[t], k0 + 16 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[j], x[t][j], acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int v = acc[t][r];
            part[wave][t][i][4 * g + r] = v;
        }
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 256; e += 64 * NW) {
        const int t = e >> 8, m = (e >> 4) & 15, n = e & 15;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < NW; ++v) sum += part[v][t][m][n];
        const int64_t row = m0 + 16 * t + m, col = n0 + n;
        if (row < p.m && col < p.n)
            ((T*)p.out)[row * p.n + col] = (T)fmaf((float)sum, p.as[row] * p.ws[col], p.bias ? p.bias[col] : 0.f);
    }
}

template <int MT, int NW, typename T>
static void launch_rows8(const char* name, const Gemm8Args& p, bool aligned) {
    const dim3 grid((unsigned)ceil_div(p.n, 16), (unsigned)ceil_div(p.m, 16 * MT));
    if (aligned)
        launch(name, gemm8_rows_k<MT, NW, T, true>, grid, dim3(64 * NW), 0, p);
    else
        launch(name, gemm8_rows_k<MT, NW, T, false>, grid, dim3(64 * NW), 0, p);
}

template <typename T>
static void launch_gemm8(const char* name, const Gemm8Args& p) {
    const bool chunks = p.k % 16 == 0 && aligned16(p.a) && aligned16(p.w);
    if (p.m <= 16) return launch_rows8<1, 16, T>(name, p, chunks);
    if (p.m <= 32) return launch_rows8<2, 16, T>(name, p, chunks);
    if (p.m <= 64) return launch_rows8<4, 8, T>(name, p, chunks);
    if (!chunks) {
        if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= cu_count()) return launch_tile8<Tile8<128, 128, 2, 2>, T, false>(name, p);
        return launch_tile8<Tile8<64, 64, 2, 2>, T, false>(name, p);
    }
    if (ceil_div(p.m, 256) * ceil_div(p.n, 256) >= cu_count()) return launch_tile8<Tile8<256, 256, 2, 4>, T, true>(name, p);
    if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= cu_count()) return launch_tile8<Tile8<128, 128, 2, 2>, T, true>(name, p);
    return launch_tile8<Tile8<64, 64, 2, 2>, T, true>(name, p);
}

}  // namespace nnc

using namespace nnc;

extern "C" {

void nnc_hip_matmul_i8(Tensor* a, Tensor* a_scale, Tensor* w, Tensor* w_scale, Tensor* bias, Tensor* out) {
    const char* name = "nnc_hip_matmul_i8";
    if (!has_data(a) || !has_data(a_scale) || !has_data(w) || !has_data(w_scale) || !has_data(out) ||
        (bias && !has_data(bias)))
        return fail(NNC_HIP_EINVAL, name, "NULL tensor or data");
    if (a->dtype != NNC_DTYPE_INT8 || w->dtype != NNC_DTYPE_INT8) return fail(NNC_HIP_EUNSUPP, name, "int8 operands only");
    if (a_scale->dtype != NNC_DTYPE_FLOAT32 || w_scale->dtype != NNC_DTYPE_FLOAT32 ||
        (bias && bias->dtype != NNC_DTYPE_FLOAT32))
        return fail(NNC_HIP_EUNSUPP, name, "float32 scales and bias only");
    if (!is_activation(out)) return fail(NNC_HIP_EUNSUPP, name, "float32 or float16 output only");
    if (!good_shape(a) || !good_shape(out) || !good_shape(w) || w->ndim != 2)
        return fail(NNC_HIP_EINVAL, name, "w must be [N][K]");
    const int64_t k = a->shape[a->ndim - 1], n = w->shape[0];
    if (w->shape[1] != k) return fail(NNC_HIP_EINVAL, name, "rows of %lld and %lld", (long long)k, (long long)w->shape[1]);
    if (out->shape[out->ndim - 1] != n) return fail(NNC_HIP_EINVAL, name, "output rows of %lld, not %lld",
                                                    (long long)out->shape[out->ndim - 1], (long long)n);
    const int64_t m = prod(a->shape, 0, a->ndim - 1);
    if (prod(out->shape, 0, out->ndim - 1) != m || numel(a_scale) != m || numel(w_scale) != n || (bias && numel(bias) != n))
        return fail(NNC_HIP_EINVAL, name, "a_scale and out need %lld rows, w_scale and bias %lld", (long long)m, (long long)n);
    if (m == 0 || n == 0) return;
    if (k < 1 || k > 131071) return fail(NNC_HIP_EUNSUPP, name, "K = %lld (1 to 131071)", (long long)k);
    if (m > (int64_t)65535 * 64 || n > (int64_t)1 << 30) return fail(NNC_HIP_EUNSUPP, name, "too many rows");
    if (!ready(name)) return;
    Gemm8Args p{(const int8_t*)a->data, (const int8_t*)w->data, (const float*)a_scale->data, (const float*)w_scale->data,
                bias ? (const float*)bias->data : nullptr, out->data, m, n, (int)k,
                aligned16(out->data) && n * activation_bytes(out) % 16 == 0};
    set_work(2.0 * m * n * k, (double)m * k + (double)n * k + (double)m * n * activation_bytes(out));
    if (out->dtype == NNC_DTYPE_FLOAT16)
        launch_gemm8<half_t>(name, p);
    else
        launch_gemm8<float>(name, p);
}

}  // extern "C"
