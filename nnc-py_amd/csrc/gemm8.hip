// Matrix product of 8-bit integers (nnc_hip_matmul_i8): activations a
// [M][K] with a scale for each row, weights w [N][K] with a scale for each
// row,
//   out[m][n] = (sum_k a[m][k] w[n][k]) * (a_scale[m] * w_scale[n]) + bias[n].
// The sum is exact (32-bit integers: K up to 131071); the scales, the bias
// and the output's rounding follow in 32 bits. No reference counterpart.
//
// [8192,4096]x[4096,4096] to f16 130 to 135 us from card to card, 2.04 to 2.11
// POPS (a library's product of the same operands to 32-bit integers 133 us on
// one of them); 8 rows 6.0 us, of which the weights' 16.8 MB are 3.2 at a
// copy's rate.
//
// v_mfma_i32_16x16x64_i8 (few rows): lane (i = lane % 16, g = lane / 16) holds
// 16 k of row i of either operand; the k order is the same in both, so it does
// not matter which 16 of the 64 a lane group has. Result register r is row
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
// Tiles: BM x BN outputs per workgroup, WM x WN waves, 128 k at a time.
//
// Slices go straight from global memory into NS LDS stages, 16 bytes per lane,
// NS - 1 of them in flight. That needs K % 16 == 0 and 16-byte aligned
// operands: a chunk is wholly inside or outside the matrix, and one outside
// gets an offset past the buffer (zeros). Other operands are laid out so
// first (pack8_k): chunks through registers instead took 107 us for
// [2048,4001]x[4096,4001], 96 with 128 x 128 tiles, unaligned loads being
// split up; with the layout 54.
//
// An LDS row is 128 k of one row of a or w, its 16-byte chunk c at position
// c ^ (row / 2 % 8): LDS has 64 banks, and 16 lanes reading a chunk of 16 rows
// hit all of them (c ^ (row % 8) has two rows on the same banks: half of all
// LDS cycles were conflicts). w's rows are the MFMA's first operand: a lane then holds four
// consecutive columns of one output row. The operands of a slice's four steps
// are read one step ahead of their MFMAs; the barrier between two slices
// comes before the last step's MFMAs, which cover the next slice's first read.
//
// splits > 1: the k of a tile are divided over so many workgroups, and the
// last to finish adds the others' sums (whole numbers: in any order).
// ---------------------------------------------------------------------------
typedef int ix16 __attribute__((ext_vector_type(16)));

template <int BM_, int BN_, int WM_, int WN_, int NS_, int PF_>
struct Tile8 {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, PF = PF_, NW = WM * WN, THREADS = 64 * NW;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 blocks per wave
    static constexpr int STAGE = (BM + BN) * 128;
    static constexpr int LOADS_A = BM / (8 * NW), LOADS_W = BN / (8 * NW);  // instructions per wave and slice
    static constexpr int LOADS = LOADS_A + LOADS_W;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM >= 1 && TN >= 1, "rows split evenly over the waves");
    static_assert(NW % 2 == 0, "a lane's chunk is the same in all its loads");
    // the epilogue's 32 rows of a wave, 16 bytes off a multiple of 128
    static constexpr int WAVE_N = 32 * TN;
    template <typename T>
    static constexpr int out_ld() { return WAVE_N * (int)sizeof(T) + 16; }
    static constexpr int OUT = NW * 32 * out_ld<float>();
    static constexpr int LDS = NS * STAGE > OUT ? NS * STAGE : OUT;
};

struct Split8 {
    int tiles_m, tiles_n, splits, each;  // each: k of a split, a multiple of 128
    int* sums;                           // [tile][split][BM * BN]
    int* counters;                       // [tile], zero
};

// The tile of a workgroup: bands of 8 tile rows, column by column, so that the
// workgroups of one XCD share slices of both operands through its L2.
__device__ __forceinline__ void tile8_pos(int t, const Split8& s, int& mt, int& nt) {
    const int band = t / (8 * s.tiles_n), in = t - band * 8 * s.tiles_n, rows = min(8, s.tiles_m - band * 8);
    nt = in / rows;
    mt = band * 8 + in - nt * rows;
}

template <class L, typename T>
__global__ void __launch_bounds__(L::THREADS) gemm8_tile_k(Gemm8Args p, Split8 sp) {
    extern __shared__ __align__(16) char lds[];
    constexpr int NS = L::NS, PF = L::PF;
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / L::WN, wn = wave % L::WN;
    const int tiles = sp.tiles_m * sp.tiles_n, wg = xcd_remap(blockIdx.x, tiles * sp.splits);
    const int split = wg / tiles, tile = wg - split * tiles;
    int mt, nt;
    tile8_pos(tile, sp, mt, nt);
    const int64_t m0 = (int64_t)mt * L::BM, n0 = (int64_t)nt * L::BN;
    const int kfrom = split * sp.each, kto = min(p.k, kfrom + sp.each), slices = (kto - kfrom + 127) / 128;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc((const float*)(p.a + m0 * p.k)), rw = make_rsrc((const float*)(p.w + n0 * p.k));
    // this lane's rows and chunk of the loads
    const int kc = ((lane & 7) ^ ((4 * wave + (lane >> 4)) & 7)) * 16;  // rows 8 wave + lane / 8 (mod 16)
    uint32_t va[L::LOADS_A], vw[L::LOADS_W];
#pragma unroll
    for (int i = 0; i < L::LOADS_A; ++i) {
        const int r = (wave + L::NW * i) * 8 + (lane >> 3);
        va[i] = keep_or_oob((uint32_t)(r * p.k + kc), m0 + r < p.m);
    }
#pragma unroll
    for (int i = 0; i < L::LOADS_W; ++i) {
        const int r = (wave + L::NW * i) * 8 + (lane >> 3);
        vw[i] = keep_or_oob((uint32_t)(r * p.k + kc), n0 + r < p.n);
    }
    // slice t's loads: as many in every call, so that they can be counted
    auto issue = [&](int t) {
        const int k0 = kfrom + t * 128;
        char* s = lds + t % NS * L::STAGE;
        const bool in = k0 + kc < kto;
#pragma unroll
        for (int i = 0; i < L::LOADS_A; ++i)
            dma_load16(ra, (float*)(s + (wave + L::NW * i) * 1024), in ? va[i] : kOutOfRange, (uint32_t)k0);
#pragma unroll
        for (int i = 0; i < L::LOADS_W; ++i)
            dma_load16(rw, (float*)(s + L::BM * 128 + (wave + L::NW * i) * 1024), in ? vw[i] : kOutOfRange, (uint32_t)k0);
    };
    ix16 acc[L::TM][L::TN];
#pragma unroll
    for (int i = 0; i < L::TM; ++i)
#pragma unroll
        for (int j = 0; j < L::TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int ra0 = (wm * 32 * L::TM + l32) * 128, rw0 = L::BM * 128 + (wn * L::WAVE_N + l32) * 128;
    ix4 x[2][PF][L::TM], y[2][PF][L::TN];
    // steps st .. st + PF of slice t into register set `set`
    auto read = [&](int t, int st, int set) {
#pragma unroll
        for (int u = 0; u < PF; ++u) {
            const char* s = lds + t % NS * L::STAGE + ((2 * (st + u) + half) ^ ((l32 >> 1) & 7)) * 16;
#pragma unroll
            for (int j = 0; j < L::TN; ++j) y[set][u][j] = *reinterpret_cast<const ix4*>(s + rw0 + j * 4096);
#pragma unroll
            for (int i = 0; i < L::TM; ++i) x[set][u][i] = *reinterpret_cast<const ix4*>(s + ra0 + i * 4096);
        }
        __builtin_amdgcn_sched_barrier(0);  // before the MFMAs that cover it
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int u = 0; u < PF; ++u)
#pragma unroll
            for (int i = 0; i < L::TM; ++i)
#pragma unroll
                for (int j = 0; j < L::TN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(y[set][u][j], x[set][u][i], acc[i][j], 0, 0, 0);
    };
    constexpr int READS = 4 / PF;  // of a slice
    auto slice = [&](int t, int par) {
#pragma unroll
        for (int n = 0; n + 1 < READS; ++n) {
            read(t, (n + 1) * PF, (par * READS + n + 1) & 1);
            multiply((par * READS + n) & 1);
        }
        if (t + 1 < slices) {
            dma_barrier<(NS - 2) * L::LOADS>();  // slice t + 1 has landed, slice t's stage is no longer read
            issue(t + NS);
            read(t + 1, 0, (par * READS + READS) & 1);
        }
        multiply((par * READS + READS - 1) & 1);
    };
#pragma unroll
    for (int t = 0; t < NS - 1; ++t) issue(t);
    dma_barrier<(NS - 2) * L::LOADS>();
    issue(NS - 1);
    read(0, 0, 0);
    int t = 0;
    for (; t + 1 < slices; t += 2) {
        slice(t, 0);
        slice(t + 1, 1);
    }
    if (t < slices) slice(t, 0);

    if (sp.splits > 1) {
        int* mine = sp.sums + (int64_t)tile * sp.splits * (L::BM * L::BN);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc((const float*)mine);
        const uint32_t at = (uint32_t)((wave * L::TM * L::TN * 4 * 64 + lane) * 16);
        constexpr uint32_t SLOT = L::BM * L::BN * 4;
#pragma unroll
        for (int i = 0; i < L::TM; ++i)
#pragma unroll
            for (int j = 0; j < L::TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int v0 = acc[i][j][4 * q], v1 = acc[i][j][4 * q + 1], v2 = acc[i][j][4 * q + 2], v3 = acc[i][j][4 * q + 3];
                    typedef unsigned ux4 __attribute__((ext_vector_type(4)));
                    __builtin_amdgcn_raw_buffer_store_b128(ux4{(unsigned)v0, (unsigned)v1, (unsigned)v2, (unsigned)v3}, rs,
                                                           (int)(at + split * SLOT + ((i * L::TN + j) * 4 + q) * 1024), 0, kDeviceScope);
                }
        if (!finish_arrive(sp.counters + tile, sp.splits - 1)) return;
        // all splits' sums, this one's too: their loads go out together
#pragma unroll
        for (int i = 0; i < L::TM; ++i)
#pragma unroll
            for (int j = 0; j < L::TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
#pragma unroll 4
        for (int o = 0; o < sp.splits; ++o) {
#pragma unroll
            for (int i = 0; i < L::TM; ++i)
#pragma unroll
                for (int j = 0; j < L::TN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const ix4 v = __builtin_bit_cast(ix4, load_partial4(rs, at + o * SLOT + ((i * L::TN + j) * 4 + q) * 1024));
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int e = v[r];
                            acc[i][j][4 * q + r] += e;
                        }
                    }
        }
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

// One operand or both with rows of k16 = K rounded up to 16, zeros behind K.
struct Pack8Args {
    const int8_t* from[2];
    int8_t* to[2];
    int64_t rows[2];
    int k, k16;
};
__global__ void __launch_bounds__(256) pack8_k(Pack8Args p) {
    const int chunks = p.k16 / 16;
    const int64_t first = p.rows[0] * chunks, all = first + p.rows[1] * chunks;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (int64_t)gridDim.x * 256) {
        const int which = e >= first;
        const int64_t at = which ? e - first : e, row = at / chunks;
        const int c = (int)(at - row * chunks) * 16;
        const ix4 v = row_chunk(p.from[which] + row * p.k, c, p.k);
        *reinterpret_cast<ix4*>(p.to[which] + row * p.k16 + c) = v;
    }
}

// The operation's work, for the launch that does it (an operand laid out again
// first is a launch of its own, with its bytes).
static void set_product_work(const Gemm8Args& p, size_t out_bytes) {
    set_work(2.0 * p.m * p.n * p.k, (double)p.m * p.k + (double)p.n * p.k + (double)p.m * p.n * out_bytes);
}

template <class L, typename T>
static void launch_tile8(const char* name, Gemm8Args p, int splits) {
    auto kernel = gemm8_tile_k<L, T>;
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::LDS) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    const int64_t tm = ceil_div(p.m, L::BM), tn = ceil_div(p.n, L::BN);
    const int slices = (int)ceil_div(p.k, 128), each = (int)ceil_div(slices, splits);
    Split8 sp{(int)tm, (int)tn, (int)ceil_div(slices, each), each * 128, nullptr, nullptr};
    // workspace: operands laid out again, partial sums
    const int k16 = (int)ceil_div(p.k, 16) * 16;
    const bool pack_a = p.k != k16 || !aligned16(p.a), pack_w = p.k != k16 || !aligned16(p.w);
    const size_t sums = sp.splits > 1 ? (size_t)(tm * tn) * sp.splits * L::BM * L::BN * sizeof(int) : 0;
    const size_t bytes = sums + (pack_a ? (size_t)p.m * k16 : 0) + (pack_w ? (size_t)p.n * k16 : 0);
    if (bytes > 0) {
        char* ws = (char*)workspace(bytes);
        sp.counters = sums ? tile_counters((size_t)(tm * tn)) : nullptr;
        if (!ws || (sums && !sp.counters)) return fail(NNC_HIP_ENOMEM, name, "no workspace for %zu bytes", bytes);
        sp.sums = (int*)ws;
        ws += sums;
        if (pack_a || pack_w) {
            Pack8Args q{{p.a, p.w}, {(int8_t*)ws, (int8_t*)ws + (pack_a ? p.m * k16 : 0)}, {pack_a ? p.m : 0, pack_w ? p.n : 0}, p.k, k16};
            set_work(0.0, (double)(q.rows[0] + q.rows[1]) * (p.k + k16));
            launch("nnc_hip_matmul_i8_pack", pack8_k, dim3(grid_for((q.rows[0] + q.rows[1]) * (k16 / 16), 1)), dim3(256), 0, q);
            if (pack_a) p.a = q.to[0];
            if (pack_w) p.w = q.to[1];
        }
    }
    set_product_work(p, sizeof(T));
    if (pack_a || pack_w) p.k = k16;
    launch(name, kernel, dim3((unsigned)(tm * tn * sp.splits)), dim3(L::THREADS), L::LDS, p, sp);
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
    for (int t = 0; t < MT; ++t) a[t] = m0 + 16 * t + i < p.m ? p.a + (m0 + 16 * t + i) * p.k : nullptr;  // no row: no loads
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
            for (int j = 0; j < 4; ++j) x[t][j] = a[t] ? chunk(a[t], k0 + 16 * j) : ix4{0, 0, 0, 0};
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
    set_product_work(p, sizeof(T));
    if (aligned)
        launch(name, gemm8_rows_k<MT, NW, T, true>, grid, dim3(64 * NW), 0, p);
    else
        launch(name, gemm8_rows_k<MT, NW, T, false>, grid, dim3(64 * NW), 0, p);
}

// Which kernel: the one whose time, in us past the launch, is least by what was
// measured (256 CUs, K 1024 to 14336, M 1 to 8192, N 1001 to 4096). A row
// kernel reads (16 + rows) K bytes per workgroup, all together at 9.8 TB/s and
// one workgroup at 40 GB/s. A tile kernel takes so long for each slice and
// round of workgroups; joining splits costs 1.5 us and 16 ns for every partial
// tile written and read back; laying operands out for the tiles costs a launch
// and their bytes. Against the neighbours, us: [64,4096]x[4096,4096] rows
// 12.2, 64 x 64 tiles 10.6, in two splits 9.6; [64,14336]x[4096,14336] rows
// 34.4, tiles 27.9, in four splits 14.7; [512,4096]x[4096,4096] tiles of 64 16.2
// (14.4 by the rule), 128 19.1; [1024,4096]x[4096,4096] tiles of 64 31.9, 128 24.3, 256 x 128 30.1,
// 256 47.9; with 8192 rows 227, 179, 154 and 130 (the matrix units busy 61% of
// the cycles, the rest waits for the next slice: one workgroup per CU, two
// stages).
struct Plan8 {
    int kernel = 0, splits = 1;
    double us = 1e30;
    void offer(int k, int s, double t) {
        if (t < us) kernel = k, splits = s, us = t;
    }
};

static Plan8 plan_gemm8(int64_t m, int64_t n, int64_t k, bool aligned) {
    Plan8 best;
    const double cus = cu_count(), slices = (double)ceil_div(k, 128);
    // laying the operands out for the tile kernels: a launch, and their bytes
    const double pack = aligned ? 0.0 : 2.5 + (double)(m + n) * k / 2e6;
    for (int mt : {1, 2, 4}) {
        if (m > 128) break;
        const int64_t rows = m < 16 * mt ? m : 16 * mt;
        const double each = (16.0 + rows) * k, all = each * ceil_div(n, 16) * ceil_div(m, 16 * mt);
        best.offer(mt, 1, all / 9.8e6 > each / 40e3 ? all / 9.8e6 : each / 40e3);
    }
    const int64_t tiles64 = ceil_div(m, 64) * ceil_div(n, 64);
    for (int s : {1, 2, 3, 4}) {
        const double wgs = (double)tiles64 * s;
        if (s > 1 && (wgs > cus || slices < 4 * s)) break;
        best.offer(64, s, pack + ceil(slices / s) * (wgs <= cus ? 0.22 : 0.45 * ceil(wgs / (2 * cus))) + (s > 1 ? 1.5 + 0.016 * wgs : 0.0));
    }
    // a slice's time in one round of few tiles, of a tile for every CU, and in more
    auto tile = [&](int kernel, int bm, int bn, double few, double full) {
        const double wgs = (double)(ceil_div(m, bm) * ceil_div(n, bn)) / cus;
        best.offer(kernel, 1, pack + slices * (wgs <= 1.0 ? few + (full - few) * wgs : full * ceil(wgs)));
    };
    tile(128, 128, 128, 0.47, 0.72);
    tile(192, 256, 128, 0.80, 1.20);
    tile(256, 256, 256, 1.25, 2.00);
    return best;
}

template <typename T>
static void launch_gemm8(const Gemm8Args& p) {
    const bool aligned = p.k % 16 == 0 && aligned16(p.a) && aligned16(p.w);
    const Plan8 plan = plan_gemm8(p.m, p.n, p.k, aligned);
    switch (plan.kernel) {
        case 1: return launch_rows8<1, 8, T>("nnc_hip_matmul_i8_rows16", p, aligned);
        case 2: return launch_rows8<2, 8, T>("nnc_hip_matmul_i8_rows32", p, aligned);
        case 4: return launch_rows8<4, 8, T>("nnc_hip_matmul_i8_rows64", p, aligned);
        case 64:
            return launch_tile8<Tile8<64, 64, 2, 2, 4, 4>, T>(plan.splits > 1 ? "nnc_hip_matmul_i8_64x64_split" : "nnc_hip_matmul_i8_64x64", p,
                                                              plan.splits);
        case 128: return launch_tile8<Tile8<128, 128, 2, 4, 4, 4>, T>("nnc_hip_matmul_i8_128x128", p, 1);
        case 192: return launch_tile8<Tile8<256, 128, 4, 2, 3, 2>, T>("nnc_hip_matmul_i8_256x128", p, 1);
        default: return launch_tile8<Tile8<256, 256, 2, 4, 2, 1>, T>("nnc_hip_matmul_i8_256x256", p, 1);
    }
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
    if (m > (int64_t)65535 * 64 || n > (int64_t)1 << 26) return fail(NNC_HIP_EUNSUPP, name, "too many rows");
    if (!ready(name)) return;
    Gemm8Args p{(const int8_t*)a->data, (const int8_t*)w->data, (const float*)a_scale->data, (const float*)w_scale->data,
                bias ? (const float*)bias->data : nullptr, out->data, m, n, (int)k,
                aligned16(out->data) && n * activation_bytes(out) % 16 == 0};
    if (out->dtype == NNC_DTYPE_FLOAT16)
        launch_gemm8<half_t>(p);
    else
        launch_gemm8<float>(p);
}

}  // extern "C"
