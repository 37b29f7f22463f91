// Attention of drafted tokens with many query rows behind long contexts
// (nnc_hip_kv_tree_attention; kvtree.hip has the formulas and the other kernels).
//
// There a wave widens a cached head's keys for 32 query rows, which takes it about
// as long as their scores. Here the eight waves of a workgroup take 32 rows each,
// and the keys go through LDS as f16, 64 at a time, widened once for all of them:
// operands and layouts as in kvattention.hip's kernel for prompts,
// v_mfma_f32_32x32x16_f16, a lane having the scores of 16 consecutive keys.
//
// The keys are cut into runs as in kvtree.hip. A workgroup that joined all shares
// of so large a tile would keep the others waiting (32 shares of 256 rows are 4
// MB), so that is a kernel of its own, 8 rows a workgroup.
//
// 64 drafts behind 65536, 32 heads over 8 of 128, f16: 102 to 111 us from card to
// card, 620 to 670 TFLOP/s of the 1170 of a large f16 product, where 32 rows a wave
// without LDS take 123; 64 sequences of 64 behind 2048 215 and 350. 64 keys of a
// tile take a CU 2.5 us; the matrix units work 32% of the time, the vector units 48%;
// storing the shares and joining them takes 8 us, the first keys' way into LDS and
// the last sums' out of registers 10.
#include "kvtree.h"

namespace nnc {

// Rows of a tile, and threads
static constexpr int kRows = 256, kThreads = 512;

template <int D>
__device__ __forceinline__ void rows_share(const TreeArgs& a, const TreeShare& w, int place, char* lds) {
    typedef half_t T;
    constexpr int STEPS = D / 16, DB = D / 32, KRB = 2 * D, STAGE = 64 * KRB + D * 128;
    static_assert(4 * D <= kThreads, "a piece of 16 bytes of each operand a thread");
    // [stage]: of 4 groups of 16 keys, K's scale, V's scale's logarithm and
    // inverse, 1 if they can be read; then the four last again
    float* units = (float*)(lds + 2 * STAGE);
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Span& span = w.span;
    const int first = span.first();
    const int from = w.lo + w.unit * 64, to = min(span.length, from + w.n * 64);
    const bool row_ok = 32 * wave + i < w.rows, idle = 32 * wave >= w.rows;
    const int64_t fr = (int64_t)w.tile * kRows + (row_ok ? 32 * wave + i : 0);
    const int tok = (int)(fr / a.group), gh = (int)(fr - (int64_t)tok * a.group);
    const int row = span.end - span.rows + tok, head = w.head_kv * a.group + gh;
    const int* mask = a.tree + (int64_t)row * a.words;

    // staging: this thread's pieces. The table entries of a chunk are read one
    // chunk before its keys and values, those two before they are used.
    const int page = a.g.page, page16 = page / 16;
    const int64_t plane = (int64_t)page * D, page_bytes = (int64_t)a.kv_heads * plane;
    const bool moves = threadIdx.x < 4 * D;
    const int kt = threadIdx.x / (D / 16) & 63;  // the key whose piece it is
    const int8_t* kbase = a.k + (int64_t)w.head_kv * plane + (kt & 15) * D + threadIdx.x % (D / 16) * 16;
    const int8_t* vbase = a.v + (int64_t)w.head_kv * plane + (int)(threadIdx.x >> 2) % D * page;
    const int* table = a.g.table + (int64_t)w.b * a.g.width;
    int kid, vid;
    auto entry = [&](int t16) { return table[min((int)slot_of(t16, a.slot_magic), a.g.width - 1)]; };
    auto find = [&](int tb) { kid = entry(tb / 16 + (kt >> 4)), vid = entry(tb / 16 + (threadIdx.x & 3)); };
    ix4 kr, vr;
    float su[2];
    bool can_read = false;
    auto load = [&](int tb) {
        const int gv = tb / 16 + (threadIdx.x & 3), gk = tb / 16 + (kt >> 4);
        const bool have = vid >= 0 && vid < a.g.pages && gv * 16 < to;
        const int64_t pv = have ? vid : 0, pk = kid >= 0 && kid < a.g.pages && gk * 16 < to ? kid : 0;
        const int offv = (gv - (int)slot_of(gv, a.slot_magic) * page16) * 16, offk = (gk - (int)slot_of(gk, a.slot_magic) * page16) * 16;
        if (moves) {
            kr = *reinterpret_cast<const ix4*>(kbase + pk * page_bytes + offk * D);
            vr = *reinterpret_cast<const ix4*>(vbase + pv * page_bytes + offv);
        }
        if (threadIdx.x < 4) {
            su[0] = a.k_scale[pv * a.kv_heads + w.head_kv];
            su[1] = a.v_scale[pv * a.kv_heads + w.head_kv];
            can_read = have;
        }
    };
    const int ktr = (kt & 32) | (kt & 12) << 1 | (kt & 16) >> 2 | (kt & 3);
    const int kput = lds_chunk<KRB>(ktr, threadIdx.x % (D / 16) * 2);
    const int vput = 64 * KRB + lds_chunk<128>((threadIdx.x >> 2) % D, (threadIdx.x & 3) * 2);
    const int kget = lds_chunk<KRB>(i, h), vget = 64 * KRB + lds_chunk<128>(i, 2 * h);
    auto store = [&](int stage) {
        const int kp = kput + stage * STAGE, vp = vput + stage * STAGE;
        if (moves) {
            *reinterpret_cast<f16x8*>(lds + kp) = widen8((uint32_t)kr[0], (uint32_t)kr[1]);
            *reinterpret_cast<f16x8*>(lds + (kp ^ 16)) = widen8((uint32_t)kr[2], (uint32_t)kr[3]);
            *reinterpret_cast<f16x8*>(lds + vp) = widen8((uint32_t)vr[0], (uint32_t)vr[1]);
            *reinterpret_cast<f16x8*>(lds + (vp ^ 16)) = widen8((uint32_t)vr[2], (uint32_t)vr[3]);
        }
        if (threadIdx.x < 4) {
            const float vu = can_read ? su[1] : 1.f, ok = can_read ? 1.f : 0.f;
            *reinterpret_cast<fx4*>(units + stage * 20 + threadIdx.x * 4) = fx4{can_read ? su[0] * a.scale : 0.f, scale_log(vu), 1.0f / vu, ok};
            units[stage * 20 + 16 + threadIdx.x] = ok;
        }
    };
    if (from < to) {
        find(from);
        load(from);
        find(from + 64);
    }

    // the query row
    const int low = a.window > 0 ? first + tree_depth(mask, a.words, span.rows) - 1 - a.window : INT_MIN;  // the last that the window hides
    f16x8 qf[STEPS];
    const T* qp = (const T*)a.q + (int64_t)row * a.ld + a.q_col + head * D + 8 * h;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
        if (a.q_vec) {
            qf[st] = *reinterpret_cast<const f16x8*>(qp + 16 * st);
        } else {
#pragma unroll
            for (int d = 0; d < 8; ++d) qf[st][d] = qp[16 * st + d];
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
        constexpr int GK = STEPS < 4 ? 2 : 4, GV = GK, GROUPS = 2 * STEPS / GK, VGROUPS = DB * 4 / GV;
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
            for (int v = 0; v < GV; ++v) {
                const int u = (n * GV + v) % 4, c = (n * GV + v) / 4;
                vf[n & 1][v] = *reinterpret_cast<const f16x8*>(lds + (va ^ ((u >> 1) * 64 + (u & 1) * 16)) + c * 32 * 128);
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
                for (int u = 0; u < GK; ++u) {
                    const bool start = n == kb * GROUPS / 2 && u == 0;
                    x[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n & 1][u], qf[n * GK % STEPS + u], start ? fx16{} : x[kb], 0, 0, 0);
                }
            }
            const fx4 un = *reinterpret_cast<const fx4*>(units + stage * 20 + (2 * kb + h) * 4);
            ku[kb] = un[0], lv[kb] = un[1], iv[kb] = un[2];
            ku[kb] = ku[kb] == 0.f ? 0x1p-126f : ku[kb];  // for the product with -inf
            // key tb + 32 kb + 16 h + r is in x[kb][r]
            if (masked) {
                const int j = tb + 32 * kb + 16 * h;
                uint32_t bits = un[3] != 0.f && row_ok ? tree_bits(mask, a.words, first, span.length, j) : 0u;
                if (a.window > 0) {  // of the context, up to low
                    const int n = min(min(low + 1, first) - j, 16);
                    if (n > 0) bits &= 0xffffffffu << n;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = x[kb][r];
                    x[kb][r] = bits >> r & 1 ? y : -INFINITY;
                }
                // a row that sees none of the 16: their scales are not its own
                if (!bits) ku[kb] = 1.f, lv[kb] = 0.f, iv[kb] = 0.f;
            }
            top[kb] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top[kb] = fmaxf(top[kb], x[kb][r]);
            mx = fmaxf(mx, fmaf(top[kb], ku[kb], lv[kb]));
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        float factor[2], most = 0.f;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) factor[kb] = ldexpf(iv[kb], (int)ex), most = fmaxf(most, factor[kb]);
        if (__any(mx > m + kSlack || most > kMostFactor)) {
            const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - mn);
            float far = reference(m, ex);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) far = fmaxf(far, top[kb] * ku[kb]);
            far = fmaxf(far, __shfl_xor(far, 32));
            const float en = exponent(mn, far);
            l *= rescale(m, ex, mn, en);
            m = mn, ex = en;
#pragma unroll
            for (int c = 0; c < DB; ++c) o[c] *= alpha;
            most = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) factor[kb] = ldexpf(iv[kb], (int)ex), most = fmaxf(most, factor[kb]);
            if (__any(most > kMostFactor)) {
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
        f16x8 pf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const float shift = lv[kb] - base;  // base: m - 12, of p's 2^12
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float s0 = x[kb][r], s1 = x[kb][r + 1];
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s0, ku[kb], shift)), p1 = __builtin_amdgcn_exp2f(fmaf(s1, ku[kb], shift));
                sum += p0;
                sum += p1;
                const f16x2 hi = __builtin_convertvector((fx2{p0, p1}), f16x2);
                pf[kb][r / 8][r % 8] = hi[0], pf[kb][r / 8][r % 8 + 1] = hi[1];
            }
            l = fmaf(sum, factor[kb], l);
        }
#pragma unroll
        for (int n = 0; n < VGROUPS; ++n) {
            if (n + 1 < VGROUPS) read_v(n + 1);
#pragma unroll
            for (int v = 0; v < GV; ++v) {
                const int u = (n * GV + v) % 4, c = (n * GV + v) / 4;
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n & 1][v], pf[u >> 1][u & 1], o[c], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (from < to) {
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
        const fx4 ok = *reinterpret_cast<const fx4*>(units + stage * 20 + 16);
        const bool clear = tb + 64 <= first && a.window <= 0 && __all(ok[0] * ok[1] * ok[2] * ok[3] != 0.f);
        if (!idle) attend(tb, stage, !clear);
    }

    l += __shfl_xor(l, 32);
    if (!row_ok) return;
    if (w.whole) {
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
        return;
    }
    const TreePlaces<D, kRows> places(a);
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float p0 = o[c][4 * q], p1 = o[c][4 * q + 1], p2 = o[c][4 * q + 2], p3 = o[c][4 * q + 3];
            places.put4(place, 32 * wave + i, 32 * c + 8 * q + 4 * h, p0, p1, p2, p3);
        }
    if (h == 0) places.put4(place, 32 * wave + i, D, m, l, ex, 0.f);
}

// Where keys are fewer than was said, runs of so many units, and tiles of no more
// left whole
static constexpr int kShortUnits = 4;

template <int D>
__global__ void __launch_bounds__(kThreads, 2) kv_tree_rows_k(TreeArgs a) {
    extern __shared__ __align__(16) char rows_lds[];
    walk_run<kRows, 64, kShortUnits>(
        a, [&](const TreeShare& w, int place) { rows_share<D>(a, w, place, rows_lds); }, [](const TreeShare&, int64_t, int, auto) {});
}

// The shares that kv_tree_rows_k left, kJoinRows rows a workgroup
static constexpr int kJoinRows = 8, kParts = kRows / kJoinRows;
template <int D>
__global__ void __launch_bounds__(256) kv_tree_rows_join_k(TreeArgs a) {
    __shared__ __align__(16) float lds[kJoinRows * (3 * kJoin + 2) + kJoin];
    const uint32_t item = blockIdx.x / kParts, row0 = blockIdx.x % kParts * kJoinRows;
    TreeShare w;
    w.head_kv = (int)(item / (uint32_t)a.tiles);
    TreeIndex<kRows, 64> index(a);
    const int64_t each = index.total(), total = each * a.kv_heads;
    int64_t begin;
    const TreePlace p = index.find_tile(item - (uint32_t)w.head_kv * a.tiles, begin);
    if (p.b < 0 || p.s.units <= kShortUnits) return;
    w.span = p.s.span, w.tile = p.tile;
    const int64_t left = (int64_t)w.span.rows * a.group - (int64_t)w.tile * kRows - row0;
    if (left <= 0) return;
    begin += w.head_kv * each;
    const int runs = tree_runs(a, total), run0 = run_of(begin, total, runs), shares = run_of(begin + p.s.units - 1, total, runs) - run0 + 1;
    if (shares == 1) return;
    join_shares<half_t, D, kRows, kJoinRows, 256>(
        TreePlaces<D, kRows>(a), (int)row0, left < kJoinRows ? (int)left : kJoinRows, shares,
        [&](int sh) { return share_place(run0 + sh, begin, total, runs); }, [&](int r) { return tree_row<half_t, D, kRows>(a, w, r); }, lds);
}

template <int D>
static void launch_rows(const char* name, TreeArgs a, int64_t rows) {
    constexpr int lds = 2 * (64 * 2 * D + D * 128) + 2 * 20 * 4;
    auto kernel = kv_tree_rows_k<D>;
    static const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess;
    if (!ok) return fail(NNC_HIP_EDEVICE, name, "hipFuncSetAttribute failed");
    a.runs = cu_count();
    a.least = kShortUnits;
    if (!tree_scratch(name, a, rows, kRows, D)) return;
    launch(name, kernel, dim3((unsigned)a.runs), dim3(kThreads), lds, a);
    set_work(0.0, 4.0 * a.runs * kRows * D);
    launch("nnc_hip_kv_tree_attention_join", kv_tree_rows_join_k<D>, dim3((unsigned)(a.tiles * a.kv_heads * kParts)), dim3(256), 0, a);
}

// For more than 128 rows of f16 behind so many keys that a CU has 24 times 64 of
// a tile, were all sequences the longest, or as long as a window leaves them. us,
// 32 heads over 8 of 128, this and 32 rows a wave: 16 sequences behind 4096 of 36
// drafts 98 and 119, of 64 115 and 128, of 128 180 and 248; with 16 times 64 keys 8
// of 64 behind 4096 71 and 63, with 8 4 of 64 50 and 44; 2 of 100 behind 16384 under
// a window of 4096 51 and 52, of 1024 44 and 32, of 100 24 and 13. Tiles of 128 rows
// in two workgroups a CU: 18 drafts 69 and 84, but 32 82 and 70; of 64 rows, two
// waves to a row's keys: 16 behind up to 8192 96 and 77. fp32 of 64 162 and 169, of
// 40 139 and 135 (dim 256 has no registers for it).
bool launch_tree_rows(const char* name, bool f16, int dim, const TreeArgs& a, int64_t rows, int64_t each, int64_t reach) {
    if (!f16 || dim > 128 || each <= kRows / 2) return false;
    const int64_t holders = rows < a.g.batch ? rows : a.g.batch;
    if (ceil_div(each, kRows) * holders * a.kv_heads * ceil_div(reach, 64) < 24 * (int64_t)cu_count()) return false;
    // (the join's grid: whole tiles for each sequence)
    if ((rows * a.group + kRows * holders) / kJoinRows * a.kv_heads * 256 > UINT32_MAX) return false;
    switch (dim) {
        case 32: launch_rows<32>(name, a, rows); break;
        case 64: launch_rows<64>(name, a, rows); break;
        default: launch_rows<128>(name, a, rows);
    }
    return true;
}

}  // namespace nnc
