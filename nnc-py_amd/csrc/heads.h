// How the heads of a row are given to waves (rope.hip), for the kernels and,
// compiled by itself, for the host.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define HEADS_HD __host__ __device__ __forceinline__
#else
#define HEADS_HD inline
#endif

namespace nnc {

// 2^bits lanes are a head, so a wave has 64 >> bits heads at once, and goes
// through `per` of these passes; `chunks` of them for each row.
struct RopeWaves {
    int bits, per, chunks;
    HEADS_HD int groups() const { return 64 >> bits; }
    // a chunk's heads [begin, end), a pass every groups() of them
    HEADS_HD int begin(int chunk) const { return chunk * per * groups(); }
    HEADS_HD int end(int chunk, int heads) const {
        const int e = begin(chunk + 1);
        return e < heads ? e : heads;
    }
};

// A wave takes all of a row's heads while rows are many; v: values of a pack
inline RopeWaves rope_waves(int64_t rows, int heads, int dim, int v, int cus) {
    RopeWaves s{};
    while ((2 * v << s.bits) < dim) ++s.bits;
    const int passes = (heads + s.groups() - 1) / s.groups();
    s.per = passes;
    while (s.per > 1 && rows * ((passes + s.per - 1) / s.per) < 16 * (int64_t)cus) s.per = (s.per + 1) / 2;
    s.chunks = (passes + s.per - 1) / s.per;
    return s;
}

}  // namespace nnc
