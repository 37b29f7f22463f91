// Host check of the mask arithmetic in csrc/ragged.h against bits taken one by
// one: prints "ok" or what is wrong.
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>

#include <vector>

#include "ragged.h"

using namespace nnc;

static uint64_t state = 88172645463325252ull;
static int rnd(int lo, int hi) {
    state ^= state << 13, state ^= state >> 7, state ^= state << 17;
    return lo + (int)(state % (uint64_t)(hi - lo + 1));
}

int main() {
    for (int trial = 0; trial < 200000; ++trial) {
        const int words = rnd(1, 4), rows = rnd(0, 150), far = rnd(0, 3) ? 0 : rnd(0, 1) ? INT_MAX / 2 - 400 : -rnd(0, 100);
        const int first = far + rnd(0, 100), length = first + rows < 0 ? 0 : first + rows;
        std::vector<int> mask(words);
        for (int& m : mask) m = (int)(uint32_t)(state = state * 6364136223846793005ull + 1442695040888963407ull, state >> 32);
        auto bit = [&](int64_t m) { return m < 32 * words && ((uint32_t)mask[m / 32] >> m % 32 & 1); };
        const int at = 16 * rnd(0, 20) + (far > 0 ? far / 16 * 16 : 0);
        const uint32_t got = tree_bits(mask.data(), words, first, length, at);
        for (int c = 0; c < 32; ++c) {
            const int64_t j = (int64_t)at + c;
            const bool want = c < 16 && j < length && (j < first || bit(j - first));
            if ((bool)(got >> c & 1) != want) return printf("bit %d in trial %d\n", c, trial), 1;
        }
        int depth = 0;
        for (int m = 0; m < rows; ++m) depth += bit(m);
        if (tree_depth(mask.data(), words, rows) != depth) return printf("depth in trial %d\n", trial), 1;
    }
    puts("ok");
}
