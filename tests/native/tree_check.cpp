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
    // runs cover the units once, and the shares of an item have places of their own
    for (int trial = 0; trial < 3000; ++trial) {
        const int parts = rnd(1, 40), items = rnd(1, 30);
        std::vector<int64_t> begin(1, 0);
        for (int n = 0; n < items; ++n) begin.push_back(begin.back() + rnd(1, rnd(0, 1) ? 3 : 60));
        const int64_t total = begin.back();
        if (parts > total) continue;
        std::vector<int> seen(total, 0), taken(2 * parts, 0);
        for (int p = 0; p < parts; ++p)
            for (int64_t i = run_begin(p, total, parts); i < run_begin(p + 1, total, parts); ++i) {
                ++seen[i];
                if (run_of(i, total, parts) != p) return printf("run of %lld in trial %d\n", (long long)i, trial), 1;
            }
        for (int n : seen)
            if (n != 1) return printf("units in trial %d\n", trial), 1;
        for (int n = 0; n < items; ++n) {
            const int first = run_of(begin[n], total, parts), last = run_of(begin[n + 1] - 1, total, parts);
            if (first == last) continue;  // whole
            for (int p = first; p <= last; ++p) {
                const int at = share_place(p, begin[n], total, parts);
                if (at < 0 || at >= 2 * parts || taken[at]++) return printf("place in trial %d\n", trial), 1;
            }
        }
    }
    puts("ok");
}
