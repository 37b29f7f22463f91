// Host check of what windows do to the keys of drafts (csrc/ragged.h): prints
// "ok" or what is wrong.
#include <stdio.h>
#include <stdlib.h>

#include "ragged.h"

using namespace nnc;

static uint64_t state = 88172645463325252ull;
static int rnd(int lo, int hi) {
    state ^= state << 13, state ^= state >> 7, state ^= state << 17;
    return lo + (int)(state % (uint64_t)(hi - lo + 1));
}

int main() {
    for (int trial = 0; trial < 200000; ++trial) {
        const int rows = rnd(1, 200), length = rnd(0, rnd(0, 1) ? 300 : 20000), longest = length + (rnd(0, 1) ? 0 : rnd(0, 5000));
        const int window = rnd(0, 2) ? rnd(1, rnd(0, 1) ? 100 : 21000) : 0, first = length - rows;
        const int lo = tree_low(first, window);
        // a row that sees no drafts but itself, and one whose mask is empty
        for (int depth = 0; depth < 2; ++depth) {
            const int p = first + depth - 1, seen = window > 0 ? imax(p - window + 1, 0) : 0;
            if (lo % 64 || lo < 0 || lo > seen) return printf("first key in trial %d\n", trial), 1;
        }
        const int64_t reach = tree_reach(window, rows, longest);
        if (reach < length - lo || reach > longest) return printf("reach in trial %d\n", trial), 1;
        if (window > 0 && reach > (int64_t)window + rows + 63) return printf("window in trial %d\n", trial), 1;
    }
    puts("ok");
}
