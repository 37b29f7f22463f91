// Host check of the keys that csrc/ragged.h gives to rows under a window, for
// windows and positions up to the largest whole numbers, rows without a
// position among them: prints "ok" or what is wrong.
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>

#include <initializer_list>

#include "ragged.h"

using namespace nnc;

static uint64_t state = 88172645463325252ull;
static int64_t rnd(int64_t lo, int64_t hi) {
    state ^= state << 13, state ^= state >> 7, state ^= state << 17;
    return lo + (int64_t)(state % (uint64_t)(hi - lo + 1));
}

int main() {
    const int most = INT_MAX / 2;  // positions that a table can have
    for (int trial = 0; trial < 400000; ++trial) {
        const int capacity = (int)(trial % 2 ? rnd(1, 5000) : rnd(1, most));
        const int rows = (int)rnd(1, 40), last = (int)rnd(-3, capacity - 1), first = last - rows + 1;
        int window = 0;
        switch (trial % 5) {
            case 0: window = INT_MAX - (int)rnd(0, 70); break;
            case 1: window = (int)rnd(1, INT_MAX); break;
            case 2: window = (int)rnd(imax(capacity - 2, 1), (int64_t)capacity + 2); break;
            case 3: window = (int)rnd(1, 3000); break;
            default: break;
        }
        const int seen = window_of(window, capacity);
        const KeyRange k(first, last, seen, 1, 64, 64);
        if (k.hi != imax(last + 1, 0) || k.lo < 0 || k.lo % 64) return printf("range in trial %d\n", trial), 1;
        // every key that the rows' positions see, and no position less than 64 before the first
        const int64_t from = window > 0 && (int64_t)first - window + 1 > 0 ? (int64_t)first - window + 1 : 0;
        if (k.lo > from || k.lo + 64 <= from) return printf("first key %d, not %lld, in trial %d\n", k.lo, (long long)from, trial), 1;
        for (int pos : {first, last}) {
            // as the kernels compare: key j is seen if j <= pos and j > pos - window
            const int low = seen > 0 ? pos - seen : INT_MIN;
            for (int64_t j : {(int64_t)0, (int64_t)pos, (int64_t)pos - window, (int64_t)pos - window + 1, rnd(0, capacity - 1)}) {
                if (j < 0 || j > pos) continue;
                const bool want = window == 0 || j > (int64_t)pos - window;
                if ((j > low) != want) return printf("key in trial %d\n", trial), 1;
            }
        }
    }
    printf("ok\n");
    return 0;
}
