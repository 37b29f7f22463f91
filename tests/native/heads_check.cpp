// Host check of csrc/heads.h: every head of a row in one pass of one chunk, and
// no pass that has none. Prints "ok" or what is wrong.
#include <stdio.h>
#include <stdlib.h>

#include <vector>

#include "heads.h"

using namespace nnc;

static uint64_t state = 88172645463325252ull;
static int rnd(int lo, int hi) {
    state ^= state << 13, state ^= state >> 7, state ^= state << 17;
    return lo + (int)(state % (uint64_t)(hi - lo + 1));
}

// The passes of a row's waves, -1 if a head is missing, twice there or none of the row's
static int passes(const RopeWaves& s, int heads) {
    std::vector<int> seen(heads, 0);
    int n = 0;
    for (int chunk = 0; chunk < s.chunks; ++chunk) {
        const int end = s.end(chunk, heads);
        for (int first = s.begin(chunk); first < end; first += s.groups(), ++n)
            for (int g = 0; g < s.groups(); ++g)
                if (first + g < end && (first + g >= heads || seen[first + g]++)) return -1;
    }
    for (int h : seen)
        if (h != 1) return -1;
    return n;
}

int main() {
    for (int trial = 0; trial < 20000; ++trial) {
        const int v = rnd(0, 1) ? 8 : 4, dim = 2 * v * rnd(1, 64), heads = rnd(1, rnd(0, 3) ? 70 : 5000), cus = rnd(1, 304);
        const int64_t rows = rnd(1, rnd(0, 2) ? 100 : 30000);
        const RopeWaves s = rope_waves(rows, heads, dim, v, cus);
        const int needed = (heads + s.groups() - 1) / s.groups();
        if ((2 * v << s.bits) < dim || s.groups() < 1 || s.per < 1) return printf("lanes in trial %d\n", trial), 1;
        const int n = passes(s, heads);
        if (n != needed) return printf("%d passes for %d in trial %d\n", n, needed, trial), 1;
    }
    const struct { int rows, heads, dim, v, needed; } calls[] = {{16, 40, 128, 8, 5}, {777, 16, 96, 4, 4}, {32, 32, 128, 8, 4}, {2000, 40, 128, 8, 5}};
    for (auto c : calls)
        if (passes(rope_waves(c.rows, c.heads, c.dim, c.v, 256), c.heads) != c.needed) return printf("[%d, %d x %d]\n", c.rows, c.heads, c.dim), 1;
    puts("ok");
}
