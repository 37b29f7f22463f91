// Host check of csrc/ragged.h over random batches, sound ones and ones with
// any numbers in starts, lengths and the table: prints "ok" or what is wrong.
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
static void no(const char* what, int trial) {
    printf("%s in trial %d\n", what, trial);
    exit(1);
}

int main() {
    for (int trial = 0; trial < 20000; ++trial) {
        const bool sound = trial % 2 == 0;
        const int batch = rnd(1, 9), page = 16 * rnd(1, 16), width = rnd(1, 6), pages = rnd(1, 60);
        std::vector<int> starts(batch + 1), lengths(batch), table(batch * width);
        for (int b = 0; b < batch; ++b) {
            lengths[b] = sound ? rnd(0, width * page) : rnd(-5, 3 * width * page);
            const int n = sound ? rnd(0, rnd(0, 3) ? 2 : lengths[b]) : rnd(-3, 400);
            starts[b + 1] = sound ? starts[b] + n : (rnd(0, 9) && starts[b] < 1000000000 ? starts[b] + n : rnd(-1000000000, 1000000000));
        }
        for (int& t : table) t = sound ? rnd(0, pages - 1) : rnd(-10, pages + 10);
        const int rows = sound ? starts[batch] + rnd(0, 3) : rnd(0, 500);
        const Ragged g{starts.data(), lengths.data(), table.data(), batch, width, rows, page, pages};
        int64_t touched = 0;
        for (int b = 0; b < batch; ++b) {
            const Span s = span_of(g, b);
            if (s.rows < 0 || s.end < s.rows || s.end > rows || s.length < 0 || s.length > width * page) no("span", trial);
            const int count = touched_pages(g, b);
            touched += count;
            std::vector<int> hit(width * page, 0);
            for (int share = 0; share < count; ++share) {
                const PageShare p(g, b, share);
                if (p.page_no < -1 || p.page_no >= pages) no("page number", trial);
                if (p.begin % page || p.fresh < p.begin || p.stop > p.begin + page || p.fresh >= p.stop) no("page range", trial);
                for (int t = p.fresh; t < p.stop; ++t) {
                    if (t < 0 || t >= s.length || t / page >= width) no("position", trial);
                    const int r = p.span.row(t);
                    if (r < s.end - s.rows || r >= s.end) no("row", trial);
                    ++hit[t];
                }
            }
            for (int t = 0; t < width * page; ++t) {
                const bool mine = t < s.length && t >= s.length - s.rows;
                if (hit[t] != (mine ? 1 : 0)) no("positions covered", trial);
            }
            for (int group : {1, 3, 16, 40})
                for (int tile : {16, 128}) {
                    const int tiles = query_tiles(s, group, tile);
                    if ((int64_t)tiles * tile < (int64_t)s.rows * group || (tiles && (int64_t)(tiles - 1) * tile >= (int64_t)s.rows * group))
                        no("tiles", trial);
                }
        }
        if (sound) {
            if (touched > touched_bound(rows, batch, page)) no("bound of touched pages", trial);
            for (int group : {1, 3, 16, 40})
                for (int tile : {16, 128}) {
                    int64_t tiles = 0;
                    for (int b = 0; b < batch; ++b) tiles += query_tiles(span_of(g, b), group, tile);
                    if (tiles > query_tiles_bound(rows, batch, group, tile)) no("bound of tiles", trial);
                }
        }
        // shares of the keys: all of them, once, none empty, no more than the splits
        const int last = rnd(-3, 20000), first = last - rnd(0, 50), window = rnd(0, 2) ? 0 : rnd(1, 3000);
        const int splits = rnd(1, 40), step = rnd(0, 1) ? 256 : 64, least = step * rnd(1, 8);
        const KeyRange k(first, last, window, splits, least, step);
        const int shares = k.shares();
        if (shares < 1 || shares > splits) no("shares", trial);
        if (k.lo < 0 || k.lo % 64 || k.chunk % step || k.hi != (last < 0 ? 0 : last + 1)) no("key range", trial);
        if (window && k.lo > (first - window + 1 > 0 ? first - window + 1 : 0)) no("window", trial);
        if ((int64_t)k.lo + (int64_t)shares * k.chunk < k.hi) no("keys left over", trial);
        if (shares > 1 && (int64_t)k.lo + (int64_t)(shares - 1) * k.chunk >= k.hi) no("empty share", trial);
    }
    for (int page16 = 1; page16 <= 16; ++page16) {
        const uint32_t magic = slot_magic(page16);
        for (uint32_t t = 0; t < 1u << 20; ++t)
            if (slot_of(t, magic) != t / page16) no("slot", (int)t);
        for (uint32_t t = (1u << 28) - 100000; t < 1u << 28; ++t)
            if (slot_of(t, magic) != t / page16) no("slot", (int)t);
    }
    printf("ok\n");
    return 0;
}
