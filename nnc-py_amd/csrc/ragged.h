// Index arithmetic of ragged batches over a paged cache, for the kernels and,
// compiled by itself, for the host. starts, lengths and the page table live on
// the device, so whatever they hold is clamped here to the rows, positions and
// pages that there are.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define RAGGED_HD __host__ __device__ __forceinline__
#else
#define RAGGED_HD inline
#endif

namespace nnc {

// Sequence b's rows of the activations are starts[b] .. starts[b + 1]; they
// are its last positions, lengths[b] being its length with them; position t is
// in page table[b][t / page].
struct Ragged {
    const int* starts;   // [batch + 1]
    const int* lengths;  // [batch]
    const int* table;    // [batch][width]
    int batch, width, rows, page;
    int64_t pages;
};

RAGGED_HD int imin(int a, int b) { return a < b ? a : b; }
RAGGED_HD int imax(int a, int b) { return a > b ? a : b; }

struct Span {
    int end;     // one past the sequence's last row
    int length;  // positions, with the rows
    int rows;    // rows; those with no position (more rows than length) included
    // the row at a position, and the first row's position: negative if there
    // are more rows than positions
    RAGGED_HD int row(int pos) const { return end - length + pos; }
    RAGGED_HD int first() const { return length - rows; }
};

RAGGED_HD Span span_of(const Ragged& g, int b) {
    Span s;
    const int r0 = imin(imax(g.starts[b], 0), g.rows);
    s.end = imin(imax(g.starts[b + 1], r0), g.rows);
    s.rows = s.end - r0;
    s.length = imin(imax(g.lengths[b], 0), g.width * g.page);
    return s;
}

// pages that a sequence's rows touch, and the most that `rows` rows of
// `batch` sequences can: each has one row at least, and a run of n rows
// touches n / page + 2 at most
RAGGED_HD int touched_pages(const Ragged& g, int b) {
    const Span s = span_of(g, b);
    if (s.rows <= 0 || s.length <= 0) return 0;
    return (s.length - 1) / g.page - imax(s.first(), 0) / g.page + 1;
}
RAGGED_HD int64_t touched_bound(int64_t rows, int64_t batch, int page) {
    const int64_t some = rows / page + 2 * batch;
    return rows < some ? rows : some;
}

// the page number of a table slot, or -1 if it is none of the cache's
RAGGED_HD int page_at(const Ragged& g, int b, int slot) {
    const int p = g.table[(int64_t)b * g.width + slot];
    return p >= 0 && p < g.pages ? p : -1;
}

// The share of a touched page: positions `begin` .. of slot, the rows' own
// from `fresh` to `stop`.
struct PageShare {
    Span span;
    int begin, fresh, stop, page_no;
    RAGGED_HD PageShare(const Ragged& g, int b, int share) {
        span = span_of(g, b);
        const int slot = imax(span.first(), 0) / g.page + share;
        begin = slot * g.page;
        fresh = imax(span.first(), begin);
        stop = imin(span.length, begin + g.page);
        page_no = page_at(g, b, slot);
    }
};

// The table slot of a group of 16 positions: t16 / page16, page16 = page / 16
// from 1 to 16, by one multiplication: slot_magic(page16) * page16 is less than
// 16 over 2^32, so the quotient is exact for t16 below 2^28. 0 stands for 2^32.
RAGGED_HD uint32_t slot_magic(int page16) { return page16 == 1 ? 0u : (uint32_t)((0xffffffffu / (uint32_t)page16) + 1u); }
RAGGED_HD uint32_t slot_of(uint32_t t16, uint32_t magic) { return magic ? (uint32_t)((uint64_t)t16 * magic >> 32) : t16; }

// Attention: the rows of one cached head's `group` query heads, tokens
// outermost, in tiles of `tile` rows.
RAGGED_HD int query_tiles(const Span& s, int group, int tile) {
    return (int)(((int64_t)s.rows * group + tile - 1) / tile);
}
RAGGED_HD int64_t query_tiles_bound(int64_t rows, int64_t batch, int group, int tile) {
    const int64_t some = rows * group / tile + (rows < batch ? rows : batch), each = rows * ((group + tile - 1) / tile);
    return some < each ? some : each;
}

// The window that is compared: none (0) if it is as long as a sequence can be,
// so that positions less it stay far from the smallest number.
RAGGED_HD int window_of(int window, int capacity) { return window < capacity ? window : 0; }

// The keys that rows at positions first .. last see, [lo, hi), in at most
// `splits` shares of at least `least` keys (a multiple of `step`): share s has
// [lo + s * chunk, ...).
struct KeyRange {
    int lo, hi, chunk;
    RAGGED_HD KeyRange(int first, int last, int window, int splits, int least, int step) {
        hi = imax(last + 1, 0);
        lo = window > 0 && first >= window ? (first - window + 1) & ~63 : 0;
        const int each = (imax(hi - lo, 0) + splits - 1) / splits;
        chunk = imax(least, (each + step - 1) / step * step);
    }
    RAGGED_HD int shares() const { return imax(1, (int)(((int64_t)imax(hi - lo, 0) + chunk - 1) / chunk)); }
};

}  // namespace nnc
