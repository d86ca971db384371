// paged_plan.h -- how the attention over a paged cache is cut into work, for
// the device and (tests) the host: integer arithmetic only.
//
// The query rows of one KV head and one sequence (its tokens times the query
// heads of the group) are cut into row tiles of 2^q tokens, the positions that
// a tile's last row sees into key tiles of 64.  A segment is one row tile with
// all its key tiles, a unit one key tile of one segment.  All units of a launch
// form one line,
//   [ shared prefix: KV head, row tile over all rows ][ sequence, KV head, row tile ],
// where a segment has kPagedLead units more than key tiles, at its beginning:
// what its start and end cost beside them (queries and first tiles from memory,
// results to it) is about as much.  A segment of at most 16 rows and 8 key
// tiles is never cut, and counts less: one wave does it alone, while others do
// theirs.  The line is cut into equal ranges, one for each workgroup, whatever the lengths
// are: a long sequence is spread over many workgroups, many short ones share
// one.  A cut close to a segment's edge is moved there.  A segment that is cut
// leaves one partial result in each range that holds a part of it; they
// are joined by a second kernel.  Lengths are known on the device only, so each
// workgroup finds its range itself: unit counts of row tiles have a closed form,
// so it needs one prefix sum over the sequences.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define TER_HD __host__ __device__ __forceinline__
#else
#define TER_HD inline
#endif

namespace terhip {

constexpr int kPagedKeys = 64;   // positions of a key tile
constexpr int kPagedRows = 128;  // rows of a row tile
constexpr int kPagedLead = 3;
constexpr int kPagedFew = 16;    // rows and key tiles of a segment that is never cut
constexpr int kPagedShort = 8;

TER_HD int paged_min(int a, int b) { return a < b ? a : b; }
TER_HD int paged_max(int a, int b) { return a > b ? a : b; }

// log2 of the tokens of a row tile: the largest power of two of them that has
// at most 128 rows.
TER_HD int paged_tokens_log2(int group) {
    int q = 0;
    while ((2 << q) * group <= kPagedRows) ++q;
    return q;
}

struct PagedSeq {
    int r0, n;  // first row, rows
    int base;   // positions before the rows (negative: rows that see nothing), at most cap
};
TER_HD PagedSeq paged_seq(int row0, int row1, int kv_len, int n_rows, int cap) {
    PagedSeq s;
    s.r0 = paged_min(paged_max(row0, 0), n_rows);
    s.n = paged_min(paged_max(row1, s.r0), n_rows) - s.r0;
    s.base = paged_min(paged_max(kv_len, 0) - s.n, cap);
    return s;
}
// Positions that row i of a sequence sees.
TER_HD int paged_limit(const PagedSeq& s, int i, int cap) { return paged_min(paged_max(s.base + i + 1, 0), cap); }

TER_HD int paged_row_tiles(const PagedSeq& s, int q) { return (s.n + (1 << q) - 1) >> q; }
// Key tiles of row tile rt of a sequence from position kv0 on, at least one (a
// row that sees nothing has an output too).
TER_HD int paged_key_tiles(const PagedSeq& s, int rt, int q, int kv0) {
    const int a = s.base - kv0 + paged_min(s.n, (rt + 1) << q);
    return a <= kPagedKeys ? 1 : (a + kPagedKeys - 1) / kPagedKeys;
}
// Key tiles of row tiles 0 .. n - 1, all of them full.  (Sums modulo 2^32, of
// which the result is less.)
TER_HD int paged_key_tiles_before(const PagedSeq& s, int n, int q, int kv0) {
    const int c = s.base - kv0, room = kPagedKeys - c;
    const int ones = paged_min(n, room >= (1 << q) ? room >> q : 0);  // tiles of at most 64 positions
    if (ones == n) return n;
    const unsigned m = (unsigned)(n - ones);
    if (q >= 6)  // ceil((c + 2^q i) / 64), i = ones + 1 .. n
        return (int)((unsigned)ones + m * (unsigned)((c + 63) >> 6) + ((m * (unsigned)(ones + 1 + n) / 2) << (q - 6)));
    // ceil(x / R) for x = e + ones + 1 .. e + n, R row tiles to a key tile
    const int lr = 6 - q, e = (c + (1 << q) - 1) >> q;
    const unsigned x1 = (unsigned)(e + n), x0 = (unsigned)(e + ones), a1 = x1 >> lr, a0 = x0 >> lr, r = (1u << lr) - 1;
    return (int)((unsigned)ones + (((a1 * (a1 + 1) / 2) << lr) + (x1 & r) * (a1 + 1)) -
                 (((a0 * (a0 + 1) / 2) << lr) + (x0 & r) * (a0 + 1)));
}
// Whether the only segment of a sequence and KV head is one that is never cut.
TER_HD bool paged_solid(const PagedSeq& s, int group, int q, int kv0) {
    return s.n * group <= kPagedFew && s.n <= 1 << q && paged_key_tiles(s, 0, q, kv0) <= kPagedShort;
}
// Units of a segment, of the row tiles before it, of a sequence for one KV head.
TER_HD int paged_length(const PagedSeq& s, int rt, int group, int q, int kv0) {
    const int n = paged_key_tiles(s, rt, q, kv0);
    return paged_solid(s, group, q, kv0) ? 1 + (n + 1) / 2 : kPagedLead + n;
}
TER_HD int paged_length_before(const PagedSeq& s, int n, int q, int kv0) {
    return n * kPagedLead + paged_key_tiles_before(s, n, q, kv0);
}
TER_HD int paged_units(const PagedSeq& s, int group, int q, int kv0) {
    const int t = paged_row_tiles(s, q);
    return t ? paged_length_before(s, t - 1, q, kv0) + paged_length(s, t - 1, group, q, kv0) : 0;
}
// The row tile that holds unit r of a sequence and KV head.
TER_HD int paged_row_tile_of(const PagedSeq& s, int r, int q, int kv0) {
    int lo = 0, hi = paged_row_tiles(s, q) - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (paged_length_before(s, mid, q, kv0) <= r)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// One launch's line of units.  The ranges: workgroup g of n_wg takes the units
// from cut g to cut g + 1, cut g being at or near total * g / n_wg.
struct PagedLine {
    int group, q, kv0;         // query heads of a KV head, row tile, first position behind the prefix
    int prefix_length;         // units of a row tile on the prefix
    int prefix_rows;           // row tiles over all rows
    int prefix_units;          // of all KV heads
    int total;
    int n_wg, near;            // ranges; cuts closer than `near` to an edge move there
    int skew, rounds, round;   // 0: equal ranges; else PagedCuts::skew, workgroups of a CU, CUs of an XCD
};
TER_HD PagedLine paged_line(int group, int q, int shared, int n_rows, int nkv) {
    PagedLine l{};
    l.group = group;
    l.q = q;
    l.kv0 = shared;
    l.prefix_length = shared ? kPagedLead + (shared + kPagedKeys - 1) / kPagedKeys : 0;
    l.prefix_rows = (n_rows + (1 << q) - 1) >> q;
    l.prefix_units = l.prefix_length * l.prefix_rows * nkv;
    return l;
}
// How the line is cut.  resident: workgroups that run at the same time; more
// ranges than that, of `target` units or more, if there is work for them: the
// hardware starts them as others end, which evens out what equal ranges do not
// (of two workgroups of a CU the older one is served first and ends a quarter
// earlier).  min_per: fewer units than that are not worth a workgroup.  uncut:
// segments of fewer key tiles are never cut.
struct PagedCuts {
    int max_wg, resident, target, min_per, uncut;
    int skew, rounds, round;
};
TER_HD void paged_cut(PagedLine& l, int total, const PagedCuts& c) {
    l.total = total;
    l.n_wg = (int)(((unsigned)total + (unsigned)c.min_per - 1) / (unsigned)c.min_per);
    int part = 8;
    if (l.n_wg > c.resident) {
        l.n_wg = paged_max(c.resident, paged_min(c.max_wg, (int)((unsigned)total / (unsigned)c.target)));
        if (l.n_wg > c.resident) part = 2;
    }
    l.n_wg = paged_min(l.n_wg, c.max_wg);  // (more work than the host knows of: sequences that overlap)
    const int step = l.n_wg ? (int)((unsigned)total / (unsigned)l.n_wg) : 0;
    l.near = paged_max(paged_max(1, step / part), (c.uncut + 1) / 2);
    l.skew = l.n_wg == c.resident && step >= 4 ? c.skew : 0;  // (so that no range is empty)
    l.rounds = c.rounds;
    l.round = c.round;
}
// Sixteenths of a mean range before range g.
TER_HD int paged_share_before(const PagedLine& l, int g) {
    if (!l.skew) return 16 * g;
    const int chunk = l.rounds * l.round, x = (int)((unsigned)g / (unsigned)chunk), y = g - x * chunk;
    const int r = (int)((unsigned)y / (unsigned)l.round), i = y - r * l.round;
    return 16 * g + l.skew * (r * (l.rounds - r) * l.round + (l.rounds - 1 - 2 * r) * i);
}
// floor(total * share before g / all shares).  (In binary64 exactly: the
// quotient is below 2^31, and at least 2^-16 off an integer if it is none.)
TER_HD int paged_cut_at(const PagedLine& l, int g) {
    return (int)((double)l.total * paged_share_before(l, g) / (16 * l.n_wg));
}
// The first cut at unit u or behind it: with at least ceil(u * all shares /
// total) before it.  (Exactly: below 2^16, at least 2^-31 off an integer.)
TER_HD int paged_cut_from(const PagedLine& l, int u) {
    if (u <= 0) return 0;
    const int a = (int)__builtin_ceil((double)u * (16 * l.n_wg) / l.total);
    if (!l.skew) return (a + 15) / 16;
    const int chunk = l.rounds * l.round, x = (int)((unsigned)a / (unsigned)(16 * chunk));
    int at = a - 16 * chunk * x, g = x * chunk;
    for (int r = 0; r < l.rounds; ++r) {
        const int w = 16 + l.skew * (l.rounds - 1 - 2 * r);
        if (at <= w * l.round) return g + (at + w - 1) / w;
        at -= w * l.round;
        g += l.round;
    }
    return g;
}

struct PagedSegment {
    int start, n;   // first unit, units
    int seq;        // -1: the prefix
    int kvh, tile;  // KV head, row tile
    int lead;       // units before its first key tile (0: never cut)
};

// The segment of unit u (0 <= u < total): b is the first sequence with units
// behind u (of no matter for the prefix), s its rows, b0 and b1 the units
// before it and behind it.
TER_HD PagedSegment paged_segment(const PagedLine& l, int u, int nkv, int b, const PagedSeq& s, int b0, int b1) {
    PagedSegment g;
    if (u < l.prefix_units) {
        const unsigned i = (unsigned)u / (unsigned)l.prefix_length;
        g.seq = -1;
        g.kvh = (int)(i / (unsigned)l.prefix_rows);
        g.tile = (int)i - g.kvh * l.prefix_rows;
        g.start = (int)i * l.prefix_length;
        g.n = l.prefix_length;
        g.lead = kPagedLead;
        return g;
    }
    const int each = (int)((unsigned)(b1 - b0) / (unsigned)nkv), at = u - b0;
    g.seq = b;
    g.kvh = (int)((unsigned)at / (unsigned)each);
    const int r = at - g.kvh * each;
    g.tile = paged_row_tile_of(s, r, l.q, l.kv0);
    g.start = b0 + g.kvh * each + paged_length_before(s, g.tile, l.q, l.kv0);
    g.n = paged_length(s, g.tile, l.group, l.q, l.kv0);
    g.lead = paged_solid(s, l.group, l.q, l.kv0) ? 0 : kPagedLead;
    return g;
}
// To the segment behind g where that is of the same sequence s (or of the
// prefix); false: it is not.
TER_HD bool paged_advance(const PagedLine& l, PagedSegment& g, const PagedSeq& s, int nkv) {
    const int tiles = g.seq < 0 ? l.prefix_rows : paged_row_tiles(s, l.q);
    if (g.tile + 1 < tiles)
        ++g.tile;
    else if (g.kvh + 1 < nkv)
        ++g.kvh, g.tile = 0;
    else
        return false;
    g.start += g.n;
    if (g.seq >= 0) g.n = paged_length(s, g.tile, l.group, l.q, l.kv0);
    return true;
}

// Where a cut at unit u of segment g goes.
TER_HD int paged_snap(const PagedLine& l, const PagedSegment& g, int u) {
    const int off = u - g.start;
    if (g.lead == 0) return 2 * off < g.n ? g.start : g.start + g.n;
    return off < g.lead + l.near ? g.start : g.n - off < l.near ? g.start + g.n : u;
}

// The ranges that hold parts of a segment: first .. last, one if it is not cut.
// Range g writes its part to slot 2 g + 1 if the part begins the segment (it is
// then the last of the range), else to slot 2 g.
struct PagedParts {
    int first, last;
};
TER_HD PagedParts paged_parts(const PagedLine& l, int start, int n, int lead) {
    PagedParts p;
    if (lead == 0) {
        p.first = p.last = 0;
        return p;
    }
    // cuts from start + lead + near to start + n - near stay inside
    const int c0 = paged_cut_from(l, start + kPagedLead + l.near), c1 = paged_cut_from(l, start + n - l.near + 1) - 1;
    p.first = c0 - 1;
    p.last = paged_max(c0 - 1, c1);
    return p;
}
TER_HD int paged_slot(const PagedParts& p, int i) { return i == p.first ? 2 * i + 1 : 2 * i; }

}  // namespace terhip
