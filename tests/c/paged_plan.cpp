// The cutting of the paged attention's work (ter_amd/csrc/paged_plan.h) on the
// CPU: every unit of every segment in one range, partial results where the
// joining kernel looks for them, closed forms against plain counting.
#include "../../ter_amd/csrc/paged_plan.h"

#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>

using namespace terhip;

#define CHECK(c)                                                            \
    do {                                                                    \
        if (!(c)) {                                                         \
            std::printf("line %d: %s (case %d)\n", __LINE__, #c, g_case); \
            std::exit(1);                                                   \
        }                                                                   \
    } while (0)

static int g_case = 0;

int main() {
    std::mt19937 r(7);
    auto in = [&](int a, int b) { return a + (int)(r() % (unsigned)(b - a + 1)); };
    for (g_case = 0; g_case < 4000; ++g_case) {
        const int n_seq = in(1, g_case % 7 == 0 ? 60 : 6), nkv = in(1, 4), group = g_case % 3 ? 1 << in(0, 7) : in(1, 128);
        const int cap = 16 * in(0, 200), q = paged_tokens_log2(group);
        CHECK((1 << q) * group <= kPagedRows && (2 << q) * group > kPagedRows);
        std::vector<int> row0(1, in(0, 9) ? 0 : in(-2, 3)), len;
        for (int b = 0; b < n_seq; ++b) {
            row0.push_back(row0.back() + (in(0, 3) ? in(0, 3) : in(0, 700)));
            const int n = row0[b + 1] - row0[b];
            len.push_back(in(0, 5) ? n + in(0, 2500) : in(-5, 300));
            if (in(0, 40) == 0) len.back() = 0x7FFFFFFF;
        }
        const int n_rows = paged_max(0, in(0, 9) ? row0.back() : row0.back() - in(0, 5)) + (in(0, 5) ? 0 : 3);
        const int shared = in(0, 2) ? 0 : 16 * in(0, cap / 16);
        PagedLine l = paged_line(group, q, shared, n_rows, nkv);
        // plain counting
        std::vector<int> before(1, l.prefix_units);
        std::vector<PagedSegment> segs;
        for (int h = 0; h < nkv && shared; ++h)
            for (int t = 0; t < (n_rows + (1 << q) - 1) >> q; ++t)
                segs.push_back({0, kPagedLead + (shared + 63) / 64, -1, h, t, kPagedLead});
        for (int b = 0; b < n_seq; ++b) {
            const PagedSeq s = paged_seq(row0[b], row0[b + 1], len[b], n_rows, cap);
            CHECK(s.r0 >= 0 && s.n >= 0 && s.r0 + s.n <= n_rows);
            int units = 0, tiles = 0;
            for (int i = 0; i < s.n; i += 1 << q, ++tiles) {
                const int last = paged_min(s.n, i + (1 << q)) - 1;
                // enough key tiles for what the last row sees behind the prefix
                const int see = paged_limit(s, last, cap) - shared;
                const int n = paged_key_tiles(s, tiles, q, shared);
                CHECK(n >= 1 && n * 64 >= see);
                if (s.base + last + 1 <= cap) CHECK(n == paged_max(1, (see + 63) / 64));
                CHECK(paged_length_before(s, tiles, q, shared) == units);
                const bool solid = s.n * group <= 16 && tiles == 0 && i + (1 << q) >= s.n && n <= 8;
                CHECK(paged_length(s, tiles, group, q, shared) == (solid ? 1 + (n + 1) / 2 : n + kPagedLead));
                CHECK(solid == paged_solid(s, group, q, shared));
                units += solid ? 1 + (n + 1) / 2 : n + kPagedLead;
            }
            CHECK(tiles == paged_row_tiles(s, q) && units == paged_units(s, group, q, shared));
            for (int h = 0; h < nkv; ++h)
                for (int t = 0; t < tiles; ++t) segs.push_back({0, paged_length(s, t, group, q, shared), b, h, t, paged_solid(s, group, q, shared) ? 0 : kPagedLead});
            before.push_back(before.back() + units * nkv);
        }
        int total = 0;
        for (auto& g : segs) g.start = total, total += g.n;
        CHECK(total == before.back());
        if (!total) continue;
        // (with a skew: workgroups of CUs in rounds, 8 times as many)
        const int skew = in(0, 1) ? in(1, 3) : 0, rounds = in(1, 4), round = in(1, 20);
        const int resident = skew ? 8 * rounds * round : in(1, 600);
        // (fewer than the resident ones where the host knows of less work, whatever the tables hold)
        const int max_wg = in(0, 3) ? resident * in(1, 4) : in(1, resident);
        paged_cut(l, total, {max_wg, resident, in(1, 40), in(1, 4), in(0, 3) ? 1 : in(2, 20), skew, rounds, round});
        CHECK(l.n_wg >= 1 && l.n_wg <= max_wg);
        std::vector<long long> share(1, 0);
        for (int w = 0; w < l.n_wg; ++w) {
            const int r = w / round % rounds;
            share.push_back(share.back() + 16 + (skew && l.n_wg == resident && total >= 4 * resident ? skew * (rounds - 1 - 2 * r) : 0));
        }
        CHECK(share.back() == 16 * l.n_wg);
        for (int w = 0; w <= l.n_wg; ++w) CHECK(paged_cut_at(l, w) == total * share[w] / share.back());
        for (int i = 0; i < 20; ++i) {
            const int u = in(0, total);
            int w = 0;
            while (total * share[w] < u * share.back()) ++w;
            CHECK(paged_cut_from(l, u) == w);
        }
        // the device's way: each range by itself
        std::vector<int> done(total, 0);
        std::map<std::pair<int, int>, int> slots;  // (segment start, range) -> slot
        std::set<int> used;
        auto find = [&](int u) {
            int b = 0;
            while (u >= l.prefix_units && before[b + 1] <= u) ++b;
            return paged_segment(l, u, nkv, b, paged_seq(row0[b], row0[b + 1], len[b], n_rows, cap), before[b],
                                 before[b + 1]);
        };
        auto cut = [&](int g) {
            const int u = paged_cut_at(l, g);
            return u >= total ? total : paged_snap(l, find(u), u);
        };
        size_t k = 0;
        for (int u = 0; u < total; ++u) {
            while (u >= segs[k].start + segs[k].n) ++k;
            if (in(0, 3) && u != segs[k].start) continue;
            const PagedSegment g = find(u);
            CHECK(g.start == segs[k].start && g.n == segs[k].n && g.seq == segs[k].seq && g.kvh == segs[k].kvh &&
                  g.tile == segs[k].tile && g.lead == segs[k].lead);
            PagedSegment next = g;
            const PagedSeq s = g.seq < 0 ? PagedSeq{} : paged_seq(row0[g.seq], row0[g.seq + 1], len[g.seq], n_rows, cap);
            if (paged_advance(l, next, s, nkv)) {
                const PagedSegment& m = segs[k + 1];
                CHECK(next.start == m.start && next.n == m.n && next.seq == m.seq && next.kvh == m.kvh &&
                      next.tile == m.tile && next.lead == m.lead);
            } else {
                CHECK(k + 1 == segs.size() || segs[k + 1].seq != g.seq);
            }
        }
        for (int w = 0; w < l.n_wg; ++w) {
            // as the kernel does: from its cut on, segment by segment
            const int raw0 = paged_cut_at(l, w), raw1 = paged_cut_at(l, w + 1);
            if (raw0 >= total) continue;
            PagedSegment g = find(raw0);
            int u = paged_snap(l, g, raw0);
            if (u == g.start + g.n) {
                if (u >= total) continue;
                g = find(u);
            }
            CHECK(u == cut(w));
            while (u < total) {
                const int e = raw1 >= g.start + g.n ? g.start + g.n : paged_snap(l, g, raw1);
                if (e <= u) break;
                for (int i = u; i < e; ++i) ++done[i];
                CHECK(u == g.start || u > g.start + kPagedLead);
                CHECK(e > g.start + g.lead && (g.lead || (u == g.start && e == u + g.n)));
                if (u > g.start || e < g.start + g.n) {
                    const int slot = u == g.start ? 2 * w + 1 : 2 * w;
                    CHECK(used.insert(slot).second);
                    slots[{g.start, w}] = slot;
                }
                u = e;
                if (u < g.start + g.n || u >= total) break;
                g = find(u);
            }
            CHECK(u == cut(w + 1));
        }
        for (int d : done) CHECK(d == 1);
        size_t seen = 0;
        for (auto& g : segs) {
            const PagedParts p = paged_parts(l, g.start, g.n, g.lead);
            if (p.first == p.last) {
                CHECK(!slots.count({g.start, p.first}));
                continue;
            }
            for (int i = p.first; i <= p.last; ++i, ++seen) {
                CHECK(slots.count({g.start, i}));
                CHECK((slots[{g.start, i}] == paged_slot(p, i)) && paged_slot(p, i) < 2 * l.n_wg);
            }
        }
        CHECK(seen == slots.size());
    }
    std::puts("ok");
    return 0;
}
