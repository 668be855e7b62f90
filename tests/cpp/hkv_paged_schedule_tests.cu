// hkv_paged_schedule_tests.cu — the host-callable arithmetic behind the paged attention kernels' schedules, run on the CPU
// (no device call): which keys a query sees, which tiles a request has, at lengths up to the end of 31 bits; how a ragged batch is cut into spans.
#include <algorithm>
#include <array>
#include <cstdint>
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "hkv_paged_decode.cuh"
#include "hkv_paged_line.cuh"

using namespace hkv;

static int g_failures = 0;
#define REQUIRE(cond, ...)                                \
    do {                                                  \
        if (!(cond) && ++g_failures <= 20) {              \
            std::printf("FAIL: %s: ", #cond);             \
            std::printf(__VA_ARGS__);                     \
            std::printf(" (%s:%d)\n", __FILE__, __LINE__); \
        }                                                 \
    } while (0)

static void passed(const char* what) {
    static int before = 0;
    std::printf("%s: %s\n", g_failures == before ? "PASS" : "FAILED", what);
    before = g_failures;
}

// A batch over host arrays, as the kernels get it over device arrays.
struct Host {
    std::vector<int32_t> start, step, len;
    PagedBatch b{};
    Host(std::vector<int32_t> s, std::vector<int32_t> n, std::vector<int32_t> k, int cols, int page, int tokens, int max_step, int window,
         bool causal)
        : start(std::move(s)), step(std::move(n)), len(std::move(k)) {
        b.q_start = start.data();
        b.step_len = step.data();
        b.key_len = len.data();
        b.requests = (int)start.size();
        b.cols = cols;
        b.page = page;
        b.pages = 1;
        b.tokens = tokens;
        b.max_step = max_step;
        b.window = window;
        b.causal = causal;
    }
};

// Keys [lo, hi) of query i in 64 bits; none: lo = hi = 0.
static void model_range(const PagedBatch& b, int64_t keys, int64_t step, int64_t i, int64_t& lo, int64_t& hi) {
    const int64_t p = b.causal ? keys - step + i : keys - 1;
    lo = b.causal && b.window > 0 ? std::max<int64_t>(0, p + 1 - b.window) : 0;
    hi = p + 1;
    if (hi <= lo) lo = hi = 0;
}

static void test_tile_and_box_bounds() {
    std::vector<int> at = {0, 1, 7, 8, 63, 64, 65, 127, 128, 1000};
    for (int d : {8, 9, 16, 64, 72, 128, 129, 1000}) at.push_back((int)((1ll << 31) - d));
    for (int rows : {8, 64, 128})
        for (int p : at)
            for (int lo : at)
                for (int hi : at) {
                    const int64_t p0 = p / rows * rows;
                    REQUIRE(paged_tile_masked((int)p0, rows, lo, hi) == (p0 < lo || p0 + rows > hi), "row %lld of %d, %d, %d", (long long)p0, rows, lo, hi);
                    REQUIRE(paged_box_hidden((int)p0, rows, lo, hi) == (p0 >= hi || p0 + rows <= lo), "box %lld of %d, %d, %d", (long long)p0, rows, lo, hi);
                }
    passed("tile and box bounds");
}

static void test_far_lengths() {
    const int page = 8, cols = (int)((1ll << 31) / 8 - 1);            // 2^31 - 8 positions
    std::vector<int32_t> keys;
    for (int d : {8, 9, 15, 16, 63, 64, 65, 66, 71, 72, 127, 128, 129, 135, 136, 191, 192, 200, 256, 1000}) keys.push_back((int)((1ll << 31) - d));
    for (int k : {0, 1, 63, 64, 65, 300, 5000}) keys.push_back(k);
    for (int k : keys)
        for (int step : {1, 2, 40, 300, 0x7fffffff})
            for (int window : {0, 1, 100, 1024, 0x7fffffff})
                for (bool causal : {true, false}) {
                    const Host h({0}, {step}, {k}, cols, page, 300, 300, window, causal);
                    const PagedRequest q = paged_request(h.b, 0);
                    REQUIRE(q.n == std::min(step, 300) && q.keys == k, "%d %d", step, k);
                    int64_t first = 0, end = 0;
                    for (int i : {0, q.n / 2, q.n - 1}) {
                        int lo, hi;
                        paged_key_range(h.b, q, i, lo, hi);
                        int64_t mlo, mhi;
                        model_range(h.b, k, step, i, mlo, mhi);
                        if (mhi > 0) REQUIRE(lo == mlo && hi == mhi, "%d..%d, wanted %lld..%lld", lo, hi, (long long)mlo, (long long)mhi);
                        else REQUIRE(hi <= lo, "%d..%d of no key (keys %d step %d window %d)", lo, hi, k, step, window);
                        if (i == 0) first = mlo;
                        if (i == q.n - 1) end = mhi;
                    }
                    int tile, n;
                    paged_tiles(h.b, q, tile, n);
                    REQUIRE(n >= 1, "%d tiles (keys %d step %d window %d)", n, k, step, window);
                    if (end > 0)
                        REQUIRE(tile == first / kTileRows && (int64_t)(tile + (int64_t)n) * kTileRows >= end && (int64_t)(tile + (int64_t)n - 1) * kTileRows < end,
                                "tiles %d + %d for keys %lld..%lld", tile, n, (long long)first, (long long)end);
                    for (int tk : {64, 128}) {
                        PagedLine l{};
                        l.G = 1; l.KVH = 1; l.QB = 256; l.keys = tk;
                        for (int p = 0; p < line_blocks(q.n, l.QB); ++p) {
                            line_tiles(h.b, l, q, p, tile, n);
                            int64_t x;
                            model_range(h.b, k, step, (int64_t)p * l.QB, first, x);
                            model_range(h.b, k, step, std::min(q.n, (p + 1) * l.QB) - 1, x, end);
                            REQUIRE(n >= 1, "%d tiles of block %d (keys %d step %d window %d)", n, p, k, step, window);
                            if (end > 0)
                                REQUIRE(tile == first / tk && (int64_t)(tile + (int64_t)n) * tk >= end && (int64_t)(tile + (int64_t)n - 1) * tk < end,
                                        "tiles %d + %d for keys %lld..%lld", tile, n, (long long)first, (long long)end);
                            // a block costs its keys and a constant, and not more than the constant, a block and the keys
                            const long long cost = line_prefix(l, h.b.window, h.b.causal, q.pos0, q.keys, p + 1) - line_prefix(l, h.b.window, h.b.causal, q.pos0, q.keys, p);
                            REQUIRE(cost >= kLineOverhead + std::max<int64_t>(0, end - first) - l.QB &&
                                        cost <= kLineOverhead + (int64_t)l.QB + kLineUnit + std::min<int64_t>(k, causal && window ? (int64_t)window : k),
                                    "cost %lld of block %d (keys %d step %d window %d)", cost, p, k, step, window);
                        }
                    }
                }
    passed("lengths up to 2^31 - 8");
}

// The table of one launch, as the kernels fill it in; returns the units of all in 64 bits.
static long long fill(const PagedBatch& b, const PagedLine& l, int small, std::vector<uint32_t>& pre) {
    pre.assign(b.requests + 1, 0);
    long long at = 0;
    for (int r = 0; r < b.requests; ++r) {
        const PagedRequest q = paged_request(b, r);
        pre[r] = (uint32_t)at;
        at += q.n > 0 && !paged_is_small(q, l.G, small) ? line_units(b, l, q) : 0;
    }
    pre[b.requests] = (uint32_t)at;
    return at;
}

// The units of the largest batches that contexts allow fit 31 bits; overlapping rows are told from them.
static void test_units_fit() {
    std::vector<uint32_t> pre;
    for (int requests : {1, 7, 300, 4096})
        for (int tokens : {1, 5000, 131072, 1 << 24})
            for (int cols : {1, 8192, (int)((1ll << 31) / 16 - 1)})
                for (int KVH : {1, 8, 128})
                    for (int G : {1, 7, 16, 128})
                        for (bool causal : {true, false}) {
                            PagedLine l{};
                            l.G = G; l.KVH = KVH; l.QB = 2 * (128 / G); l.keys = 128;
                            l.shift = line_shift((double)cols * 16, tokens, requests, KVH, l.QB);
                            // all tokens dealt evenly; all in the last request; one each and the rest in the first
                            for (int deal = 0; deal < 3; ++deal) {
                                std::vector<int32_t> start(requests), step(requests), len(requests, cols * 16);
                                int at = 0;
                                for (int r = 0; r < requests; ++r) {
                                    step[r] = deal == 0 ? tokens / requests : deal == 1 ? (r + 1 == requests ? tokens : 0)
                                            : r == 0 ? std::max(0, tokens - requests + 1) : (tokens >= requests ? 1 : 0);
                                    start[r] = at;
                                    at += step[r];
                                }
                                const Host h(start, step, len, cols, 16, tokens, tokens, 0, causal);
                                const long long units = fill(h.b, l, 0, pre);
                                REQUIRE(line_fits(units) && units <= 1100000000ll, "%lld units (%d requests, %d tokens, %d pages)", units, requests, tokens, cols);
                            }
                        }
    // 4 096 requests that all start at row 0 and all have 16k tokens: beyond 32 bits, refused
    PagedLine l{};
    l.G = 4; l.KVH = 8; l.QB = 64; l.keys = 128;
    l.shift = line_shift(131072.0, 16384, 4096, 8, 64);
    const Host h(std::vector<int32_t>(4096, 0), std::vector<int32_t>(4096, 16384), std::vector<int32_t>(4096, 131072), 8192, 16, 16384, 16384, 0, true);
    const long long units = fill(h.b, l, 0, pre);
    REQUIRE(units > 0xffffffffll && !line_fits(units), "%lld units", units);
    passed("units of the largest batches, and of overlapping ones");
}

// Random ragged batches cut into spans: every key tile of every item is in exactly one piece, a piece that is not a whole
// item lies in the workspace slot that the finishing kernel's entry for the item points at, and no slot is used twice.
static void test_spans() {
    std::mt19937 rng(31);
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    std::vector<uint32_t> pre;
    long long batches = 0, pieces = 0, cut_items = 0;
    for (int round = 0; round < 1500; ++round) {
        const int R = round % 5 == 0 ? pick(1, 3) : pick(1, 60), page = 1 << pick(3, 8);
        const bool causal = rng() % 3 != 0, wide = rng() % 2;
        const int G = std::vector<int>{1, 2, 3, 7, 8, 16, 40, 128}[rng() % 8], KVH = pick(1, 9);
        const int window = rng() % 2 ? 0 : pick(1, 2000), most = std::vector<int>{1, 20, 600, 5000}[rng() % 4];
        std::vector<int32_t> start(R), step(R), len(R);
        int at = 0, longest = 1;
        for (int r = 0; r < R; ++r) {
            step[r] = rng() % 6 == 0 ? 0 : pick(1, most);
            len[r] = rng() % 8 == 0 ? pick(0, 50) : step[r] + pick(0, rng() % 3 ? 3000 : 60000);
            start[r] = at;
            at += step[r];
            longest = std::max(longest, (int)len[r]);
        }
        const Host h(start, step, len, (longest + page - 1) / page, page, std::max(at, 1), most, window, causal);
        PagedLine l{};
        l.G = G; l.KVH = KVH; l.QB = (wide ? 1 : 2) * (128 / G); l.keys = wide ? 64 : 128;
        l.shift = line_shift((double)h.b.cols * page, h.b.tokens, R, KVH, l.QB);
        const int small = rng() % 2 ? 0 : G <= 8 ? 8 / G * G : G;
        const uint32_t W = (uint32_t)fill(h.b, l, small, pre);
        l.pre = pre.data();
        const int grid = std::vector<int>{148, 148, 148, 7, 1}[rng() % 5], ctas = line_ctas(W, grid);
        struct Piece { int cta, t0, t1, slot; };
        std::map<std::array<int, 3>, std::vector<Piece>> items;
        std::vector<LineCut> cut(ctas + 1);
        for (int c = 0; c <= ctas; ++c) cut[c] = line_locate(h.b, l, line_boundary(W, ctas, c), W);
        for (int cta = 0; cta < ctas && W > 0; ++cta) {          // as the producers walk
            LineCut c = cut[cta];
            const LineCut e = cut[cta + 1];
            while (c.r < R && line_before(c, e)) {
                if (pre[c.r + 1] == pre[c.r]) { ++c.r; c.kvh = c.p = c.t = 0; continue; }
                const PagedRequest q = paged_request(h.b, c.r);
                int kt0, nt;
                line_tiles(h.b, l, q, c.p, kt0, nt);
                const int end = line_same_item(c, e) ? e.t : nt;
                if (end > c.t) items[{c.r, c.kvh, c.p}].push_back({cta, c.t, end, c.t == 0 && end == nt ? -1 : 2 * cta + (c.t == 0 ? 1 : 0)});
                c.t = 0;
                if (++c.p >= line_blocks(q.n, l.QB)) {
                    c.p = 0;
                    if (++c.kvh == l.KVH) { c.kvh = 0; ++c.r; }
                }
            }
        }
        std::map<std::array<int, 3>, std::pair<int, int>> entries;   // item -> first CTA, parts (as the entries are written)
        for (int cta = 0; cta < ctas; ++cta) {
            const LineCut c0 = cut[cta], c1 = cut[cta + 1];
            if (c1.r >= R || c1.t == 0 || (line_same_item(c0, c1) && c0.t > 0)) continue;
            int parts = 2;
            for (int c = cta + 2; c < ctas && line_same_item(cut[c], c1) && cut[c].t > 0; ++c) ++parts;
            entries[{c1.r, c1.kvh, c1.p}] = {cta, parts};
        }
        std::set<int> slots;
        size_t expected = 0;
        for (int r = 0; r < R; ++r) {
            const PagedRequest q = paged_request(h.b, r);
            if (q.n == 0 || paged_is_small(q, G, small)) continue;
            for (int kvh = 0; kvh < KVH; ++kvh)
                for (int p = 0; p < line_blocks(q.n, l.QB); ++p, ++expected) {
                    int kt0, nt, t = 0;
                    line_tiles(h.b, l, q, p, kt0, nt);
                    const auto it = items.find({r, kvh, p});
                    REQUIRE(it != items.end(), "item %d %d %d has no piece", r, kvh, p);
                    if (it == items.end()) continue;
                    const auto en = entries.find({r, kvh, p});
                    for (size_t i = 0; i < it->second.size(); ++i) {
                        const Piece& x = it->second[i];
                        REQUIRE(x.t0 == t, "item %d %d %d: tile %d after %d", r, kvh, p, x.t0, t);
                        t = x.t1;
                        if (it->second.size() == 1) REQUIRE(x.slot == -1 && en == entries.end(), "a whole item with a slot or an entry");
                        else REQUIRE(en != entries.end() && x.cta == en->second.first + (int)i && x.slot == 2 * x.cta + (i == 0) && slots.insert(x.slot).second,
                                     "item %d %d %d: piece %d in CTA %d, slot %d", r, kvh, p, (int)i, x.cta, x.slot);
                        ++pieces;
                    }
                    REQUIRE(t == nt, "item %d %d %d: %d of %d tiles", r, kvh, p, t, nt);
                    if (en != entries.end()) {
                        REQUIRE(en->second.second == (int)it->second.size(), "item %d %d %d: %d parts of %d", r, kvh, p, en->second.second, (int)it->second.size());
                        ++cut_items;
                    }
                }
        }
        REQUIRE(items.size() == expected, "%d items of %d", (int)items.size(), (int)expected);
        ++batches;
    }
    REQUIRE(batches == 1500 && pieces > 40000 && cut_items > 4000, "%lld pieces, %lld cut items", pieces, cut_items);
    passed("spans of random batches");
}

int main() {
    test_tile_and_box_bounds();
    test_far_lengths();
    test_units_fit();
    test_spans();
    std::printf(g_failures ? "%d FAILED\n" : "ALL PASSED\n", g_failures);
    return g_failures ? 1 : 0;
}
