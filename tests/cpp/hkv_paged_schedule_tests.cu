// hkv_paged_schedule_tests.cu — the host-callable arithmetic behind the paged attention kernels' schedules, run on the CPU
// (no device call): which keys a query sees, which tiles a request has, at lengths up to the end of 31 bits.
#include <algorithm>
#include <cstdint>
#include <cstdio>
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

int main() {
    test_tile_and_box_bounds();
    test_far_lengths();
    test_units_fit();
    std::printf(g_failures ? "%d FAILED\n" : "ALL PASSED\n", g_failures);
    return g_failures ? 1 : 0;
}
