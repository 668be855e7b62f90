// hkv_paged_line.cuh — the work of one ragged prompt call as a line: items (request, KV head, block of queries) with the
// keys each spans, cut into equal contiguous spans, one per CTA. Everything follows from the device-side lengths; every
// CTA finds its own span by bisection, and neighbours compute the same cut.
//
// The cost of an item is its keys plus a constant for what a piece of work costs besides (pipeline fill, query load,
// output). Within a request and KV head the costs of consecutive blocks grow linearly until a window caps them, so their
// prefix sums have a closed form and no table over blocks is needed: one entry per request is kept in shared memory.
#pragma once

#include "hkv_paged.cuh"

namespace hkv {

constexpr int kLineOverhead = 256;        // cost of an item besides its keys, in keys
constexpr int kLineUnit = 128;            // the table counts units of 128 << shift keys
// Shortest span. An item of nt >= 2 tiles costs at most 128 nt + 640 (its keys, rounding to blocks and tiles, the
// constant), so cuts 512 apart fall on different tiles of it, and every span inside an item holds at least one.
constexpr int kLineSpanUnits = 4;

struct PagedLine {
    int G, KVH, QB;           // query heads per KV head; KV heads; queries per item
    int keys;                 // positions per key tile
    int shift;
    int ctas;
    const uint32_t* pre;      // shared memory: [requests + 1] units before each request
};

// The table's shift for the largest batch a context allows (requests, tokens and positions per request): at most 10^9 units.
inline int line_shift(double positions, double tokens, double requests, int KVH, int QB) {
    const double units = (tokens / QB + requests) * KVH * ((positions + kLineOverhead + QB) / kLineUnit + 1.0);
    int shift = 0;
    while (units / (double)(1ll << shift) > 1.0e9) ++shift;
    return shift;
}
// Whether a batch's units fit the table. They do where the requests' rows lie apart; arrays in which they overlap (starts
// left at zero, say) can ask for thousands of times the context's tokens, and sums that wrapped would send the bisections
// below to requests without work, whose cost of 0 no division ends on.
__host__ __device__ inline bool line_fits(long long units) { return units >= 0 && units <= 0x7fffffffll; }

struct LineCut { int r, kvh, p, t; };     // request, KV head, block of queries, key tile inside the item

__host__ __device__ inline int line_blocks(int n, int QB) { return (n + QB - 1) / QB; }

// Sum of the costs of the first p blocks of a request and KV head.
__host__ __device__ inline long long line_prefix(const PagedLine& l, int window, int causal, const int pos0, const int keys, const int p) {
    if (!causal) return p * ((long long)keys + kLineOverhead);
    // blocks that end before position 0 attend nothing; then base + (i + 1) * QB keys, up to the cap
    const long long none = pos0 < 0 ? (-(long long)pos0 / l.QB < p ? -(long long)pos0 / l.QB : p) : 0;
    const long long base = pos0 + none * l.QB, rest = p - none;
    long long grow = rest, cap = 0;
    if (window > 0) {
        cap = (long long)window + l.QB + kLineUnit;
        const long long g = cap > base ? (cap - base) / l.QB : 0;
        if (g < grow) grow = g;
    }
    return p * (long long)kLineOverhead + grow * base + l.QB * (grow * (grow + 1) / 2) + (rest - grow) * cap;
}

// Key tiles of a block: at least one, so that rows that attend nothing are written too.
__host__ __device__ __forceinline__ void line_tiles(const PagedBatch& b, const PagedLine& l, const PagedRequest& q, int p, int& kt0, int& nt) {
    int lo, hi, lo2, hi2;
    const int i0 = p * l.QB, i1 = (i0 + l.QB < q.n ? i0 + l.QB : q.n) - 1;
    paged_key_range(b, q, i0, lo, hi);
    paged_key_range(b, q, i1, lo2, hi2);
    kt0 = lo / l.keys;
    nt = hi2 > lo ? (hi2 - 1) / l.keys + 1 - kt0 : 1;
}

// Units of a request on the line, all KV heads.
__host__ __device__ __forceinline__ long long line_units(const PagedBatch& b, const PagedLine& l, const PagedRequest& q) {
    const long long s = line_prefix(l, b.window, b.causal, q.pos0, q.keys, line_blocks(q.n, l.QB)) * l.KVH;
    const long long unit = (long long)kLineUnit << l.shift;
    return (s + unit - 1) / unit;
}

// floor(x / d): a 64-bit division costs a hundred instructions in front of a CTA's first load; the 32-bit estimate is off by
// one at most below 2^22 and by a few at the largest quotients (2^24 tiles).
__host__ __device__ __forceinline__ int line_div(const long long x, const long long d) {
    long long q = (long long)((float)x / (float)d);
    while (q * d > x) --q;
    while ((q + 1) * d <= x) ++q;
    return (int)q;
}

// The cut at unit u of the line (W units in all). A cut that would fall behind an item's last tile is the start of the
// next item; u = W is the cut behind everything ({requests, 0, 0, 0}).
__host__ __device__ __forceinline__ LineCut line_locate(const PagedBatch& b, const PagedLine& l, const uint32_t u, const uint32_t W) {
    LineCut c{b.requests, 0, 0, 0};
    if (u >= W) return c;
    int lo = 0, hi = b.requests - 1;      // the last request that starts at or before u
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.pre[mid] <= u) lo = mid; else hi = mid - 1;
    }
    const PagedRequest q = paged_request(b, lo);
    const int P = line_blocks(q.n, l.QB);
    const long long per = line_prefix(l, b.window, b.causal, q.pos0, q.keys, P);
    long long x = (long long)(u - l.pre[lo]) * ((long long)kLineUnit << l.shift);
    c.r = lo;
    c.kvh = line_div(x, per);
    if (c.kvh >= l.KVH) { c.r = lo + 1; c.kvh = 0; return c; }     // rounding at the request's end
    x -= (long long)c.kvh * per;
    int p0 = 0, p1 = P - 1;
    while (p0 < p1) {
        const int mid = (p0 + p1 + 1) >> 1;
        if (line_prefix(l, b.window, b.causal, q.pos0, q.keys, mid) <= x) p0 = mid; else p1 = mid - 1;
    }
    c.p = p0;
    const long long at = line_prefix(l, b.window, b.causal, q.pos0, q.keys, p0);
    const long long cost = line_prefix(l, b.window, b.causal, q.pos0, q.keys, p0 + 1) - at;
    int kt0, nt;
    line_tiles(b, l, q, p0, kt0, nt);
    c.t = line_div((x - at) * nt + cost / 2, cost);
    if (c.t >= nt) {
        c.t = 0;
        if (++c.p == P) {
            c.p = 0;
            if (++c.kvh == l.KVH) { c.kvh = 0; c.r = lo + 1; }
        }
    }
    return c;
}
__host__ __device__ __forceinline__ bool line_same_item(const LineCut& a, const LineCut& b) { return a.r == b.r && a.kvh == b.kvh && a.p == b.p; }
__host__ __device__ __forceinline__ bool line_before(const LineCut& a, const LineCut& b) {
    if (a.r != b.r) return a.r < b.r;
    if (a.kvh != b.kvh) return a.kvh < b.kvh;
    if (a.p != b.p) return a.p < b.p;
    return a.t < b.t;
}
// CTAs that share W units.
__host__ __device__ inline int line_ctas(uint32_t W, int grid) {
    const uint32_t c = W / kLineSpanUnits;
    return c < 1 ? 1 : (c < (uint32_t)grid ? (int)c : grid);
}
__host__ __device__ inline uint32_t line_boundary(uint32_t W, int ctas, int c) { return (uint32_t)((uint64_t)W * c / ctas); }

}  // namespace hkv
