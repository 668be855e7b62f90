// hkv_paged.cuh — what the kernels of the paged cache share: element types, the packed batch as the kernels see it,
// and the kernels around attention: block tables and slot maps, release, append, any-geometry attention.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hkv_common.cuh"

namespace hkv {

// ---- element types --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// Two values rounded to nearest and packed, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_half2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));   // bf16 is the upper half of fp32
}

// ---- division by a page size ----------------------------------------------------------------------------------------
// n / d for 0 <= n < 2^31 as a product: with l = ceil(log2 d) and m = floor(2^(31+l) / d) + 1 <= 2^32 - 1 (d > 1), m d is
// above 2^(31+l) by at most 2^l, so n m / 2^(31+l) is above n / d by less than 1 / d.
struct FastDiv {
    uint32_t mul, shift;      // mul 0: d = 1
};
__host__ inline FastDiv fast_div(uint32_t d) {
    if (d == 1) return FastDiv{0, 0};
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    return FastDiv{(uint32_t)((1ull << (31 + l)) / d + 1), l - 1};
}
__device__ __forceinline__ int div_by(const FastDiv f, int n) { return f.mul ? (int)(__umulhi((uint32_t)n, f.mul) >> f.shift) : n; }
__device__ __forceinline__ int ceil_div_by(const FastDiv f, int n) { return n > 0 ? div_by(f, n - 1) + 1 : 0; }

// ---- the packed batch -----------------------------------------------------------------------------------------------
struct PagedBatch {
    const int32_t* table;     // [requests][cols]
    const int32_t* q_start;   // [requests(+1)]
    const int32_t* step_len;
    const int32_t* key_len;   // positions in the cache, the new tokens included (cross attention: encoder states)
    int32_t* status;
    int requests, cols, page, pages;   // page = rows per page
    int tokens, max_step;
    int window;               // 0 = none
    int causal;               // 0: every query attends [0, key_len)
};

// One request, with every value that comes from device memory brought into the range the buffers allow: no array
// content can lead an access out of bounds.
struct PagedRequest {
    int start, n;      // packed rows of its queries
    int pos0;          // position of query 0 (causal); may be negative: such queries attend nothing
    int keys;          // positions held, at most cols * page
};
__host__ __device__ __forceinline__ PagedRequest paged_request(const PagedBatch& a, int r) {
    PagedRequest q;
    q.start = a.q_start[r];
    const int step = a.step_len[r], len = a.key_len[r];
    q.n = step < a.max_step ? step : a.max_step;
    if (q.start < 0 || q.start > a.tokens) q.n = 0;
    else if (q.n > a.tokens - q.start) q.n = a.tokens - q.start;
    if (q.n < 0) q.n = 0;
    const int cap = a.cols * a.page;
    q.keys = len < cap ? (len > 0 ? len : 0) : cap;
    q.pos0 = q.keys - (step > 0 ? step : 0);
    return q;
}
// Keys [lo, hi) that query i of a request attends, 0 <= lo; hi <= lo: none. Lengths may come up to the end of 31 bits
// (whatever the arrays hold, and with max_pages * page_size near it also in earnest), so a bound is never added to: tiles
// are counted as (hi - 1) / rows + 1, and what lies behind a tile or box is asked by a difference.
__host__ __device__ __forceinline__ void paged_key_range(const PagedBatch& a, const PagedRequest& q, int i, int& lo, int& hi) {
    lo = 0;
    hi = q.keys;
    if (a.causal) {
        const int p = q.pos0 + i;
        if (p + 1 < hi) hi = p >= 0 ? p + 1 : 0;
        if (a.window > 0 && p >= a.window) lo = p - a.window + 1;
    }
}
// Whether a tile of `rows` positions from `row0` on holds one that not all of a run of queries attend (their lower bounds
// up to lo_last, their upper ones from hi_first on).
__host__ __device__ __forceinline__ bool paged_tile_masked(int row0, int rows, int lo_last, int hi_first) {
    return row0 < lo_last || hi_first - row0 < rows;
}
// Whether none of `rows` positions from p on is in [lo, hi).
__host__ __device__ __forceinline__ bool paged_box_hidden(int p, int rows, int lo, int hi) { return p >= hi || lo - p >= rows; }

// ---- launches that overlap --------------------------------------------------------------------------------------------
// The dependent launch may be set up from here on; it waits for this one's end before it reads anything.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- scans of a block -----------------------------------------------------------------------------------------------
// Exclusive prefix sum of one value per thread over the block (at most 1024 threads); `total` gets the sum.
// `buf` holds 33 values; ends with the block synchronised.
__device__ __forceinline__ long long block_scan(long long v, long long* buf, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
    }
    if (lane == 31) buf[warp] = x;
    __syncthreads();
    if (warp == 0) {
        long long s = lane < warps ? buf[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        buf[lane] = s;
    }
    __syncthreads();
    const long long before = warp > 0 ? buf[warp - 1] : 0;
    total = buf[warps - 1];
    __syncthreads();
    return before + x - v;
}

// ---- plan -----------------------------------------------------------------------------------------------------------
// Every CTA scans all requests itself (at most four per thread: cheaper than passing sums between CTAs) and leaves their
// starts, lengths and places on the free stack in shared memory, then writes its share of the tables. A packed token
// finds its request by bisection over the starts, a new page by bisection over the places on the stack, so both are dealt
// evenly and read and written in order whatever the lengths. New pages come from the stack directly, so no CTA waits for
// another's table writes. Where lengths or count are updated in place, the CTA that finishes last writes them: every
// other one has read them before it says that it is done.
// Bound: latency — the launch and three dependent trips to memory (lengths, then table or stack entry, then the store).
struct PlanArgs {
    const int32_t *past, *fresh, *free_pages, *free_count;
    int32_t *table, *total, *step, *q_start, *slots, *positions, *free_left;
    int* done;                        // CTAs that have finished; null: nothing is updated in place
    int requests, tokens, cols, page, pages;
    FastDiv by_page;
};
constexpr int kPlanThreads = 1024;
constexpr int kPagedMaxRequests = 4096;
constexpr int kPlanPer = 4;           // requests per thread
__host__ __device__ constexpr size_t plan_smem_bytes(int requests) { return (size_t)(3 * requests + 4) * 4; }

// Exclusive prefix sum over the block, sums held at `cap` (min(a + b, cap) is associative for values up to cap <= 2^31).
__device__ __forceinline__ uint32_t block_scan_cap(uint32_t v, const uint32_t cap, uint32_t* buf, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = min(x + u, cap);
    }
    if (lane == 31) buf[warp] = x;
    __syncthreads();
    // every warp sums the warps before it on its own: one barrier, no second round
    uint32_t w = lane < warps ? buf[lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w = min(w + u, cap);
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    uint32_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    if (warp == 0) before = 0;
    const uint32_t left = __shfl_up_sync(0xffffffffu, x, 1);
    return min(before + (lane > 0 ? left : 0u), cap);
}
// The last index r in [0, n) with key[r] <= x (key[0] <= x), for U values at a time: their dependent reads overlap.
template <int U>
__device__ __forceinline__ void last_at_most(const int32_t* key, const int n, const int (&x)[U], int (&r)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = 0;
    int step = 1;
    while (step < n) step <<= 1;
    for (step >>= 1; step > 0; step >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r[u] + step < n && key[r[u] + step] <= x[u]) r[u] += step;
}

__global__ void __launch_bounds__(kPlanThreads, 1) hkv_paged_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t plan_smem[];
    __shared__ uint32_t buf[2][32];
    __shared__ int s_last;
    __shared__ uint32_t s_taken;                     // pages taken by all admitted requests
    const int R = a.requests, tid = threadIdx.x, threads = blockDim.x;
    int32_t* s_start = plan_smem;                    // [R + 1] first packed row
    int32_t* s_take = s_start + R + 1;               // [R + 1] pages wanted before this request, as far as they are taken
    int32_t* s_past = s_take + R + 1;                // [R] past length; -1: not admitted
    if (tid == 0) s_taken = 0;
    const int per = (R + threads - 1) / threads, r0 = tid * per;
    const uint32_t cap = (uint32_t)a.tokens + 1u;    // beyond the packed rows: further ones do not matter
    int past[kPlanPer], fresh[kPlanPer];
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        past[i] = fresh[i] = 0;
        if (i < per && r0 + i < R) {
            past[i] = a.past[r0 + i];
            fresh[i] = a.fresh[r0 + i];
            sum = min(sum + min((uint32_t)(fresh[i] > 0 ? fresh[i] : 0), cap), cap);
        }
    }
    const int count = *a.free_count, avail = count < a.pages ? count : a.pages;
    uint32_t tokens_all, need_all;
    uint32_t at = block_scan_cap(sum, cap, buf[0], tokens_all);
    uint32_t need[kPlanPer], need_sum = 0;
    bool fits[kPlanPer];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        need[i] = 0;
        fits[i] = false;
        if (i < per && r0 + i < R) {
            s_start[r0 + i] = (int)min(at, (uint32_t)a.tokens);
            const uint32_t end = min(at + min((uint32_t)(fresh[i] > 0 ? fresh[i] : 0), cap), cap);
            const long long len = (long long)past[i] + fresh[i];
            fits[i] = past[i] >= 0 && fresh[i] >= 0 && len <= (long long)a.cols * a.page && end <= (uint32_t)a.tokens;
            if (fits[i]) need[i] = (uint32_t)(ceil_div_by(a.by_page, (int)len) - ceil_div_by(a.by_page, past[i]));
            need_sum += need[i];                     // at most tokens / page + requests in all
            at = end;
        }
    }
    uint32_t before = block_scan_cap(need_sum, 0x7fffffffu, buf[1], need_all);
    // A request that wants pages gets them if all wanted up to and including it are there; those admitted are the first
    // ones that want any, so what they take is the largest such sum.
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        if (i < per && r0 + i < R) {
            const bool ok = fits[i] && (need[i] == 0 || (long long)before + need[i] <= avail);
            s_take[r0 + i] = (int)before;
            s_past[r0 + i] = ok ? past[i] : -1;
            before += need[i];
            if (ok && need[i] > 0) atomicMax(&s_taken, before);
        }
    }
    if (tid == 0) {
        s_start[R] = (int)min(tokens_all, (uint32_t)a.tokens);
        s_take[R] = (int)need_all;
    }
    __syncthreads();

    const int taken = (int)s_taken, gsize = (int)gridDim.x * threads, g = (int)blockIdx.x * threads + tid;
    const int live = s_start[R];
    constexpr int U = 2;
    // new block-table entries: the j-th page off the stack
    for (int j0 = g; j0 < taken; j0 += U * gsize) {
        int x[U], r[U], pg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x[u] = j0 + u * gsize;
            pg[u] = x[u] < taken ? a.free_pages[avail - 1 - x[u]] : 0;
        }
        last_at_most<U>(s_take, R, x, r);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x[u] < taken) {
                const int p = s_past[r[u]];          // (an admitted request: only those hold places below `taken`)
                a.table[(long long)r[u] * a.cols + ceil_div_by(a.by_page, p) + x[u] - s_take[r[u]]] = pg[u];
            }
    }
    // slot and position of every packed token
    for (int t0 = g; t0 < a.tokens; t0 += U * gsize) {
        int x[U], r[U], pos[U], pg[U], in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = t0 + u * gsize;
        if (R > 0) last_at_most<U>(s_start, R, x, r);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            pos[u] = pg[u] = -1;
            in[u] = 0;
            if (x[u] < live) {
                const int p = s_past[r[u]];
                if (p >= 0) {
                    pos[u] = p + x[u] - s_start[r[u]];
                    const int j = div_by(a.by_page, pos[u]), held = ceil_div_by(a.by_page, p);
                    in[u] = pos[u] - j * a.page;
                    pg[u] = j < held ? a.table[(long long)r[u] * a.cols + j] : a.free_pages[avail - 1 - s_take[r[u]] - (j - held)];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x[u] < a.tokens) {
                a.slots[x[u]] = pg[u] >= 0 && pg[u] < a.pages ? pg[u] * a.page + in[u] : -1;
                a.positions[x[u]] = pos[u];
            }
    }
    // per-request outputs: from one CTA, every thread still holds its requests' lengths
    if (a.done) {
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(a.done, 1) == (int)gridDim.x - 1;
            if (s_last) *a.done = 0;
        }
        __syncthreads();
        if (!s_last) return;
    } else if (blockIdx.x != 0) {
        return;
    }
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        if (i < per && r0 + i < R) {
            const int n = s_past[r0 + i] >= 0 ? fresh[i] : 0;
            a.q_start[r0 + i] = s_start[r0 + i];
            a.step[r0 + i] = n;
            a.total[r0 + i] = past[i] + n;
        }
    }
    if (tid == 0) {
        a.q_start[R] = live;
        *a.free_left = avail - taken;
    }
}

// ---- release --------------------------------------------------------------------------------------------------------
struct ReleaseArgs {
    const int32_t *finished, *table;
    int32_t *seq_len, *free_pages, *free_count;
    int requests, cols, page, pages;
};
__global__ void __launch_bounds__(kPlanThreads, 1) hkv_paged_release_kernel(const ReleaseArgs a) {
    extern __shared__ int32_t rel_smem[];            // [R] first place on the stack, [R] pages
    __shared__ long long buf[33];
    const int R = a.requests, tid = threadIdx.x;
    const int per = (R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = tid * per;
    int n[kPlanPer];
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        n[i] = 0;
        if (i < per && r0 + i < R && a.finished[r0 + i]) {
            const int len = a.seq_len[r0 + i];
            const int held = len > 0 ? (int)(((long long)len + a.page - 1) / a.page) : 0;
            n[i] = held < a.cols ? held : a.cols;
            a.seq_len[r0 + i] = 0;                   // this thread alone reads and writes it
        }
        sum += n[i];
    }
    const int count = *a.free_count, have = count > 0 ? (count < a.pages ? count : a.pages) : 0;
    long long all;
    long long at = block_scan(sum, buf, all);
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i)
        if (i < per && r0 + i < R) {
            rel_smem[r0 + i] = (int)at;
            rel_smem[R + r0 + i] = n[i];
            at += n[i];
        }
    __syncthreads();
    const int warp = tid >> 5, lane = tid & 31;
    for (int r = warp; r < R; r += kPlanThreads / 32)
        for (int j = lane; j < rel_smem[R + r]; j += 32) {
            const long long to = (long long)have + rel_smem[r] + j;
            if (to < a.pages) a.free_pages[to] = a.table[(long long)r * a.cols + j];
        }
    if (tid == 0) {
        const long long now = have + all;
        *a.free_count = (int)(now < a.pages ? now : a.pages);
    }
}

// ---- append ---------------------------------------------------------------------------------------------------------
// A warp per token: its K row and its V row are one list of pieces dealt to the lanes, four loads in flight per lane.
// Bound: HBM (each row read once, written once).
struct PagedAppendArgs {
    const void *k, *v;
    void *k_cache, *v_cache;
    const int32_t* slots;
    int32_t* status;
    long long stride;      // elements between tokens
    long long rows;        // pages * page
    int tokens, row_elems;
};
template <typename VecT>
__global__ void __launch_bounds__(256) hkv_paged_append_kernel(const PagedAppendArgs a) {
    constexpr int kPer = (int)(sizeof(VecT) / 2);
    const int lane = threadIdx.x & 31, pieces = a.row_elems / kPer;
    for (long long t = (blockIdx.x * 256ll + threadIdx.x) >> 5; t < a.tokens; t += gridDim.x * 8ll) {
        const int slot = a.slots[t];
        if (slot < 0) continue;
        if (slot >= a.rows) {
            if (lane == 0) atomicOr(a.status, kStatusBoundCheck);
            continue;
        }
        const VecT* src[2] = {reinterpret_cast<const VecT*>((const uint16_t*)a.k + t * a.stride),
                              reinterpret_cast<const VecT*>((const uint16_t*)a.v + t * a.stride)};
        VecT* dst[2] = {reinterpret_cast<VecT*>((uint16_t*)a.k_cache + (long long)slot * a.row_elems),
                        reinterpret_cast<VecT*>((uint16_t*)a.v_cache + (long long)slot * a.row_elems)};
        for (int p0 = lane; p0 < 2 * pieces; p0 += 128) {
            VecT x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int p = p0 + 32 * u;
                if (p < 2 * pieces) x[u] = p < pieces ? src[0][p] : src[1][p - pieces];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int p = p0 + 32 * u;
                if (p < pieces) dst[0][p] = x[u];
                else if (p < 2 * pieces) dst[1][p - pieces] = x[u];
            }
        }
    }
}

// ---- attention, any geometry ----------------------------------------------------------------------------------------
// One CTA of 4 warps per (packed token, query head): warp w takes the keys lo+w, lo+w+4, ..., lanes stride the head
// dimension, online softmax per warp in the log2 domain, the warps merged in shared memory. For what the staged kernels
// do not take (head sizes, page sizes, alignment); every K/V row is read once per query head.
struct PagedAttnArgs {
    PagedBatch b;
    const void *q, *k_cache, *v_cache;
    void* out;
    long long q_stride;
    int H, KVH, HD;
    float scale_log2;
};
constexpr int kPagedGenWarps = 4;
constexpr float kLow = -3.3e38f;          // start of a running maximum: below every score that is finite
// A row sum beyond this comes from a score that is not a number: sums of n probabilities stay below n * 2^8.
constexpr float kSumLimit = 1.0e30f;

// One output row: query i of request r (packed row t), head h. The whole block of WARPS warps takes part.
template <typename T, int WARPS>
__device__ __forceinline__ void paged_row(const PagedAttnArgs& a, const int r, const PagedRequest& rq, const int i, const int h) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t = rq.start + i;
    int k_lo, k_hi;
    paged_key_range(a.b, rq, i, k_lo, k_hi);
    const int kvh = h / (a.H / a.KVH);
    const T* qp = (const T*)a.q + t * a.q_stride + (long long)h * a.HD;
    float qr[16], acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int d = lane + 32 * e;
        qr[e] = d < a.HD ? to_f32(qp[d]) : 0.0f;
        acc[e] = 0.0f;
    }
    float m = kLow, l = 0.0f;
    const int32_t* table = a.b.table + (long long)r * a.b.cols;
    for (uint32_t s = (uint32_t)k_lo + warp; s < (uint32_t)k_hi; s += WARPS) {
        const int pg = table[s / (uint32_t)a.b.page];
        const bool in = pg >= 0 && pg < a.b.pages;   // an entry outside the planes: rows of zeros
        if (!in && lane == 0) atomicOr(a.b.status, kStatusBoundCheck);
        const long long row = (((long long)(in ? pg : 0) * a.b.page + s % (uint32_t)a.b.page) * a.KVH + kvh) * a.HD;
        const T* kr = (const T*)a.k_cache + row;
        const T* vr = (const T*)a.v_cache + row;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = lane + 32 * e;
            if (in && d < a.HD) dot = fmaf(qr[e], to_f32(kr[d]), dot);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float sc = dot * a.scale_log2;
        const float mn = fmaxf(m, sc);
        const float corr = exp2f(m - mn), e2 = exp2f(sc - mn);
        l = l * corr + e2;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = lane + 32 * e;
            if (d < a.HD) acc[e] = fmaf(e2, in ? to_f32(vr[d]) : 0.0f, acc[e] * corr);
        }
        m = mn;
    }
    __shared__ float s_m[WARPS], s_l[WARPS];
    __shared__ float s_acc[WARPS][512];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int e = 0; e < 16; ++e) s_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    float gm = s_m[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) gm = fmaxf(gm, s_m[w]);
    float gl = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) gl += s_l[w] * exp2f(s_m[w] - gm);
    const float inv = gl > 0.0f ? 1.0f / gl : 0.0f;
    T* op = (T*)a.out + (t * a.H + h) * a.HD;
    for (int d = threadIdx.x; d < a.HD; d += WARPS * 32) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) o += s_acc[w][d] * exp2f(s_m[w] - gm);
        op[d] = from_f32<T>(o * inv);
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kPagedGenWarps * 32) hkv_paged_generic_kernel(const PagedAttnArgs a) {
    const int t = blockIdx.x;
    int lo = 0, hi = a.b.requests - 1;               // the last request that starts at or before t
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.b.q_start[mid] <= t) lo = mid; else hi = mid - 1;
    }
    PagedRequest rq = paged_request(a.b, lo);
    // An empty request may start on or inside the rows of one before it: the nearest that has rows, 32 at a time, as far
    // back as max_step rows reach.
    while (rq.n == 0) {
        if (lo == 0 || (long long)a.b.q_start[lo - 1] + a.b.max_step <= t) return;
        const int r = lo - 1 - (int)(threadIdx.x & 31);
        const unsigned some = __ballot_sync(0xffffffffu, r >= 0 && paged_request(a.b, r).n > 0);
        lo = some ? lo - __ffs(some) : (lo > 32 ? lo - 32 : 0);
        rq = paged_request(a.b, lo);
    }
    const int i = t - rq.start;
    if (i < 0 || i >= rq.n) return;                  // a row of no query
    paged_row<T, kPagedGenWarps>(a, lo, rq, i, blockIdx.y);
}

// Work to be done again: the staged kernels drop values of V that are not finite where only some queries of an item look
// (0 * NaN would reach the others) and leave the item here. An item is a block of queries of a request and KV head;
// block -1: all its queries. More items than the list holds: every row of the call is done again.
constexpr int kFixMax = 1020;
struct PagedFix {
    int* head;        // items; CTAs done
    int4* items;      // [kFixMax]
    __device__ __forceinline__ void push(int r, int block, int kvh) const {
        const int at = atomicAdd(head, 1);
        if (at < kFixMax) items[at] = make_int4(r, block, kvh, 0);
        else atomicMin(head, 2 * kFixMax);   // (the count stays far from its range's end)
    }
};

// Whether an item is on the list of `count` entries.
__device__ __forceinline__ bool paged_to_fix(const PagedFix& f, const int count, const int r, const int block, const int kvh) {
    if (count > kFixMax) return true;
    for (int e = 0; e < count; ++e) {
        const int4 x = f.items[e];
        if (x.x == r && x.y == block && x.z == kvh) return true;
    }
    return false;
}
// The rows of the listed items, key by key, so that each query sees exactly its own keys; all blocks of the grid take
// part, the last one to finish empties the list. Blocks of WARPS warps; only called where count > 0.
template <typename T, int WARPS>
__device__ __noinline__ void paged_fix_rows(const PagedAttnArgs& a, const PagedFix& fix, const int count, const int QB) {
    const int G = a.H / a.KVH;
    if (count <= kFixMax) {
        for (int e = 0; e < count; ++e) {
            const int4 item = fix.items[e];
            if (item.x >= a.b.requests) continue;    // left behind by a call whose second launch failed
            const PagedRequest rq = paged_request(a.b, item.x);
            const int i0 = item.y < 0 ? 0 : item.y * QB, i1 = item.y < 0 || i0 + QB > rq.n ? rq.n : i0 + QB;
            for (int x = blockIdx.x; x < (i1 - i0) * G; x += gridDim.x) paged_row<T, WARPS>(a, item.x, rq, i0 + x / G, item.z * G + x % G);
        }
    } else {
        for (int r = 0; r < a.b.requests; ++r) {
            const PagedRequest rq = paged_request(a.b, r);
            for (long long x = blockIdx.x; x < (long long)rq.n * a.H; x += gridDim.x) paged_row<T, WARPS>(a, r, rq, (int)(x / a.H), (int)(x % a.H));
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(fix.head + 1, 1) == (int)gridDim.x - 1) {
        fix.head[1] = 0;
        *reinterpret_cast<volatile int*>(fix.head) = 0;
    }
}

}  // namespace hkv
