// hkv_paged_decode.cuh — attention of a few new tokens per request over a paged cache: requests with step_len * group
// <= 16 query rows per KV head (one token at group sizes up to 16, two at 8, sixteen without grouping).
//
// Bound: HBM — every K and V row of a request is read once, for all query rows of its KV head together.
//   * The 64-position tiles of all requests form one line that is cut into equal contiguous spans, one per gang of CTAs
//     (a gang = neighbouring CTAs with one share of the KV heads each, so that whole cache rows are streamed together):
//     every CTA does the same number of tiles whatever the lengths. The lengths are read on the device.
//   * One producer warp fills a ring of stages with bulk-tensor copies. A tile is 64 / min(page, 64) pieces, each a box
//     of min(page, 64) rows of one page; the lanes look up one page each and issue their boxes side by side, so a tile of
//     small pages costs no more issue time than one box. Positions that no query looks at and entries outside the planes are
//     fetched from a coordinate behind the tensor: the copy engine writes zeros and reads nothing.
//   * Four consumer warps per tile, 16 rows each:  S^T = K Q^T  and  O^T += V^T P^T  with mma.m16n8k16, the query rows in
//     N (8 or 16), K and V by ldmatrix, P^T from the score fragment by movmatrix; softmax over rows by shuffles, with a
//     running maximum and sum in 32 bits. P is rounded to the element type for the second product (its sum is not), the
//     usual choice: it keeps the product on the tensor cores and costs half a step of the type (against 64 bits 2.4e-4 to
//     2.9e-4 of a row in fp16 where its rounding alone is 2.0e-4, 2.1e-3 to 2.3e-3 against 1.6e-3 in bf16).
//   * A request inside one span is finished here. One that is cut leaves a partial row (o, maximum, sum) per span; a span
//     has at most two (its first and its last request), so the workspace does not grow with the batch. The
//     finishing kernel joins them.
//   * Measured: 64 requests of 16k to 32k keys, 28 heads of 4, 128 wide, 16-row pages: 470 us (7.0 TB/s); 60 windows of
//     1 024 keys, 8 KV heads 256 wide: 88 us (5.7 TB/s); 32 requests of 1 500 keys, 16 heads 64 wide: 33 us (4.4 TB/s), of
//     which 8 us are the two launches. With a copy per column block 8-row pages took 222 us where 64-row pages took 171,
//     now 182 us: a copy costs some 50 ns whatever it brings.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "hkv_paged.cuh"

namespace hkv {

constexpr int kSmallCols = 16;            // query rows per KV head this kernel takes (two n8 tiles)
constexpr int kPagedMaxStages = 8;
constexpr int kReqCache = 64;             // requests of a span kept in shared memory

__host__ __device__ constexpr int paged_chunk_width(int HD) { return HD % 64 == 0 ? 64 : 32; }

struct PagedDecodeArgs {
    PagedAttnArgs t;
    float* part;          // [2 * spans][KVH][cols][HD + 2]: o, maximum (log2 domain), sum
    int4* cuts;           // [spans]: request that starts in this span and goes on behind it: {request, spans, first packed row, queries}; spans 0: none
    PagedFix fix;
    int gang, cols;       // cols = query rows per KV head that the partial rows hold
    int box_rows, pieces; // rows of a box, boxes per tile and column block
};

// Tiles of a request on the line: at least one for every request with queries, so that rows that attend nothing are
// written too.
__host__ __device__ __forceinline__ void paged_tiles(const PagedBatch& b, const PagedRequest& q, int& tile_lo, int& n_tiles) {
    int lo, hi, lo2, hi2;
    paged_key_range(b, q, 0, lo, hi);
    paged_key_range(b, q, q.n - 1, lo2, hi2);
    tile_lo = lo / kTileRows;
    n_tiles = hi2 > lo ? (hi2 - 1) / kTileRows + 1 - tile_lo : 1;
}
// Whether the few-token kernel (this file) takes a request: at most `limit` query rows per KV head.
__host__ __device__ __forceinline__ bool paged_is_small(const PagedRequest& q, int G, int limit) { return q.n > 0 && (long long)q.n * G <= limit; }

template <typename T>
__device__ __forceinline__ void mma_16816_t(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816_t<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16816_t<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Replaces the values of 8 packed elements that are not finite by zero; true if there was one.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint4& x) {
    const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;   // exponent bits
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & e) == e) { w[i] &= 0xffff0000u; bad = true; }
        if (((w[i] >> 16) & e) == e) { w[i] &= 0x0000ffffu; bad = true; }
    }
    x = make_uint4(w[0], w[1], w[2], w[3]);
    return bad;
}

struct PagedDecodePlan { int stages; size_t bytes; };
inline PagedDecodePlan paged_decode_plan(int HD, int cols, int ncw, int requests, size_t budget) {
    const size_t stage = 2ull * kTileRows * HD * 2;
    const size_t fixed = 1024 + (size_t)ncw * cols * (HD + 4) * 4 + (size_t)ncw * cols * 2 * 4 + 2 * kPagedMaxStages * 8 +
                         (size_t)(requests + 1) * 4 + 64;
    int s = (int)((budget > fixed ? budget - fixed : 0) / stage);
    if (s > kPagedMaxStages) s = kPagedMaxStages;
    s -= s % (ncw / 4);    // a stage always serves the same consumer group
    return PagedDecodePlan{s, fixed + (size_t)s * stage};
}

template <typename T, int HD, int NT, int NGROUPS>   // NT: n8 tiles of query rows
__global__ void __launch_bounds__((NGROUPS * 4 + 1) * 32, NGROUPS == 1 && HD <= 128 ? 2 : 1)
hkv_paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const PagedDecodeArgs a, const int stages) {
    constexpr int CW = paged_chunk_width(HD);
    constexpr int NCH = HD / CW;
    constexpr int ROWB = CW * 2;
    constexpr int TILE_BYTES = kTileRows * HD * 2;
    // A staged tile: [8-row group][column block][8 rows], so that one box brings all column blocks of a page's rows.
    constexpr int CHUNK_OFF = 8 * ROWB;
    auto row_off = [](int row) { return (row >> 3) * (NCH * CHUNK_OFF) + (row & 7) * ROWB; };
    constexpr int STAGE_BYTES = 2 * TILE_BYTES;
    constexpr int NCW = NGROUPS * 4;
    constexpr int KS = HD / 16;
    constexpr int OS = HD + 4;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const PagedBatch& bt = a.t.b;
    const int G = a.t.H / a.t.KVH, R = bt.requests, KVH = a.t.KVH;
    float* mrg_o = reinterpret_cast<float*>(smem + (size_t)stages * STAGE_BYTES);   // [NCW][cols][OS]
    float* mrg_ml = mrg_o + (size_t)NCW * a.cols * OS;                              // [NCW][cols][2]
    uint64_t* bars = reinterpret_cast<uint64_t*>(mrg_ml + (size_t)NCW * a.cols * 2);
    int* prefix = reinterpret_cast<int*>(bars + 2 * kPagedMaxStages);               // [R + 1]
    __shared__ long long scan_buf[33];
    __shared__ int4 s_req[kReqCache];     // the span's first requests: {start, n, pos0, keys}
    const uint32_t smem_base = smem_u32(smem);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + kPagedMaxStages);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 4);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    // prefix[r] = tiles of the requests before r
    {
        const int per = (R + (int)blockDim.x - 1) / (int)blockDim.x, r0 = tid * per, r1 = r0 + per < R ? r0 + per : R;
        long long sum = 0;
        for (int r = r0; r < r1; ++r) {
            const PagedRequest q = paged_request(bt, r);
            int lo, n = 0;
            if (paged_is_small(q, G, a.cols)) paged_tiles(bt, q, lo, n);
            prefix[r] = n;
            sum += n;
        }
        long long all;
        long long at = block_scan(sum, scan_buf, all);
        for (int r = r0; r < r1; ++r) {
            const int n = prefix[r];
            prefix[r] = (int)at;
            at += n;
        }
        if (tid == 0) prefix[R] = (int)all;
    }
    __syncthreads();
    const int W = prefix[R];
    const int GS = a.gang;
    const int NS = span_count(W, (int)gridDim.x / GS);
    const int span = blockIdx.x / GS, member = blockIdx.x % GS;
    int u0 = 0, u1 = 0, r_first = 0;
    if (span < NS) {
        u0 = (int)((long long)W * span / NS);
        u1 = (int)((long long)W * (span + 1) / NS);
        int lo = 0, hi = R - 1;            // the last request that starts at or before tile u0
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= u0) lo = mid; else hi = mid - 1;
        }
        r_first = lo;
    }
    if (u1 > u0) {
        for (int i = tid; i < kReqCache && r_first + i < R; i += blockDim.x) {
            const PagedRequest q = paged_request(bt, r_first + i);
            s_req[i] = make_int4(q.start, q.n, q.pos0, q.keys);
        }
    }
    __syncthreads();
    auto request = [&](int r) -> PagedRequest {
        if (r - r_first >= kReqCache) return paged_request(bt, r);
        const int4 x = s_req[r - r_first];
        return PagedRequest{x.x, x.y, x.z, x.w};
    };
    if (member == 0 && tid == 0 && span < (int)gridDim.x / GS) {
        // the request that starts in this span and goes on behind it is merged from this span's entry
        int4 cut = make_int4(0, 0, 0, 0);
        if (u1 > u0) {
            int lo = r_first, hi = R - 1;  // the request that holds tile u1 - 1
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (prefix[mid] <= u1 - 1) lo = mid; else hi = mid - 1;
            }
            if (prefix[lo] >= u0 && prefix[lo + 1] > u1) {
                const PagedRequest q = paged_request(bt, lo);
                cut = make_int4(lo, span_owner(prefix[lo + 1] - 1, W, NS) - span + 1, q.start, q.n);
            }
        }
        a.cuts[span] = cut;
    }

    if (warp == NCW) {
        // ------------------------------ producer (the whole warp) ------------------------------
        int stage = 0, round = 0, issued = 0;
        bool ok = true;
        const int page_shift = 31 - __clz(bt.page);   // page sizes here are powers of two
        const int my_piece = lane % a.pieces;         // (pieces divides 32)
        for (int kvh = member; kvh < KVH && ok; kvh += GS) {
            int r = r_first;
            for (int u = u0; u < u1 && ok; ++r) {
                const int nb = prefix[r + 1] - prefix[r];
                if (nb == 0) continue;
                const int off = u - prefix[r];
                const int nt = nb - off < u1 - u ? nb - off : u1 - u;
                u += nt;
                const PagedRequest q = request(r);
                int tile_lo, n_tiles, lo, hi, x_;
                paged_tiles(bt, q, tile_lo, n_tiles);
                paged_key_range(bt, q, 0, lo, x_);
                paged_key_range(bt, q, q.n - 1, x_, hi);
                const int32_t* table = bt.table + (long long)r * bt.cols;
                // page of this lane's box: behind the tensor (zeros, nothing read) where no query looks
                auto look_up = [&](int p) -> int {
                    if (paged_box_hidden(p, a.box_rows, lo, hi)) return bt.pages;
                    const int pg = __ldg(table + (p >> page_shift));
                    if (pg >= 0 && pg < bt.pages) return pg;
                    atomicOr(bt.status, kStatusBoundCheck);
                    return bt.pages;
                };
                int pg = look_up((tile_lo + off) * kTileRows + my_piece * a.box_rows);
                for (int t = 0; t < nt; ++t) {
                    const int pos0 = (tile_lo + off + t) * kTileRows;
                    const int pg_next = t + 1 < nt ? look_up(pos0 + kTileRows + my_piece * a.box_rows) : 0;   // a tile ahead
                    if (round > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * stage, (uint32_t)(round - 1) & 1u, bt.status));
                    if (!ok) break;
                    const uint32_t full = full0 + 8 * stage;
                    const uint32_t dst = smem_base + (uint32_t)stage * STAGE_BYTES;
                    if (lane == 0) mbar_expect_tx(full, STAGE_BYTES);
                    __syncwarp();
                    if (lane < 2 * a.pieces) {             // one box per page and operand (at most 16), all column blocks
                        const int kv = lane >= a.pieces, at = my_piece * a.box_rows;
                        tma_load_4d(dst + kv * TILE_BYTES + row_off(at), kv ? &tm_v : &tm_k, full, 0, 0, kvh * NCH,
                                    (pg << (page_shift - 3)) + (((pos0 + at) & (bt.page - 1)) >> 3));
                    }
                    pg = pg_next;
                    ++issued;
                    if (++stage == stages) { stage = 0; ++round; }
                }
            }
        }
        // every copy issued has landed before the CTA retires
        const int back = issued < stages ? issued : stages;
        for (int i = 0; i < back; ++i) {
            if (--stage < 0) { stage = stages - 1; --round; }
            mbar_wait(full0 + 8 * stage, (uint32_t)round & 1u, bt.status);
        }
        return;
    }

    // ------------------------------ consumers ------------------------------
    const int grp = warp >> 2, wig = warp & 3;
    const int r4 = lane >> 2, c4 = lane & 3;
    const int k_row = wig * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;   // K: matrices 1,3 are rows+8
    const int k_sel = lane >> 4;                                       // K: matrices 2,3 are k+8
    const int v_row = wig * 16 + (lane & 7) + (lane >> 4) * 8;         // V^T: matrices 2,3 are rows+8
    const int v_sel = (lane >> 3) & 1;                                 // V^T: matrices 1,3 are d+8
    const int k_swz = (CW == 64) ? (k_row & 7) : ((k_row >> 1) & 3);
    const int v_swz = (CW == 64) ? (v_row & 7) : ((v_row >> 1) & 3);

    const int k_off = row_off(k_row), v_off = row_off(v_row);

    int stage = 0, round = 0, tile_seq = 0;
    bool ok = true;
    for (int kvh = member; kvh < KVH; kvh += GS)
    for (int r = r_first, u = u0; u < u1; ++r) {
        const int nb = prefix[r + 1] - prefix[r];
        if (nb == 0) continue;
        const int off = u - prefix[r];
        const int nt = nb - off < u1 - u ? nb - off : u1 - u;
        const bool begins = off == 0, ends = off + nt == nb;
        u += nt;
        const PagedRequest q = request(r);
        const int ncol = q.n * G;
        int tile_lo, n_tiles, lo_first, hi_first, lo_last, hi_last;
        paged_tiles(bt, q, tile_lo, n_tiles);
        paged_key_range(bt, q, 0, lo_first, hi_first);
        paged_key_range(bt, q, q.n - 1, lo_last, hi_last);   // lo and hi grow with the query
        const int t0 = tile_lo + off;

        // Query fragments: B operand [16 d x 8 columns], column = r4 (query i, head g = column i*G + g), d pair = c4*2 (+8).
        uint32_t qb[NT][KS][2];
        int k_lo[NT][2], k_hi[NT][2];         // keys attended by this thread's score columns n*8 + c4*2 (+1)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int col = n * 8 + r4;
            const T* qp = (const T*)a.t.q + (long long)(q.start + col / G) * a.t.q_stride + ((long long)kvh * G + col % G) * HD;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qb[n][ks][0] = col < ncol ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + c4 * 2) : 0u;
                qb[n][ks][1] = col < ncol ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + c4 * 2 + 8) : 0u;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = n * 8 + c4 * 2 + e;
                k_lo[n][e] = k_hi[n][e] = 0;
                if (c < ncol) paged_key_range(bt, q, c / G, k_lo[n][e], k_hi[n][e]);
            }
        }
        float m_run[NT][2], l_run[NT][2], o_acc[NT][KS][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m_run[n][0] = m_run[n][1] = kLow;
            l_run[n][0] = l_run[n][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o_acc[n][mt][e] = 0.0f;
        }

        for (int t = 0; t < nt; ++t) {
            const bool mine = (tile_seq % NGROUPS) == grp;
            ++tile_seq;
            // After a wait has run out this warp stops waiting and computing but keeps walking its list, so that it
            // still meets the others at the merge barrier.
            if (mine && ok && !mbar_wait(full0 + 8 * stage, (uint32_t)round & 1u, bt.status)) ok = false;
            if (mine && ok) {
                const uint32_t kbase = smem_base + (uint32_t)stage * STAGE_BYTES;
                const uint32_t vbase = kbase + TILE_BYTES;
                uint8_t* vgen = smem + (size_t)stage * STAGE_BYTES + TILE_BYTES;
                const int row0 = (t0 + t) * kTileRows;
                const bool masked = paged_tile_masked(row0, kTileRows, lo_last, hi_first);
                if (masked) {
                    // V rows that no query attends are zeroed; values that are not finite in rows that only some attend are
                    // dropped and the request is marked, because 0 * NaN would reach the queries they are hidden from.
                    bool touched = false, bad = false;
                    for (int i = 0; i < 16; ++i) {
                        const int p = row0 + wig * 16 + i;
                        const bool none = p < lo_first || p >= hi_last, some = p < lo_last || p >= hi_first;
                        if (!none && !some) continue;
                        const int tr = wig * 16 + i;
                        const int swz = (CW == 64) ? (tr & 7) : ((tr >> 1) & 3);
                        for (int e = lane; e < HD / 8; e += 32) {
                            const int c = (e * 8) / CW, uu = (e * 8 % CW) / 8;
                            uint4* at = reinterpret_cast<uint4*>(vgen + c * CHUNK_OFF + row_off(tr) + ((uu ^ swz) << 4));
                            uint4 x = none ? make_uint4(0, 0, 0, 0) : *at;
                            if (!none) {
                                if (!drop_nonfinite<T>(x)) continue;
                                bad = true;
                            }
                            *at = x;
                            touched = true;
                        }
                    }
                    if (__any_sync(0xffffffffu, bad) && lane == 0) a.fix.push(r, -1, kvh);
                    if (__any_sync(0xffffffffu, touched)) fence_proxy_async_smem();
                    __syncwarp();
                }

                // ---- scores: S^T = K Q^T ----
                float sc[NT][2][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][0][e] = sc[n][1][e] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int d0 = ks * 16 + k_sel * 8;
                    const int c = d0 / CW, uu = (d0 % CW) / 8;
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4(kbase + c * CHUNK_OFF + k_off + ((uu ^ k_swz) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816_t<T>(sc[n][ks & 1], a0, a1, a2, a3, qb[n][ks][0], qb[n][ks][1]);
                }

                // ---- online softmax over rows, per column ----
                uint32_t pb[NT][2];
                const int pA = row0 + wig * 16 + r4, pB = pA + 8;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float s0 = (sc[n][0][0] + sc[n][1][0]) * a.t.scale_log2;
                    float s1 = (sc[n][0][1] + sc[n][1][1]) * a.t.scale_log2;
                    float s2 = (sc[n][0][2] + sc[n][1][2]) * a.t.scale_log2;
                    float s3 = (sc[n][0][3] + sc[n][1][3]) * a.t.scale_log2;
                    if (masked) {
                        if (pA < k_lo[n][0] || pA >= k_hi[n][0]) s0 = -INFINITY;
                        if (pA < k_lo[n][1] || pA >= k_hi[n][1]) s1 = -INFINITY;
                        if (pB < k_lo[n][0] || pB >= k_hi[n][0]) s2 = -INFINITY;
                        if (pB < k_lo[n][1] || pB >= k_hi[n][1]) s3 = -INFINITY;
                    }
                    float mx0 = fmaxf(s0, s2), mx1 = fmaxf(s1, s3);
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) {
                        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
                        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
                    }
                    const float mn0 = fmaxf(m_run[n][0], mx0), mn1 = fmaxf(m_run[n][1], mx1);
                    const float al0 = exp2f(m_run[n][0] - mn0), al1 = exp2f(m_run[n][1] - mn1);
                    const float p0 = exp2f(s0 - mn0), p1 = exp2f(s1 - mn1);
                    const float p2 = exp2f(s2 - mn0), p3 = exp2f(s3 - mn1);
                    m_run[n][0] = mn0;
                    m_run[n][1] = mn1;
                    l_run[n][0] = l_run[n][0] * al0 + p0 + p2;
                    l_run[n][1] = l_run[n][1] * al1 + p1 + p3;
#pragma unroll
                    for (int mt = 0; mt < KS; ++mt) {
                        o_acc[n][mt][0] *= al0;
                        o_acc[n][mt][1] *= al1;
                        o_acc[n][mt][2] *= al0;
                        o_acc[n][mt][3] *= al1;
                    }
                    pb[n][0] = movmatrix_t(pack2<T>(p0, p1));
                    pb[n][1] = movmatrix_t(pack2<T>(p2, p3));
                }

                // ---- output: O^T += V^T P^T ----
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    const int d0 = mt * 16 + v_sel * 8;
                    const int c = d0 / CW, uu = (d0 % CW) / 8;
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4_t(vbase + c * CHUNK_OFF + v_off + ((uu ^ v_swz) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816_t<T>(o_acc[n][mt], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty0 + 8 * stage);
            }
            if (++stage == stages) { stage = 0; ++round; }
        }
        // ---- merge the consumer warps; write the rows, or a partial of a request that is cut ----
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) {
                l_run[n][0] += __shfl_xor_sync(0xffffffffu, l_run[n][0], o);
                l_run[n][1] += __shfl_xor_sync(0xffffffffu, l_run[n][1], o);
            }
            const int h0 = n * 8 + c4 * 2;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                const int d = mt * 16 + r4;
                if (h0 < ncol) {
                    mrg_o[((size_t)warp * a.cols + h0) * OS + d] = o_acc[n][mt][0];
                    mrg_o[((size_t)warp * a.cols + h0) * OS + d + 8] = o_acc[n][mt][2];
                }
                if (h0 + 1 < ncol) {
                    mrg_o[((size_t)warp * a.cols + h0 + 1) * OS + d] = o_acc[n][mt][1];
                    mrg_o[((size_t)warp * a.cols + h0 + 1) * OS + d + 8] = o_acc[n][mt][3];
                }
            }
            if (r4 == 0) {
                if (h0 < ncol) {
                    mrg_ml[((size_t)warp * a.cols + h0) * 2] = m_run[n][0];
                    mrg_ml[((size_t)warp * a.cols + h0) * 2 + 1] = l_run[n][0];
                }
                if (h0 + 1 < ncol) {
                    mrg_ml[((size_t)warp * a.cols + h0 + 1) * 2] = m_run[n][1];
                    mrg_ml[((size_t)warp * a.cols + h0 + 1) * 2 + 1] = l_run[n][1];
                }
            }
        }
        named_bar_sync(1, NCW * 32);
        const bool whole = begins && ends;
        float* prow = a.part + ((long long)(2 * span + (begins ? 1 : 0)) * KVH + kvh) * a.cols * (HD + 2);
        for (int idx = tid; idx < ncol * (HD / 2); idx += NCW * 32) {
            const int c = idx / (HD / 2), d = idx % (HD / 2) * 2;
            float M = kLow;
#pragma unroll
            for (int w = 0; w < NCW; ++w) M = fmaxf(M, mrg_ml[((size_t)w * a.cols + c) * 2]);
            float o0 = 0.0f, o1 = 0.0f, L = 0.0f;
#pragma unroll
            for (int w = 0; w < NCW; ++w) {
                const float f = exp2f(mrg_ml[((size_t)w * a.cols + c) * 2] - M);
                const float2 x = *reinterpret_cast<const float2*>(mrg_o + ((size_t)w * a.cols + c) * OS + d);
                o0 = fmaf(x.x, f, o0);
                o1 = fmaf(x.y, f, o1);
                L = fmaf(mrg_ml[((size_t)w * a.cols + c) * 2 + 1], f, L);
            }
            if (whole) {
                const float inv = L > 0.0f ? 1.0f / L : 0.0f;
                T* op = (T*)a.t.out + ((long long)(q.start + c / G) * a.t.H + (long long)kvh * G + c % G) * HD;
                *reinterpret_cast<uint32_t*>(op + d) = pack2<T>(o0 * inv, o1 * inv);
            } else {
                *reinterpret_cast<float2*>(prow + (long long)c * (HD + 2) + d) = make_float2(o0, o1);
                if (d == 0) *reinterpret_cast<float2*>(prow + (long long)c * (HD + 2) + HD) = make_float2(M, L);
            }
        }
        named_bar_sync(1, NCW * 32);
    }
}

}  // namespace hkv
