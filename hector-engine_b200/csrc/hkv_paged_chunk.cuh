// hkv_paged_chunk.cuh — attention of prompt chunks over a paged cache on the 5th-generation tensor cores (tcgen05, tensor
// memory): the requests of a ragged batch that have more query rows per KV head than the few-token kernel takes.
// head_dim 64, 128, and 96 staged as 128 with columns of zeros.
//
// Bound: the tensor cores (4 H HD flops per attended pair), with exp2 and the softmax warps' issue slots close behind.
//   * Item = two tiles A and B of 128 query rows (row = query, head of the group) of one request and KV head; both are
//     contracted with the same staged K and V tiles of 128 positions. A block of queries that fits one tile leaves B out.
//   * The items of the batch form a line that is cut into equal spans, one per CTA (hkv_paged_line.cuh): a batch of any
//     mix keeps every SM busy to the end, and one short chunk over a long request is spread over all of them. An item that
//     is cut leaves partial rows, two sets per CTA at most, which the finishing kernel joins.
//   * Warps: 0-3 softmax of tile A, 4-7 of tile B (one thread per row), 8 producer, 9 MMA issuer, 10 writes the
//     finishing kernel's entry, 11 completes the warpgroup for setmaxnreg. A key tile is a set of boxes, one per page: the
//     producer's lanes look up one page each, a tile ahead, and issue side by side.
//   * Tensor memory: S_A, S_B (128 columns each; P is written over the first half of its S), O_A, O_B. Per key tile:
//     PV_A QK_A(next) PV_B QK_B(next), so that one tile's softmax runs under the other's products; P V of the first half
//     of a tile's keys starts while P of the second half is computed. O is rescaled only when a row's maximum outgrows
//     its reference by 2^8. (Two threads per row halve nothing: the softmax is bound by its instructions, the exchange and
//     the doubled bookkeeping cost a tenth.) P is rounded to the element type (its sum is not). In fp16 1 of
//     8 pairs take a polynomial on the FMA pipe instead of ex2, the narrowest unit; bf16 takes none (kCkEmuOf8).
//   * Measured (B200, one launch and the finishing one): 2 048 queries over 32k keys, 28 heads of 4, 128 wide, bf16: 716 us
//     at full clocks (1 302 TFLOP/s), 785 to 850 us back to back under the power limit; 8 x 224 to 448 queries over 2k to 4k
//     keys, fp16: 147 us. A pair of query tiles takes 2.0 us per 128 keys against 1.5 us of products at the library's rate.
//     A call costs 10 us until its first scores are there, an item 2 us of output; a tile on the diagonal takes 3.8 us. A
//     rehearsal of the tile code in front of the first tile, to warm the instruction caches, made every tile 7 % slower.
//   * Every wait is bounded and reports through the status word; tensor memory is freed on every path.
#pragma once

#include <cuda.h>

#include "hkv_paged_decode.cuh"
#include "hkv_paged_line.cuh"
#include "hkv_tc_ops.cuh"

namespace hkv {

constexpr int kCkRows = 128, kCkKeys = 128;
constexpr int kCkStages = 2;              // K tiles and V tiles in flight
constexpr int kCkThreads = 384;
// Pairs of every 8 whose exp2 runs on the FMA pipe, fp16 only. The polynomial ends at 2^-100, for a hidden key too: fp16
// rounds that to zero, but bf16 carries it to the second product, where 2^-100 times a large hidden value is not nothing.
// (2 048 queries over 32k keys, with and without in turn, best of replays: head_dim 128 bf16 713 and 721 us, fp16 739 and
// 747; head_dim 64 bf16 329 and 318. 8 x 224 to 448 queries over 4k keys 145 and 147. 2 and 3 of 8: 10 and 16 % slower than 1.)
constexpr int kCkEmuOf8 = 1;
constexpr int kCkDesc = 16;               // words of a work descriptor

struct PagedChunkArgs {
    PagedAttnArgs t;
    PagedLine line;           // `pre` is filled in by the kernel
    float* part;              // [2 * grid] sets of partial rows, see store_partial
    int4* cuts;               // [grid]: the item that starts in a CTA's span and goes on behind it: {request, kv head, block, parts}
    PagedFix fix;
    int QT;                   // queries per 128-row tile
    int box_rows, pieces;     // rows of a box; pages per tile
    int small;                // query rows per KV head up to which the few-token kernel takes a request; 0: none
};
__host__ __device__ constexpr size_t chunk_smem_bytes(int HD /*staged*/, int requests) {
    return 1024 + (size_t)(2 + 2 * kCkStages) * kCkRows * HD * 2 + 32 * 8 + 16 + 4 * kCkDesc * 4 + (size_t)(requests + 1) * 4 + 16;
}
__device__ __forceinline__ bool chunk_takes(const PagedChunkArgs& a, const PagedRequest& q) {
    return q.n > 0 && !paged_is_small(q, a.line.G, a.small);
}

// Units before each request, over the block; returns the units of all, 0 (and the status bit) where they do not fit.
// `pre` [requests + 1] in shared memory.
template <typename Args>
__device__ __forceinline__ uint32_t chunk_line(const Args& a, uint32_t* pre, long long* buf) {
    const PagedBatch& b = a.t.b;
    const int tid = threadIdx.x, R = b.requests;
    const int per = (R + (int)blockDim.x - 1) / (int)blockDim.x, r0 = tid * per, r1 = r0 + per < R ? r0 + per : R;
    long long sum = 0;
    for (int r = r0; r < r1; ++r) {
        const PagedRequest q = paged_request(b, r);
        const long long n = chunk_takes(a, q) ? line_units(b, a.line, q) : 0;
        pre[r] = (uint32_t)n;
        sum += n;
    }
    long long all;
    long long at = block_scan(sum, buf, all);
    for (int r = r0; r < r1; ++r) {
        const uint32_t n = pre[r];
        pre[r] = (uint32_t)at;
        at += n;
    }
    if (tid == 0) pre[R] = (uint32_t)all;
    __syncthreads();
    if (!line_fits(all)) {
        if (tid == 0) atomicOr(b.status, kStatusBoundCheck);
        return 0;
    }
    return (uint32_t)all;
}

// The finishing kernel's entry of CTA `cta`, by one warp: the item that starts in its span and goes on behind it.
__device__ __forceinline__ void chunk_cut_entry(const PagedBatch& b, const PagedLine& l, const uint32_t W, const int ctas, const int cta,
                                                int4* cuts) {
    const int lane = threadIdx.x & 31;
    int4 entry = make_int4(0, 0, 0, 0);
    if (cta < ctas) {
        // lanes 0 and 1: this span's cuts; an item that goes on past the end cut was begun here if the span does not start inside it
        const LineCut mine = line_locate(b, l, line_boundary(W, ctas, cta + (lane & 1)), W);
        LineCut c0, c1;
        c0.r = __shfl_sync(0xffffffffu, mine.r, 0); c0.kvh = __shfl_sync(0xffffffffu, mine.kvh, 0);
        c0.p = __shfl_sync(0xffffffffu, mine.p, 0); c0.t = __shfl_sync(0xffffffffu, mine.t, 0);
        c1.r = __shfl_sync(0xffffffffu, mine.r, 1); c1.kvh = __shfl_sync(0xffffffffu, mine.kvh, 1);
        c1.p = __shfl_sync(0xffffffffu, mine.p, 1); c1.t = __shfl_sync(0xffffffffu, mine.t, 1);
        if (c1.r < b.requests && c1.t > 0 && !(line_same_item(c0, c1) && c0.t > 0)) {
            int parts = 2;
            for (int base = cta + 2;; base += 32) {          // further cuts inside the same item
                const int c = base + lane;
                const LineCut x = line_locate(b, l, line_boundary(W, ctas, c < ctas ? c : ctas), W);
                const unsigned in = __ballot_sync(0xffffffffu, c < ctas && line_same_item(x, c1) && x.t > 0);
                parts += __popc(in);
                if (in != 0xffffffffu) break;
            }
            entry = make_int4(c1.r, c1.kvh, c1.p, parts);
        }
    }
    if (lane == 0) cuts[cta] = entry;
}

// The producer's walk over its span: calls piece(r, request, kvh, p, first key tile, tiles, slot) for every piece of work;
// slot -1: the whole item. Warp-uniform. Stops when piece() returns false.
template <typename F>
__device__ __forceinline__ void chunk_walk(const PagedBatch& b, const PagedLine& l, const uint32_t W, const int ctas, const int cta, F piece) {
    if (cta >= ctas || W == 0) return;
    const int lane = threadIdx.x & 31;
    const LineCut mine = line_locate(b, l, line_boundary(W, ctas, cta + (lane & 1)), W);
    LineCut c, e;
    c.r = __shfl_sync(0xffffffffu, mine.r, 0); c.kvh = __shfl_sync(0xffffffffu, mine.kvh, 0);
    c.p = __shfl_sync(0xffffffffu, mine.p, 0); c.t = __shfl_sync(0xffffffffu, mine.t, 0);
    e.r = __shfl_sync(0xffffffffu, mine.r, 1); e.kvh = __shfl_sync(0xffffffffu, mine.kvh, 1);
    e.p = __shfl_sync(0xffffffffu, mine.p, 1); e.t = __shfl_sync(0xffffffffu, mine.t, 1);
    while (c.r < b.requests && line_before(c, e)) {
        if (l.pre[c.r + 1] == l.pre[c.r]) { ++c.r; c.kvh = c.p = c.t = 0; continue; }   // not this kernel's request
        const PagedRequest q = paged_request(b, c.r);
        int kt0, nt;
        line_tiles(b, l, q, c.p, kt0, nt);
        const int end = line_same_item(c, e) ? e.t : nt;
        const int slot = c.t == 0 && end == nt ? -1 : 2 * cta + (c.t == 0 ? 1 : 0);
        if (end > c.t && !piece(c.r, q, c.kvh, c.p, kt0 + c.t, end - c.t, slot)) return;
        c.t = 0;
        if (++c.p >= line_blocks(q.n, l.QB)) {
            c.p = 0;
            if (++c.kvh == l.KVH) { c.kvh = 0; ++c.r; }
        }
    }
}

// ---- rows out of tensor memory ----------------------------------------------------------------------------------------
// A thread holds a row, but 32 stores of 16 bytes at 32 rows are 32 half-used sectors: a warp's 4 KB then takes a quarter
// of a microsecond of the store path, 3.2 us an item. So the four lanes of a quad swap 16-byte pieces (a 4 x 4 transpose)
// and each store writes 64 contiguous bytes of 8 rows.
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[16]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int bit = 1; bit <= 2; bit <<= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b & bit) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t &x = w[4 * b + e], &y = w[4 * (b | bit) + e];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? x : y, bit);
                if (up) x = got; else y = got;
            }
        }
    }
}
// Element offsets of the four rows of this lane's quad; -1: a row that is not written.
__device__ __forceinline__ void quad_rows(const long long mine, long long (&rows)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = __shfl_sync(0xffffffffu, mine, (threadIdx.x & 28) + i);
}
// 32 columns of a row per thread, scaled and rounded, to the quad's rows. Whole warps.
template <typename T>
__device__ __forceinline__ void store_rows32(T* out, const long long (&rows)[4], const int col, const uint32_t (&v)[32], const float inv) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack2<T>(__uint_as_float(v[2 * j]) * inv, __uint_as_float(v[2 * j + 1]) * inv);
    quad_transpose(w);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (rows[i] >= 0)
            *reinterpret_cast<uint4*>(out + rows[i] + col + (threadIdx.x & 3) * 8) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}
// A set of partial rows: [head_dim / 4][rows] float4 of o, then [rows] {maximum (log2 domain), sum}: a warp writes its rows
// side by side, and the finishing kernel reads them so.
__host__ __device__ constexpr long long partial_floats(int rows, int hd) { return (long long)rows * (hd + 2); }
__device__ __forceinline__ void store_partial32(float* set, const int rows, const int row, const int col, const uint32_t (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<uint4*>(set + ((long long)((col + j) / 4) * rows + row) * 4) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
}

// V rows [kstart, kstart + keys) of a staged tile that not every query of a block sees: rows that none attends are zeroed,
// values that are not finite are dropped from the others (0 * NaN would reach the queries they are hidden from). `threads`
// threads take part; true if this one dropped a value.
template <typename T, int NCH, int threads>
static __device__ __noinline__ bool clean_values(const PagedBatch& b, const PagedRequest q, const int i0, const int QB, const int kstart,
                                                 const int keys, uint8_t* tile, const int chunk_off, const int group_off, const int tid) {
    int lo_first, hi_first, lo_last, hi_last;
    paged_key_range(b, q, i0, lo_first, hi_first);
    paged_key_range(b, q, (i0 + QB < q.n ? i0 + QB : q.n) - 1, lo_last, hi_last);
    const int head = lo_last - kstart < 0 ? 0 : (lo_last - kstart < keys ? lo_last - kstart : keys);
    int tail = hi_first - kstart < 0 ? 0 : (hi_first - kstart < keys ? hi_first - kstart : keys);
    if (tail < head) tail = head;
    bool bad = false;
    // a thread keeps its 16-byte column and steps over rows, four loads in flight
    constexpr int kStep = threads / (8 * NCH);
    const int u = tid % (8 * NCH), rows = head + keys - tail;
    uint8_t* col = tile + (u / 8) * chunk_off + (u % 8) * 16;
    for (int k0 = tid / (8 * NCH); k0 < rows; k0 += 4 * kStep) {
        uint4 x[4];
        uint4* at[4];
        bool seen[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = k0 + e * kStep, vr = k < head ? k : tail + k - head, pos = kstart + vr;
            at[e] = k < rows ? reinterpret_cast<uint4*>(col + (vr >> 3) * group_off + (vr & 7) * 128) : nullptr;
            seen[e] = pos >= lo_first && pos < hi_last;
            x[e] = make_uint4(0, 0, 0, 0);
            if (at[e] && seen[e]) x[e] = *at[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool drop = at[e] && seen[e] && drop_nonfinite<T>(x[e]);
            bad |= drop;
            if (at[e] && (drop || !seen[e])) *at[e] = x[e];
        }
    }
    return bad;
}

// WHOLE: one box brings all column blocks of its rows, a staged K or V tile is [8-row group][column block][8 rows of 128
// bytes]. Otherwise (head_dim 96) a box per block, [column block][8-row group], so that the columns behind it are zeros.
template <typename T, int HD, bool WHOLE>
__global__ void __launch_bounds__(kCkThreads, 1)
hkv_paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const PagedChunkArgs a) {
    static_assert(HD == 64 || HD == 128, "staged head_dim 64 or 128");
    constexpr int NCH = HD / 64;                       // 64-element column blocks
    constexpr int CHUNK_BYTES = kCkRows * 128;
    constexpr int TILE_BYTES = kCkRows * HD * 2;
    constexpr int CHUNK_OFF = WHOLE ? 1024 : CHUNK_BYTES, GROUP_OFF = WHOLE ? NCH * 1024 : 1024;
    constexpr int COL_BOXES = WHOLE ? 1 : NCH, HEAD_STEP = WHOLE ? NCH : 1;   // boxes per piece; coordinate step of a KV head
    constexpr int EMU = std::is_same<T, __half>::value ? kCkEmuOf8 : 0;
    constexpr uint32_t TMEM_COLS = 512;
    constexpr uint32_t COL_S = 0, COL_O = 256;         // + 128 * group
    constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);   // operand type of the MMA
    constexpr uint32_t IDESC_QK = FMT | (1u << 4) | ((uint32_t)(kCkKeys >> 3) << 17) | ((uint32_t)(kCkRows >> 4) << 24);
    constexpr uint32_t IDESC_PV = FMT | (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kCkRows >> 4) << 24);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* k_gen = smem + 2 * TILE_BYTES;                   // after the query tiles A, B
    uint8_t* v_gen = k_gen + kCkStages * TILE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_gen + kCkStages * TILE_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
    volatile int* queue = reinterpret_cast<volatile int*>(tmem_slot + 4);   // [4][kCkDesc]
    uint32_t* pre = tmem_slot + 4 + 4 * kCkDesc;                            // [requests + 1]
    __shared__ long long scan_buf[33];
    const uint32_t q_smem = smem_u32(smem), k_smem = smem_u32(k_gen), v_smem = smem_u32(v_gen), bar0 = smem_u32(bars);
    const uint32_t B_QFULL = bar0, B_QEMPTY = bar0 + 8, B_KFULL = bar0 + 16, B_KEMPTY = bar0 + 32, B_VFULL = bar0 + 48,
                   B_VEMPTY = bar0 + 64, B_SFULL = bar0 + 80, B_PFULL = bar0 + 96 /* [tile][half] */, B_OFULL = bar0 + 128,
                   B_DONE = bar0 + 144, B_WF = bar0 + 152, B_WE = bar0 + 184;      // work queue: slot full [4], slot read [4]
    const PagedBatch& bt = a.t.b;
    const int G = a.line.G, H = a.t.H, D = a.t.HD;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    launch_dependents();
    if (tid == 0) {
        mbar_init(B_QFULL, 1); mbar_init(B_QEMPTY, 1); mbar_init(B_DONE, 1);
        for (int s = 0; s < kCkStages; ++s) {
            mbar_init(B_KFULL + 8 * s, 1); mbar_init(B_KEMPTY + 8 * s, 1);
            mbar_init(B_VFULL + 8 * s, 1); mbar_init(B_VEMPTY + 8 * s, 1);
        }
        for (int g = 0; g < 2; ++g) { mbar_init(B_SFULL + 8 * g, 1); mbar_init(B_OFULL + 8 * g, 1); }
        for (int i = 0; i < 4; ++i) { mbar_init(B_PFULL + 8 * i, 4); mbar_init(B_WF + 8 * i, 1); mbar_init(B_WE + 8 * i, 9); }
        fence_mbar_init();
        tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
    }
    const uint32_t W = chunk_line(a, pre, scan_buf);
    PagedLine line = a.line;
    line.pre = pre;
    const int ctas = line_ctas(W, (int)gridDim.x);
    if (warp == 9) tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // entry k of the queue lives in slot k % 4, phase k / 4
    auto queue_wait = [&](uint32_t k) -> bool { return mbar_wait(B_WF + 8 * (k & 3), (k >> 2) & 1, bt.status); };

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 8) {
        // ------------------------------ producer (the whole warp) ------------------------------
        uint32_t gt = 0, it = 0;
        bool ok = true;
        auto publish = [&](int r, const PagedRequest& q, int kvh, int p, int kt, int nt, int slot, int two) -> bool {
            const uint32_t s = it & 3;
            if (it >= 4 && !__all_sync(0xffffffffu, mbar_wait(B_WE + 8 * s, ((it >> 2) - 1) & 1, bt.status))) return false;
            if (lane == 0) {
                volatile int* d = queue + s * kCkDesc;
                d[0] = r; d[1] = kvh; d[2] = p; d[3] = kt; d[4] = nt; d[5] = slot; d[6] = two;
                d[7] = q.start; d[8] = q.n; d[9] = q.pos0; d[10] = q.keys;
                mbar_arrive(B_WF + 8 * s);
            }
            __syncwarp();
            return true;
        };
        const int page_shift = 31 - __clz(bt.page);
        const int my_piece = lane % a.pieces;          // the page this lane looks up: one per box of a column block
        chunk_walk(bt, line, W, ctas, blockIdx.x, [&](int r, const PagedRequest& q, int kvh, int p, int kt, int nt, int slot) -> bool {
            const int i0 = p * a.line.QB, two = i0 + a.QT < q.n ? 1 : 0;
            if (!publish(r, q, kvh, p, kt, nt, slot, two)) { ok = false; return false; }
            if (!__all_sync(0xffffffffu, mbar_wait(B_QEMPTY, (it & 1) ^ 1, bt.status))) { ok = false; return false; }
            if (lane == 0) {
                mbar_expect_tx(B_QFULL, (uint32_t)((1 + two) * NCH * a.QT * G * 128));
                for (int t2 = 0; t2 <= two; ++t2)
#pragma unroll
                    for (int c = 0; c < NCH; ++c)
                        tma_load_3d(q_smem + t2 * TILE_BYTES + c * CHUNK_BYTES, &tm_q, B_QFULL, c * 64, kvh * G, q.start + i0 + t2 * a.QT);
            }
            __syncwarp();
            ++it;
            int lo, hi, x, y;
            paged_key_range(bt, q, i0, lo, x);
            const int i1 = (i0 + a.line.QB < q.n ? i0 + a.line.QB : q.n) - 1;
            paged_key_range(bt, q, i1, y, hi);
            const int32_t* table = bt.table + (long long)r * bt.cols;
            // page of a box: behind the tensor (zeros, nothing read) where no query of the item looks
            auto look_up = [&](int pos) -> int {
                if (paged_box_hidden(pos, a.box_rows, lo, hi)) return bt.pages;
                const int pg = __ldg(table + (pos >> page_shift));
                if (pg >= 0 && pg < bt.pages) return pg;
                atomicOr(bt.status, kStatusBoundCheck);
                return bt.pages;
            };
            int pg = look_up(kt * kCkKeys + my_piece * a.box_rows);
            for (int t = 0; t < nt; ++t, ++gt) {
                const int pos0 = (kt + t) * kCkKeys;
                const int pg_next = t + 1 < nt ? look_up(pos0 + kCkKeys + my_piece * a.box_rows) : 0;
                const uint32_t s = gt % kCkStages, ph = (gt / kCkStages) & 1;
                for (int kv = 0; kv < 2; ++kv) {
                    const uint32_t full = (kv ? B_VFULL : B_KFULL) + 8 * s, empty = (kv ? B_VEMPTY : B_KEMPTY) + 8 * s;
                    if (!__all_sync(0xffffffffu, mbar_wait(empty, ph ^ 1, bt.status))) {
                        if (kv && lane == 0) mbar_wait(B_KFULL + 8 * s, ph, bt.status);   // the K copies above are in flight
                        ok = false;
                        return false;
                    }
                    if (lane == 0) mbar_expect_tx(full, TILE_BYTES);
                    __syncwarp();
                    const uint32_t dst = (kv ? v_smem : k_smem) + s * TILE_BYTES;
                    if (lane < COL_BOXES * a.pieces) {             // (at most 32)
                        const int c = COL_BOXES > 1 ? lane / a.pieces : 0, at = my_piece * a.box_rows;
                        tma_load_4d(dst + c * CHUNK_OFF + (at >> 3) * GROUP_OFF, kv ? &tm_v : &tm_k, full, c * 64, 0, kvh * HEAD_STEP,
                                    (pg << (page_shift - 3)) + (((pos0 + at) & (bt.page - 1)) >> 3));
                    }
                }
                pg = pg_next;
            }
            return true;
        });
        // no more work (also after a wait that ran out: the other roles leave at once)
        const uint32_t pieces_done = it;
        const PagedRequest none{0, 0, 0, 0};
        publish(-1, none, 0, 0, 0, 0, 0, 0);
        // copies in flight have landed before the CTA retires (tiles 0..gt-1 were issued)
        if (lane == 0) {
            if (pieces_done > 0) mbar_wait(B_QFULL, (pieces_done - 1) & 1, bt.status);
            for (uint32_t i = 1; i <= (uint32_t)kCkStages && i <= gt; ++i) {
                const uint32_t g = gt - i;
                mbar_wait(B_KFULL + 8 * (g % kCkStages), (g / kCkStages) & 1, bt.status);
                mbar_wait(B_VFULL + 8 * (g % kCkStages), (g / kCkStages) & 1, bt.status);
            }
        }
        __syncwarp();
    } else if (warp == 10) {
        chunk_cut_entry(bt, line, W, ctas, blockIdx.x, a.cuts);
    } else if (warp == 9) {
        // ------------------------------ MMA issuer ------------------------------
        if (elect_one()) {
            uint32_t gt = 0, it = 0, gb = 0;               // tiles; items; tiles of tile B
            bool ok = true;
            const uint64_t qdesc0 = umma_desc_sw128(q_smem, 16), kdesc0 = umma_desc_sw128(k_smem, 16, GROUP_OFF);
            const uint64_t vdesc0 = umma_desc_sw128(v_smem, CHUNK_OFF, GROUP_OFF);
            const uint32_t q_hi = (uint32_t)(qdesc0 >> 32), kv_hi = (uint32_t)(kdesc0 >> 32);
            const uint32_t q_lo = (uint32_t)qdesc0, k_lo = (uint32_t)kdesc0, v_lo = (uint32_t)vdesc0;
            const int ksteps = (D + 15) / 16;              // zero-filled k-steps are skipped
            auto issue_qk = [&](uint32_t g, int grp) {     // S_grp = Q_grp K(g)^T
                const uint32_t kd = k_lo + (((g % kCkStages) * TILE_BYTES) >> 4);
                const uint32_t qd = q_lo + ((grp * TILE_BYTES) >> 4);
                const uint32_t d = tmem + COL_S + 128u * grp;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t qo = (uint32_t)(((kk / 4) * CHUNK_BYTES + (kk % 4) * 32) >> 4), ko = (uint32_t)(((kk / 4) * CHUNK_OFF + (kk % 4) * 32) >> 4);
                    if (kk == 0) tc_mma_ss_ii<false>(d, qd + qo, q_hi, kd + ko, kv_hi, IDESC_QK);
                    else if (kk < ksteps) tc_mma_ss_ii<true>(d, qd + qo, q_hi, kd + ko, kv_hi, IDESC_QK);
                }
                tc_commit(B_SFULL + 8 * grp);
            };
            // O_grp (+)= P_grp V(g) over one half of the tile's keys
            auto issue_pv = [&](uint32_t g, int grp, int half, bool accumulate) {
                const uint32_t vd = v_lo + (((g % kCkStages) * TILE_BYTES) >> 4);
                const uint32_t pbase = tmem + COL_S + 128u * grp, d = tmem + COL_O + 128u * grp;
#pragma unroll
                for (int k = 0; k < kCkKeys / 32; ++k) {
                    const int kk = half * (kCkKeys / 32) + k;
                    const uint32_t at = vd + (uint32_t)((kk * 2 * GROUP_OFF) >> 4);
                    if (k > 0 || accumulate) tc_mma_ts_i<true>(d, pbase + kk * 8, at, kv_hi, IDESC_PV);
                    else tc_mma_ts_i<false>(d, pbase + kk * 8, at, kv_hi, IDESC_PV);
                }
            };
            for (; ok; ++it) {
                if (!queue_wait(it)) { ok = false; break; }
                const volatile int* d = queue + (it & 3) * kCkDesc;
                const int r = d[0], nt = d[4], two = d[6];
                mbar_arrive(B_WE + 8 * (it & 3));
                if (r < 0) break;
                if (!mbar_wait(B_QFULL, it & 1, bt.status) ||
                    !mbar_wait(B_KFULL + 8 * (gt % kCkStages), (gt / kCkStages) & 1, bt.status)) { ok = false; break; }
                tc_fence_after();
                issue_qk(gt, 0);
                if (two) issue_qk(gt, 1);
                tc_commit(B_KEMPTY + 8 * (gt % kCkStages));
                if (nt == 1) tc_commit(B_QEMPTY);
                for (int t = 0; t < nt && ok; ++t, ++gt) {
                    const bool more = t + 1 < nt;
                    const uint32_t vs = gt % kCkStages, ks1 = (gt + 1) % kCkStages;
                    // operand tiles first (they land long before P does)
                    if (!mbar_wait(B_VFULL + 8 * vs, (gt / kCkStages) & 1, bt.status) ||
                        (more && !mbar_wait(B_KFULL + 8 * ks1, ((gt + 1) / kCkStages) & 1, bt.status))) { ok = false; break; }
#pragma unroll
                    for (int grp = 0; grp < 2; ++grp) {
                        if (grp == 1 && !two) break;
                        const uint32_t ph = (grp ? gb : gt) & 1;
                        if (!mbar_wait(B_PFULL + 16 * grp, ph, bt.status)) { ok = false; break; }
                        tc_fence_after();
                        issue_pv(gt, grp, 0, t > 0);
                        if (!mbar_wait(B_PFULL + 16 * grp + 8, ph, bt.status)) { ok = false; break; }
                        tc_fence_after();
                        issue_pv(gt, grp, 1, true);
                        if (!more) tc_commit(B_OFULL + 8 * grp);
                        if (grp == two) tc_commit(B_VEMPTY + 8 * vs);       // every tile has consumed V(g)
                        if (more) {
                            issue_qk(gt + 1, grp);
                            if (grp == two) {
                                tc_commit(B_KEMPTY + 8 * ks1);
                                if (t + 2 == nt) tc_commit(B_QEMPTY);       // last score products of the item issued
                            }
                        }
                    }
                    gb += two;
                }
            }
            // every product issued has completed before tensor memory is freed
            tc_commit(B_DONE);
            mbar_wait(B_DONE, 0, bt.status);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ------------------------------ softmax / output rows ------------------------------
        const int quad = warp & 3, grp = warp >> 2;
        const int row = quad * 32 + lane;          // row of the tile = lane of tensor memory
        const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + lane_sel + COL_S + 128u * grp;
        const uint32_t o_addr = tmem + lane_sel + COL_O + 128u * grp;
        const uint32_t b_sfull = B_SFULL + 8 * grp, b_pfull = B_PFULL + 16 * grp, b_ofull = B_OFULL + 8 * grp;
        const int ql = row / G, g = row % G;
        uint32_t gt = 0, si = 0;   // tiles and items of this group (barrier phases); group A's tiles are the CTA's
        bool ok = true;            // kept warp-uniform: a wait that ran out for any lane stops the warp
        for (uint32_t qk = 0; ok; ++qk) {
            ok = __all_sync(0xffffffffu, queue_wait(qk));
            if (!ok) break;
            const volatile int* d = queue + (qk & 3) * kCkDesc;
            const int r = d[0], kvh = d[1], p = d[2], kt = d[3], nt = d[4], slot = d[5], two = d[6];
            const PagedRequest q{d[7], d[8], d[9], d[10]};
            __syncwarp();
            if (lane == 0) mbar_arrive(B_WE + 8 * (qk & 3));
            if (r < 0) break;
            if (grp > two) continue;               // the block of queries fits tile A
            const int i0 = p * a.line.QB, qi = i0 + grp * a.QT + ql, kbase = kt * kCkKeys;
            // rows without a query take the bounds of the last one, so that they never hold up their warp
            int lo_row, hi_row, head, tail;        // tiles that not every query of the item sees whole: before head, from tail on
            paged_key_range(bt, q, qi < q.n ? qi : q.n - 1, lo_row, hi_row);
            {
                int x, lo_last, hi_first;
                paged_key_range(bt, q, i0, x, hi_first);
                paged_key_range(bt, q, (i0 + a.line.QB < q.n ? i0 + a.line.QB : q.n) - 1, lo_last, x);
                head = lo_last > kbase ? (lo_last - kbase + kCkKeys - 1) / kCkKeys : 0;
                tail = hi_first > kbase ? (hi_first - kbase) / kCkKeys : 0;
            }
            float m_ref = kLow, l_run = 0.0f;      // m_ref: the reference P and O are scaled by

            for (int t = 0; t < nt; ++t, ++gt) {
                ok = __all_sync(0xffffffffu, ok && mbar_wait(b_sfull, gt & 1, bt.status));
                if (!ok) continue;
                tc_fence_after();
                uint32_t sv[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(sv[c], s_addr + c * 32);
                const int lo = lo_row - (kt + t) * kCkKeys, hi = hi_row - (kt + t) * kCkKeys;   // attended columns [lo, hi)
                const bool all_in = __all_sync(0xffffffffu, lo <= 0 && hi >= kCkKeys);
#pragma unroll
                for (int c = 0; c < 4; ++c) tc_wait_ld_dep(sv[c]);
                if (!all_in) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c * 32 + j < lo || c * 32 + j >= hi) sv[c][j] = 0xff800000u;   // -infinity
                }
                // ---- row maximum of the raw scores (the scale is positive) ----
                float mx;
                {
                    float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;   // independent chains
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            m0 = fmax3(m0, __uint_as_float(sv[c][j]), __uint_as_float(sv[c][j + 1]));
                            m1 = fmax3(m1, __uint_as_float(sv[c][j + 2]), __uint_as_float(sv[c][j + 3]));
                            m2 = fmax3(m2, __uint_as_float(sv[c][j + 4]), __uint_as_float(sv[c][j + 5]));
                            m3 = fmax3(m3, __uint_as_float(sv[c][j + 6]), __uint_as_float(sv[c][j + 7]));
                        }
                    mx = fmaxf(fmax3(m0, m1, m2), m3) * a.t.scale_log2;
                }
                const bool move = mx > m_ref + 8.0f;
                if (__any_sync(0xffffffffu, move)) {
                    const float m_to = move ? mx : m_ref;
                    const float alpha = ex2_approx(m_ref - m_to);   // 1 for rows that keep their reference
                    // the score product of this tile was issued after P V of the previous one: O is complete up to t-1
                    if (t > 0) tmem_scale_columns(o_addr, HD / 32, alpha);
                    l_run *= alpha;
                    m_ref = m_to;
                }
                // Tiles that not every query of the item sees whole: group A cleans the V rows before its arrival, which
                // precedes both output products.
                if (grp == 0 && (t < head || t >= tail)) {
                    const uint32_t vs = gt % kCkStages;
                    ok = __all_sync(0xffffffffu, mbar_wait(B_VFULL + 8 * vs, (gt / kCkStages) & 1, bt.status));
                    if (!ok) continue;
                    const bool bad = clean_values<T, NCH, 128>(bt, q, i0, a.line.QB, (kt + t) * kCkKeys, kCkKeys,
                                                               v_gen + (size_t)vs * TILE_BYTES, CHUNK_OFF, GROUP_OFF, tid);
                    if (__any_sync(0xffffffffu, bad) && lane == 0) a.fix.push(r, p, kvh);
                    fence_proxy_async_smem();
                }
                // ---- p = 2^(s*scale - m_ref), row sum, P back to tensor memory, half a tile at a time ----
                float lsum0 = 0.0f, lsum1 = 0.0f, lsum2 = 0.0f, lsum3 = 0.0f;
                const float neg_m = -m_ref;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float x0, x1, x2, x3;
                        ffma2_bcast(x0, x1, __uint_as_float(sv[c][j]), __uint_as_float(sv[c][j + 1]), a.t.scale_log2, neg_m);
                        ffma2_bcast(x2, x3, __uint_as_float(sv[c][j + 2]), __uint_as_float(sv[c][j + 3]), a.t.scale_log2, neg_m);
                        float p0, p1, p2, p3;
                        if (((j / 4) * 2) % 8 < EMU) ex2_emu2_nan(p0, p1, x0, x1);
                        else { p0 = ex2_approx(x0); p1 = ex2_approx(x1); }
                        if (((j / 4) * 2 + 1) % 8 < EMU) ex2_emu2_nan(p2, p3, x2, x3);
                        else { p2 = ex2_approx(x2); p3 = ex2_approx(x3); }
                        fadd2_acc(lsum0, lsum1, p0, p1);
                        fadd2_acc(lsum2, lsum3, p2, p3);
                        pk[j / 2] = pack2<T>(p0, p1);
                        pk[j / 2 + 1] = pack2<T>(p2, p3);
                    }
                    tmem_st16(s_addr + c * 16, pk);    // over the scores, all of which are in registers
                    if (c & 1) {
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(b_pfull + 4 * (c & 2));
                    }
                }
                l_run += (lsum0 + lsum1) + (lsum2 + lsum3);
            }
            // the item's last P V of this tile, then the row goes out
            ok = __all_sync(0xffffffffu, ok && mbar_wait(b_ofull, si & 1, bt.status));
            ++si;
            if (!ok) continue;
            tc_fence_after();
            const bool row_valid = ql < a.QT && qi < q.n;
            if (m_ref == kLow) l_run = 0.0f;       // every score was masked: what the polynomial makes of -infinity is no weight
            const float inv = l_run == 0.0f ? 0.0f : (l_run < kSumLimit ? 1.0f / l_run : NAN);
            float* set = slot >= 0 ? a.part + slot * partial_floats(2 * kCkRows, D) : nullptr;
            long long rows[4];
            quad_rows(row_valid ? ((long long)(q.start + qi) * H + (long long)kvh * G + g) * D : -1, rows);
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {            // (a loop: straight-line code is fetched once per item here)
                uint32_t v[32];
                tmem_ld32(v, o_addr + c * 32);
                tc_wait_ld_dep(v);
                if (c * 32 >= D) continue;                 // columns of zeros (head_dim 96)
                if (set) store_partial32(set, 2 * kCkRows, grp * kCkRows + row, c * 32, v);
                else store_rows32<T>((T*)a.t.out, rows, c * 32, v, inv);
            }
            if (set) *reinterpret_cast<float2*>(set + (2 * kCkRows) * D + 2 * (grp * kCkRows + row)) = make_float2(m_ref, l_run);
            tc_fence_before();
        }
    }
    if (tid == 0) wait_for_previous();         // the few-token kernel of the call, where it ran ahead: this launch ends behind it
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace hkv
