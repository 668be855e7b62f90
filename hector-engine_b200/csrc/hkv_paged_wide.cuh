// hkv_paged_wide.cuh — attention of prompt chunks over a paged cache on the 5th-generation tensor cores, head_dim 256.
//
// Two query tiles do not fit tensor memory beside 256 output columns, and a 64 KB query tile would take the shared memory
// that K and V need. So one tile of 128 query rows per CTA, and its queries live in TENSOR memory as the A operand:
//   columns: O [0,256)  Q [256,384) (two elements per column)  S_0 [384,448)  S_1 [448,512), P over the first half of its S.
// Shared memory holds K and V tiles of 64 positions only (32 KB each, rings of 3), and the score product reads nothing but
// K from it: with Q in shared memory too, an M128 x N64 product would want 192 bytes a clock where 128 are to be had.
// Two threads per row (each half of the score columns, half of the output dimensions) exchange their maxima through
// shared memory. Issue order: QK(0) QK(1) | PV(0) QK(2) | PV(1) QK(3) ...: the scores of tile t+1 are computed under the
// softmax of tile t. Work comes off the same line as in hkv_paged_chunk.cuh, with items of one tile.
// Bound: K and V out of the L2 (64 KB per tile and SM, read again for every 128 query rows) and the products, 0.8 us of a
// tile's 1.0 to 1.25 us. Measured: 1 024 queries over 16k keys, 16 heads of 8, 279 us (955 TFLOP/s); 4 x 500 tokens in a
// window of 1 024: 93 us, of which 12 us joining cut items. Half of the traffic would go with two SMs sharing a tile's
// products.
#pragma once

#include "hkv_paged_chunk.cuh"

namespace hkv {

constexpr int kWdKeys = 64;
constexpr int kWdStages = 3;
constexpr int kWdThreads = 320;           // 8 softmax warps, producer, MMA issuer
constexpr int kWdHD = 256;
__host__ __device__ constexpr size_t wide_smem_bytes(int requests) {
    return 1024 + (size_t)2 * kWdStages * kWdKeys * kWdHD * 2 + 40 * 8 + 16 + 4 * kCkDesc * 4 + 6 * kCkRows * 4 + (size_t)(requests + 1) * 4 + 16;
}

template <typename T>
__global__ void __launch_bounds__(kWdThreads, 1)
hkv_paged_wide_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PagedChunkArgs a) {
    constexpr int HD = kWdHD, NCH = HD / 64;
    constexpr int TILE_BYTES = kWdKeys * HD * 2;
    constexpr int CHUNK_OFF = 1024, GROUP_OFF = NCH * 1024;   // staged tiles: [8-row group][column block][8 rows of 128 bytes]
    constexpr uint32_t TMEM_COLS = 512, COL_O = 0, COL_Q = 256, COL_S = 384;   // S: + 64 * (tile & 1)
    constexpr int KH = kWdKeys / 2, HH = HD / 2;           // score columns, output dimensions per thread
    constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t IDESC_QK = FMT | (1u << 4) | ((uint32_t)(kWdKeys >> 3) << 17) | ((uint32_t)(kCkRows >> 4) << 24);
    constexpr uint32_t IDESC_PV = FMT | (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kCkRows >> 4) << 24);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* v_gen = smem + kWdStages * TILE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_gen + kWdStages * TILE_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 40);
    volatile int* queue = reinterpret_cast<volatile int*>(tmem_slot + 4);      // [4][kCkDesc]
    float* xch = reinterpret_cast<float*>(tmem_slot + 4 + 4 * kCkDesc);        // [2 tiles][2 halves][128] maxima, [2][128] sums
    uint32_t* pre = reinterpret_cast<uint32_t*>(xch + 6 * kCkRows);            // [requests + 1]
    __shared__ long long scan_buf[33];
    const uint32_t k_smem = smem_u32(smem), v_smem = smem_u32(v_gen), bar0 = smem_u32(bars);
    const uint32_t B_QFULL = bar0, B_PV = bar0 + 16, B_OFULL = bar0 + 24, B_DONE = bar0 + 32, B_XCH = bar0 + 40,
                   B_SFULL = bar0 + 48 /* [2] */, B_KFULL = bar0 + 64 /* [3] */, B_KEMPTY = bar0 + 88, B_VFULL = bar0 + 112,
                   B_VEMPTY = bar0 + 136, B_WF = bar0 + 160 /* [4] */, B_WE = bar0 + 192,
                   // one per score buffer: P(t+1) may be complete before the issuer, held up by V(t), looks for P(t)
                   B_PFULL = bar0 + 224 /* [2] */;
    const PagedBatch& bt = a.t.b;
    const int G = a.line.G, H = a.t.H;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    launch_dependents();
    if (tid == 0) {
        mbar_init(B_QFULL, 256); mbar_init(B_PV, 1); mbar_init(B_OFULL, 1); mbar_init(B_DONE, 1);
        mbar_init(B_XCH, 256);
        for (int s = 0; s < 2; ++s) { mbar_init(B_SFULL + 8 * s, 1); mbar_init(B_PFULL + 8 * s, 256); }
        for (int s = 0; s < kWdStages; ++s) {
            mbar_init(B_KFULL + 8 * s, 1); mbar_init(B_KEMPTY + 8 * s, 1);
            mbar_init(B_VFULL + 8 * s, 1); mbar_init(B_VEMPTY + 8 * s, 1);
        }
        for (int i = 0; i < 4; ++i) { mbar_init(B_WF + 8 * i, 1); mbar_init(B_WE + 8 * i, 9); }
        fence_mbar_init();
        tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
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
    auto queue_wait = [&](uint32_t k) -> bool { return mbar_wait(B_WF + 8 * (k & 3), (k >> 2) & 1, bt.status); };

    if (warp == 8) {
        // ------------------------------ producer (the whole warp) ------------------------------
        uint32_t gt = 0, it = 0;
        bool ok = true;
        auto publish = [&](int r, const PagedRequest& q, int kvh, int p, int kt, int nt, int slot) -> bool {
            const uint32_t s = it & 3;
            if (it >= 4 && !__all_sync(0xffffffffu, mbar_wait(B_WE + 8 * s, ((it >> 2) - 1) & 1, bt.status))) return false;
            if (lane == 0) {
                volatile int* d = queue + s * kCkDesc;
                d[0] = r; d[1] = kvh; d[2] = p; d[3] = kt; d[4] = nt; d[5] = slot;
                d[7] = q.start; d[8] = q.n; d[9] = q.pos0; d[10] = q.keys;
                mbar_arrive(B_WF + 8 * s);
            }
            __syncwarp();
            return true;
        };
        const int page_shift = 31 - __clz(bt.page);
        const int my_piece = lane % a.pieces;
        chunk_walk(bt, line, W, ctas, blockIdx.x, [&](int r, const PagedRequest& q, int kvh, int p, int kt, int nt, int slot) -> bool {
            if (!publish(r, q, kvh, p, kt, nt, slot)) { ok = false; return false; }
            ++it;
            const int i0 = p * a.line.QB, i1 = (i0 + a.line.QB < q.n ? i0 + a.line.QB : q.n) - 1;
            int lo, hi, x;
            paged_key_range(bt, q, i0, lo, x);
            paged_key_range(bt, q, i1, x, hi);
            const int32_t* table = bt.table + (long long)r * bt.cols;
            auto look_up = [&](int pos) -> int {       // behind the tensor (zeros) where no query of the item looks
                if (paged_box_hidden(pos, a.box_rows, lo, hi)) return bt.pages;
                const int pg = __ldg(table + (pos >> page_shift));
                if (pg >= 0 && pg < bt.pages) return pg;
                atomicOr(bt.status, kStatusBoundCheck);
                return bt.pages;
            };
            int pg = look_up(kt * kWdKeys + my_piece * a.box_rows);
            for (int t = 0; t < nt; ++t, ++gt) {
                const int pos0 = (kt + t) * kWdKeys;
                const int pg_next = t + 1 < nt ? look_up(pos0 + kWdKeys + my_piece * a.box_rows) : 0;
                const uint32_t s = gt % kWdStages, ph = (gt / kWdStages) & 1;
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
                    if (lane < a.pieces) {             // one box per page, all column blocks
                        const int at = lane * a.box_rows;
                        tma_load_4d(dst + (at >> 3) * GROUP_OFF, kv ? &tm_v : &tm_k, full, 0, 0, kvh * NCH,
                                    (pg << (page_shift - 3)) + (((pos0 + at) & (bt.page - 1)) >> 3));
                    }
                }
                pg = pg_next;
            }
            return true;
        });
        const PagedRequest none{0, 0, 0, 0};
        publish(-1, none, 0, 0, 0, 0, 0);
        if (lane == 0)
            for (uint32_t i = 1; i <= (uint32_t)kWdStages && i <= gt; ++i) {
                const uint32_t g = gt - i;
                mbar_wait(B_KFULL + 8 * (g % kWdStages), (g / kWdStages) & 1, bt.status);
                mbar_wait(B_VFULL + 8 * (g % kWdStages), (g / kWdStages) & 1, bt.status);
            }
        __syncwarp();
        chunk_cut_entry(bt, line, W, ctas, blockIdx.x, a.cuts);
    } else if (warp == 9) {
        // ------------------------------ MMA issuer ------------------------------
        if (elect_one()) {
            uint32_t gt = 0, it = 0;
            bool ok = true;
            const uint64_t kdesc0 = umma_desc_sw128(k_smem, 16, GROUP_OFF), vdesc0 = umma_desc_sw128(v_smem, CHUNK_OFF, GROUP_OFF);
            const uint32_t desc_hi = (uint32_t)(kdesc0 >> 32), k_lo = (uint32_t)kdesc0, v_lo = (uint32_t)vdesc0;
            auto issue_qk = [&](uint32_t g) -> bool {      // S_(g&1) = Q K(g)^T
                const uint32_t s = g % kWdStages;
                if (!mbar_wait(B_KFULL + 8 * s, (g / kWdStages) & 1, bt.status)) return false;
                tc_fence_after();
                const uint32_t kd = k_lo + ((s * TILE_BYTES) >> 4), d = tmem + COL_S + 64u * (g & 1), qa = tmem + COL_Q;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t off = (uint32_t)(((kk / 4) * CHUNK_OFF + (kk % 4) * 32) >> 4);
                    if (kk == 0) tc_mma_ts_i<false>(d, qa + kk * 8, kd + off, desc_hi, IDESC_QK);
                    else tc_mma_ts_i<true>(d, qa + kk * 8, kd + off, desc_hi, IDESC_QK);
                }
                tc_commit(B_SFULL + 8 * (g & 1));
                tc_commit(B_KEMPTY + 8 * s);
                return true;
            };
            for (; ok; ++it) {
                if (!queue_wait(it)) { ok = false; break; }
                const volatile int* d = queue + (it & 3) * kCkDesc;
                const int r = d[0], nt = d[4];
                mbar_arrive(B_WE + 8 * (it & 3));
                if (r < 0) break;
                if (!mbar_wait(B_QFULL, it & 1, bt.status)) { ok = false; break; }
                tc_fence_after();
                if (!issue_qk(gt) || (nt > 1 && !issue_qk(gt + 1))) { ok = false; break; }
                for (int t = 0; t < nt; ++t, ++gt) {
                    const uint32_t s = gt % kWdStages;
                    if (!mbar_wait(B_VFULL + 8 * s, (gt / kWdStages) & 1, bt.status) || !mbar_wait(B_PFULL + 8 * (gt & 1), (gt >> 1) & 1, bt.status)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t vd = v_lo + ((s * TILE_BYTES) >> 4), pbase = tmem + COL_S + 64u * (gt & 1), o = tmem + COL_O;
                    if (t > 0) tc_mma_ts_i<true>(o, pbase, vd, desc_hi, IDESC_PV);
                    else tc_mma_ts_i<false>(o, pbase, vd, desc_hi, IDESC_PV);
#pragma unroll
                    for (int kk = 1; kk < kWdKeys / 16; ++kk)
                        tc_mma_ts_i<true>(o, pbase + kk * 8, vd + (uint32_t)((kk * 2 * GROUP_OFF) >> 4), desc_hi, IDESC_PV);
                    tc_commit(B_PV);
                    if (t + 1 == nt) tc_commit(B_OFULL);
                    tc_commit(B_VEMPTY + 8 * s);
                    // the scores of tile t+2 go where P(t) was: behind its product on the same in-order pipe
                    if (t + 2 < nt && !issue_qk(gt + 2)) { ok = false; break; }
                }
            }
            tc_commit(B_DONE);
            mbar_wait(B_DONE, 0, bt.status);
        }
    } else {
        // ------------------------------ softmax / output rows ------------------------------
        const int quad = warp & 3, half = warp >> 2;
        const int row = quad * 32 + lane;
        const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
        const int ql = row / G, g = row % G;
        uint32_t gt = 0, xn = 0, si = 0;   // tiles, exchanges, items (barrier phases)
        bool ok = true;
        for (uint32_t qk = 0; ok; ++qk) {
            ok = __all_sync(0xffffffffu, queue_wait(qk));
            if (!ok) break;
            const volatile int* d = queue + (qk & 3) * kCkDesc;
            const int r = d[0], kvh = d[1], p = d[2], kt = d[3], nt = d[4], slot = d[5];
            PagedRequest q;
            q.start = d[7]; q.n = d[8]; q.pos0 = d[9]; q.keys = d[10];
            __syncwarp();
            if (lane == 0) mbar_arrive(B_WE + 8 * (qk & 3));
            if (r < 0) break;
            const int i0 = p * a.line.QB, qi = i0 + ql;
            const bool row_valid = ql < a.QT && qi < q.n;
            // ---- this thread's half of the query row into tensor memory (rows without a query: zeros). The previous item's
            // products, the last readers of these columns, have completed: its output was waited for. ----
            {
                const T* qp = (const T*)a.t.q + (long long)(q.start + qi) * a.t.q_stride + ((long long)kvh * G + g) * HD + half * HH;
#pragma unroll
                for (int c = 0; c < HH / 64; ++c) {
                    uint32_t v[32];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint4 x = row_valid ? *reinterpret_cast<const uint4*>(qp + c * 64 + e * 8) : make_uint4(0, 0, 0, 0);
                        v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
                    }
                    tmem_st32(tmem + lane_sel + COL_Q + half * (HH / 2) + c * 32, v);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(B_QFULL);
            }
            int lo_row, hi_row, lo_last, hi_first, x;
            paged_key_range(bt, q, qi < q.n ? qi : q.n - 1, lo_row, hi_row);
            paged_key_range(bt, q, i0, x, hi_first);
            paged_key_range(bt, q, (i0 + a.line.QB < q.n ? i0 + a.line.QB : q.n) - 1, lo_last, x);
            float m_ref = kLow, l_run = 0.0f;

            for (int t = 0; t < nt; ++t, ++gt) {
                const uint32_t sb = gt & 1;
                const uint32_t s_base = tmem + lane_sel + COL_S + 64u * sb;
                ok = __all_sync(0xffffffffu, ok && mbar_wait(B_SFULL + 8 * sb, (gt >> 1) & 1, bt.status));
                if (!ok) continue;
                tc_fence_after();
                uint32_t sv[KH];
                tmem_ld32(sv, s_base + half * KH);
                const int kstart = (kt + t) * kWdKeys;
                const int lo = lo_row - kstart - half * KH, hi = hi_row - kstart - half * KH;   // attended columns [lo, hi) of this half
                const bool all_in = __all_sync(0xffffffffu, lo <= 0 && hi >= KH);
                tc_wait_ld_dep(sv);
                float mx;
                {
                    float m0 = -INFINITY, m1 = -INFINITY;
                    if (all_in) {
#pragma unroll
                        for (int j = 0; j < KH; j += 4) {
                            m0 = fmax3(m0, __uint_as_float(sv[j]), __uint_as_float(sv[j + 1]));
                            m1 = fmax3(m1, __uint_as_float(sv[j + 2]), __uint_as_float(sv[j + 3]));
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < KH; ++j) {
                            const float sc = (j >= lo && j < hi) ? __uint_as_float(sv[j]) : -INFINITY;
                            sv[j] = __float_as_uint(sc);
                            m0 = fmaxf(m0, sc);
                        }
                    }
                    mx = fmaxf(m0, m1) * a.t.scale_log2;
                }
                // the row's maximum over both halves; past this exchange both have their scores in registers
                xch[(sb * 2 + half) * kCkRows + row] = mx;
                mbar_arrive(B_XCH);
                ok = __all_sync(0xffffffffu, mbar_wait(B_XCH, xn & 1, bt.status));
                ++xn;
                if (!ok) continue;
                mx = fmaxf(mx, xch[(sb * 2 + (half ^ 1)) * kCkRows + row]);
                const bool move = mx > m_ref + 8.0f;
                if (__any_sync(0xffffffffu, move)) {
                    const float m_to = move ? mx : m_ref;
                    const float alpha = ex2_approx(m_ref - m_to);
                    if (t > 0) {
                        // every earlier P V must have landed. (The scores of this tile were issued after P V of tile t-2, so
                        // the barrier is at most one phase behind and the parity wait is sound.)
                        ok = __all_sync(0xffffffffu, mbar_wait(B_PV, (gt - 1) & 1, bt.status));
                        if (!ok) continue;
                        tc_fence_after();
                        tmem_scale_columns(tmem + lane_sel + COL_O + half * HH, HH / 32, alpha);
                    }
                    l_run *= alpha;
                    m_ref = m_to;
                }
                float lsum0 = 0.0f, lsum1 = 0.0f;
                const float neg_m = -m_ref;
                uint32_t pk[KH / 2];
#pragma unroll
                for (int j = 0; j < KH; j += 2) {
                    float x0, x1;
                    ffma2_bcast(x0, x1, __uint_as_float(sv[j]), __uint_as_float(sv[j + 1]), a.t.scale_log2, neg_m);
                    const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                    fadd2_acc(lsum0, lsum1, p0, p1);
                    pk[j / 2] = pack2<T>(p0, p1);
                }
                tmem_st16(s_base + half * (KH / 2), pk);
                tc_wait_st();
                l_run += lsum0 + lsum1;
                // tiles that not every query of the item sees whole: rows that none attends and values that are not finite
                if (paged_tile_masked(kstart, kWdKeys, lo_last, hi_first)) {
                    const uint32_t vs = gt % kWdStages;
                    ok = __all_sync(0xffffffffu, mbar_wait(B_VFULL + 8 * vs, (gt / kWdStages) & 1, bt.status));
                    if (!ok) continue;
                    const bool bad = clean_values<T, NCH, 256>(bt, q, i0, a.line.QB, kstart, kWdKeys, v_gen + (size_t)vs * TILE_BYTES,
                                                               CHUNK_OFF, GROUP_OFF, tid);
                    if (__any_sync(0xffffffffu, bad) && lane == 0) a.fix.push(r, p, kvh);
                    fence_proxy_async_smem();
                }
                tc_fence_before();
                mbar_arrive(B_PFULL + 8 * sb);
            }
            float l_tot = l_run;
            if (ok) {                              // sum of both halves (same reference)
                xch[4 * kCkRows + half * kCkRows + row] = l_run;
                mbar_arrive(B_XCH);
                ok = __all_sync(0xffffffffu, mbar_wait(B_XCH, xn & 1, bt.status));
                ++xn;
                l_tot += xch[4 * kCkRows + (half ^ 1) * kCkRows + row];
            }
            ok = __all_sync(0xffffffffu, ok && mbar_wait(B_OFULL, si & 1, bt.status));
            ++si;
            if (!ok) continue;
            tc_fence_after();
            const float inv = l_tot == 0.0f ? 0.0f : (l_tot < kSumLimit ? 1.0f / l_tot : NAN);
            float* set = slot >= 0 ? a.part + slot * partial_floats(kCkRows, HD) : nullptr;
            long long rows[4];
            quad_rows(row_valid ? ((long long)(q.start + qi) * H + (long long)kvh * G + g) * HD : -1, rows);
#pragma unroll 1
            for (int c = 0; c < HH / 32; ++c) {
                const int d0 = half * HH + c * 32;
                uint32_t v[32];
                tmem_ld32(v, tmem + lane_sel + COL_O + d0);
                tc_wait_ld_dep(v);
                if (set) store_partial32(set, kCkRows, row, d0, v);
                else store_rows32<T>((T*)a.t.out, rows, d0, v, inv);
            }
            if (set && half == 0) *reinterpret_cast<float2*>(set + kCkRows * HD + 2 * row) = make_float2(m_ref, l_tot);
            tc_fence_before();
        }
    }
    if (tid == 0) wait_for_previous();         // the few-token kernel of the call, where it ran ahead: this launch ends behind it
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace hkv
