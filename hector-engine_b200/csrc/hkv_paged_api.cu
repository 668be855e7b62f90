// hkv_paged_api.cu — C ABI of the paged cache (declared in include/hkv.h): argument checks, the context with its
// workspace, dispatch. Host side only enqueues work; there is no CPU compute path.

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <new>
#include <string>

#include "../../include/hkv.h"
#include "hkv_paged.cuh"
#include "hkv_paged_chunk.cuh"
#include "hkv_paged_decode.cuh"
#include "hkv_paged_finish.cuh"
#include "hkv_paged_rope.cuh"
#include "hkv_paged_wide.cuh"

using namespace hkv;

struct hkv_paged_ctx {
    hkv_paged_geometry g;
    int device = -1;
    int sm_count = 0;
    int32_t* d_status = nullptr;
    int* plan_done = nullptr;       // CTAs of a plan launch that have finished (zero between launches)
    size_t smem_optin = 0, smem_sm = 0;
    bool staged = false;            // the geometry allows the staged kernels
    // attention workspace: partial rows of cut requests and where they are, items to be done again
    float *part = nullptr, *chunk_part = nullptr;
    int4 *cuts = nullptr, *chunk_cuts = nullptr;
    int4* fix = nullptr;            // [1 + kFixMax], the count in the first
    size_t workspace_bytes = 0;
    bool ready = false;
    std::string err;
};

namespace {

int fail(hkv_paged_ctx* c, int code, const char* msg) {
    if (c) {
        try { c->err = msg; } catch (...) {}
    }
    return code;
}
int fail_cuda(hkv_paged_ctx* c, cudaError_t e, const char* where) {
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", where, cudaGetErrorString(e));
    return fail(c, HKV_ERR_CUDA, buf);
}
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

int validate(const hkv_paged_geometry* g, const char** why) {
    if (!g) { *why = "geometry is null"; return HKV_ERR_INVALID_ARG; }
    if (g->dtype != HKV_DTYPE_F16 && g->dtype != HKV_DTYPE_BF16) { *why = "unknown dtype"; return HKV_ERR_INVALID_ARG; }
    if (g->head_dim <= 0 || g->head_dim > 512 || g->num_kv_heads <= 0 || g->num_heads <= 0 ||
        g->num_heads % g->num_kv_heads != 0 || g->num_heads > 65535) {
        *why = "unsupported head geometry";
        return HKV_ERR_GEOMETRY;
    }
    if (g->page_size <= 0 || g->num_pages <= 0 || g->max_requests <= 0 || g->max_pages <= 0 || g->max_tokens <= 0 ||
        g->window_size < 0) {
        *why = "page_size, num_pages, max_requests, max_pages and max_tokens must be positive, window_size non-negative";
        return HKV_ERR_INVALID_ARG;
    }
    if (g->kernel_select < 0 || g->kernel_select > 2 || (g->flags & ~HKV_FLAG_APPEND_ONLY) != 0 || g->reserved[0] ||
        g->reserved[1] || g->reserved[2] || g->reserved[3]) {
        *why = "unknown kernel_select or flag, or a reserved field set";
        return HKV_ERR_INVALID_ARG;
    }
    if (g->max_requests > HKV_PAGED_MAX_REQUESTS) { *why = "max_requests exceeds HKV_PAGED_MAX_REQUESTS"; return HKV_ERR_TOO_LARGE; }
    if ((long long)g->num_pages * g->page_size > 0x7fffffffll || (long long)g->max_pages * g->page_size > 0x7fffffffll) {
        *why = "num_pages * page_size and max_pages * page_size are limited to 2^31 - 1";
        return HKV_ERR_TOO_LARGE;
    }
    return HKV_OK;
}

int check(hkv_paged_ctx* c) {
    if (!c) return HKV_ERR_INVALID_ARG;
    if (!c->ready) return fail(c, HKV_ERR_INVALID_ARG, "context not initialised");
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return fail(c, HKV_ERR_CUDA, "cudaGetDevice failed");
    }
    if (dev != c->device) {
        char buf[96];
        snprintf(buf, sizeof buf, "context belongs to device %d, current device is %d", c->device, dev);
        return fail(c, HKV_ERR_INVALID_ARG, buf);
    }
    return HKV_OK;
}
#define PAGED_CHECK(c)                  \
    do {                                \
        const int chk_ = check(c);      \
        if (chk_ != HKV_OK) return chk_; \
    } while (0)

int launched(hkv_paged_ctx* c, const char* what) {
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? HKV_OK : fail_cuda(c, e, what);
}

// ---- staged kernels -----------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            return reinterpret_cast<EncodeTiledFn>(p);
        return (EncodeTiledFn) nullptr;
    }();
    return fn;
}

// head_dim 64, 96, 128, 256; pages of a power of two of rows, at least 8 (a box of the copy engine is a whole number of
// 8-row swizzle groups and never crosses a page); groups up to 128.
bool staged_geometry(const hkv_paged_geometry& g) {
    const int G = g.num_heads / g.num_kv_heads;
    const bool hd = g.head_dim == 64 || g.head_dim == 96 || g.head_dim == 128 || g.head_dim == 256;
    // (the few-token kernel counts the tiles of all requests in 31 bits)
    const bool count = (double)g.max_requests * ((double)g.max_pages * g.page_size / kTileRows + 1.0) < 2.0e9;
    return hd && count && G <= 128 && g.page_size >= 8 && (g.page_size & (g.page_size - 1)) == 0;
}

// Map of a plane with its rows in groups of 8, [group of the pool][column block][row][width elements], so that one box holds
// `rows` rows of one KV head and lands as whole swizzle groups; the third coordinate counts column blocks. Where head_dim is
// not a whole number of blocks (96 in blocks of 64) it counts heads and a box is one block, the last one half outside (zeros).
int encode_tiles(hkv_paged_ctx* c, const void* base, int width, int rows, CUtensorMap* out) {
    const hkv_paged_geometry& g = c->g;
    const bool whole = g.head_dim % width == 0;
    const int blocks = whole ? g.head_dim / width : 1;
    const cuuint64_t row = (cuuint64_t)g.num_kv_heads * g.head_dim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)(whole ? width : g.head_dim), 8u, (cuuint64_t)g.num_kv_heads * blocks,
                                (cuuint64_t)g.num_pages * g.page_size / 8};
    const cuuint64_t strides[3] = {row, (cuuint64_t)(whole ? width : g.head_dim) * 2, row * 8};
    const cuuint32_t box[4] = {(cuuint32_t)width, 8u, (cuuint32_t)blocks, (cuuint32_t)rows / 8}, one[4] = {1u, 1u, 1u, 1u};
    const CUresult r = encode_tiled_fn()(
        out, g.dtype == HKV_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
        width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return HKV_OK;
    char buf[96];
    snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return fail(c, HKV_ERR_CUDA, buf);
}

// A launch configuration; `early`: it may be set up (and run, up to its own wait) while the launch before it still runs.
struct Launch {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    Launch(unsigned blocks, unsigned threads, size_t smem, cudaStream_t st, bool early) {
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    Launch(const Launch&) = delete;
};

PagedFix fix_of(const hkv_paged_ctx* c) { return PagedFix{reinterpret_cast<int*>(c->fix), c->fix + 1}; }

typedef void (*DecodeKernel)(const CUtensorMap, const CUtensorMap, const PagedDecodeArgs, const int);
template <typename T, int HD>
DecodeKernel pick_decode_hd(int nt, int groups) {
    if (nt == 1) return groups == 1 ? hkv_paged_decode_kernel<T, HD, 1, 1> : hkv_paged_decode_kernel<T, HD, 1, 2>;
    if (HD == 256) return hkv_paged_decode_kernel<T, HD, 2, 1>;    // (two groups of it do not fit the registers)
    return groups == 1 ? hkv_paged_decode_kernel<T, HD, 2, 1> : hkv_paged_decode_kernel<T, HD, 2, 2>;
}
template <typename T>
DecodeKernel pick_decode_t(int hd, int nt, int groups) {
    return hd == 64 ? pick_decode_hd<T, 64>(nt, groups) : hd == 96 ? pick_decode_hd<T, 96>(nt, groups)
         : hd == 128 ? pick_decode_hd<T, 128>(nt, groups) : pick_decode_hd<T, 256>(nt, groups);
}
DecodeKernel pick_decode(int dtype, int hd, int nt, int groups) {
    return dtype == HKV_DTYPE_F16 ? pick_decode_t<__half>(hd, nt, groups) : pick_decode_t<__nv_bfloat16>(hd, nt, groups);
}

// CTAs that share a span: one per KV head, or two, four, eight heads per CTA where that leaves fewer CTAs idle. Up to 6 %
// idle CTAs are taken rather than more heads one after the other, each with its own first copies and merge. (4 requests of
// 4k keys, this rule / one head per CTA wherever they fit / the fewest idle: 64 heads of 64 49.6 / 50.9 / 55.1 us, 32 heads of 256
// 94 / 87 / 111, 40 heads of 128 57 / 57 / 71, 12 heads of 64 14.4 / 14.4 / 15.5; 32 such requests: 64 heads of 64 334 / 348 / 346,
// 40 of 128 387 / 390 / 406, 32 of 256 633 / 637 / 640.)
int gang_for(int kv_heads, int grid) {
    int best = 1;
    double best_util = 0.0;
    for (int per_cta = 1; per_cta <= 8; per_cta *= 2) {
        if (kv_heads % per_cta != 0) break;
        const int gang = kv_heads / per_cta;
        if (gang > grid) continue;
        const double util = (double)(grid / gang) * gang / grid;
        if (util >= 0.94) return gang;
        if (util > best_util) { best_util = util; best = gang; }
    }
    return best;
}
size_t part_bytes(const hkv_paged_geometry& g, int sm_count) {
    size_t most = 0;
    for (int grid : {sm_count, 2 * sm_count})
        most = std::max(most, (size_t)2 * (grid / gang_for(g.num_kv_heads, grid)) * g.num_kv_heads * kSmallCols * (g.head_dim + 2) * 4);
    return most;
}

// Shape of the few-token kernel: two CTAs per SM with one consumer group each, or one CTA with two groups. Two stream a
// little faster and hide each other's merges; they also double the spans, and with them the parts a request is cut into,
// which is what a launch of one or two requests spends its time on: one CTA where a request would be cut into more than 40.
// (us, two CTAs / one: 1 request of 512 keys, 2 KV heads of 64 9.1 / 8.0, of 64k keys 17.4 / 18.6; 4 KV heads of 128 10.4 / 9.6
// and 32.3 / 32.6. 4 requests of 512 9.5 / 8.5 and 11.6 / 10.5, of 64k keys 33.6 / 46.3 and 90 / 95; 16 requests of 64k keys 96 / 157 and
// 315 / 340.)
struct DecodeShape { int groups, grid, gang; PagedDecodePlan plan; };
DecodeShape decode_shape(const hkv_paged_ctx* c, int cols, int requests) {
    const hkv_paged_geometry& g = c->g;
    DecodeShape s{};
    const int two = 2 * c->sm_count / gang_for(g.num_kv_heads, 2 * c->sm_count);
    const bool wide = g.head_dim == 256;     // its tiles need the whole shared memory
    s.groups = two / requests > 40 || wide ? 2 : 1;
    if (s.groups == 1) {
        s.plan = paged_decode_plan(g.head_dim, cols, 4, requests, c->smem_sm / 2 - 1024 - 2048);
        if (s.plan.stages < 2) s.groups = 2;
    }
    if (s.groups == 2) s.plan = paged_decode_plan(g.head_dim, cols, 8, requests, c->smem_optin);
    s.grid = s.groups == 1 ? 2 * c->sm_count : c->sm_count;
    if (s.plan.stages < 2 || (wide && cols > 8)) {   // one CTA per SM, one consumer group, the whole shared memory
        s.groups = 1;
        s.plan = paged_decode_plan(g.head_dim, cols, 4, requests, c->smem_optin);
        s.grid = c->sm_count;
    }
    s.gang = gang_for(g.num_kv_heads, s.grid);
    return s;
}

int launch_small(hkv_paged_ctx* c, const PagedAttnArgs& t, int cols, PagedFinishArgs& f, cudaStream_t st) {
    const hkv_paged_geometry& g = c->g;
    const DecodeShape s = decode_shape(c, cols, t.b.requests);
    if (s.plan.stages < 2) return fail(c, HKV_ERR_GEOMETRY, "attention: shared memory too small for two stages");
    CUtensorMap mk, mv;
    PagedDecodeArgs a{};
    a.t = t;
    a.part = c->part;
    a.cuts = c->cuts;
    a.fix = fix_of(c);
    a.gang = s.gang;
    a.cols = cols;
    a.box_rows = std::min(g.page_size, kTileRows);
    a.pieces = kTileRows / a.box_rows;
    int e = encode_tiles(c, t.k_cache, paged_chunk_width(g.head_dim), a.box_rows, &mk);
    if (!e) e = encode_tiles(c, t.v_cache, paged_chunk_width(g.head_dim), a.box_rows, &mv);
    if (e) return e;
    pick_decode(g.dtype, g.head_dim, cols > 8 ? 2 : 1, s.groups)<<<s.grid, (s.groups * 4 + 1) * 32, s.plan.bytes, st>>>(mk, mv, a, s.plan.stages);
    f.small_part = c->part;
    f.small_cuts = c->cuts;
    f.spans = s.grid / s.gang;
    f.cols = cols;
    return launched(c, "attention launch");
}

// ---- prompt chunks ----
int staged_hd(int hd) { return hd == 96 ? 128 : hd; }
bool wide(const hkv_paged_geometry& g) { return g.head_dim == kWdHD; }    // one query tile per item, keys by 64
// Queries per item of the prompt kernels.
int block_queries(const hkv_paged_geometry& g) { return (wide(g) ? 1 : 2) * (kCkRows / (g.num_heads / g.num_kv_heads)); }
size_t chunk_smem(const hkv_paged_geometry& g, int requests) {
    return wide(g) ? wide_smem_bytes(requests) : chunk_smem_bytes(staged_hd(g.head_dim), requests);
}

typedef void (*ChunkKernel)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const PagedChunkArgs);
template <typename T>
ChunkKernel pick_chunk_t(int hd) {
    return hd == 64 ? hkv_paged_chunk_kernel<T, 64, true> : hd == 128 ? hkv_paged_chunk_kernel<T, 128, true> : hkv_paged_chunk_kernel<T, 128, false>;
}
ChunkKernel pick_chunk(int dtype, int hd) {
    return dtype == HKV_DTYPE_F16 ? pick_chunk_t<__half>(hd) : pick_chunk_t<__nv_bfloat16>(hd);
}
const void* chunk_kernel(const hkv_paged_geometry& g) {
    if (wide(g)) return g.dtype == HKV_DTYPE_F16 ? (const void*)hkv_paged_wide_kernel<__half> : (const void*)hkv_paged_wide_kernel<__nv_bfloat16>;
    return (const void*)pick_chunk(g.dtype, g.head_dim);
}
size_t chunk_part_bytes(const hkv_paged_geometry& g, int sm_count) { return 2ull * sm_count * partial_floats((wide(g) ? 1 : 2) * kCkRows, g.head_dim) * sizeof(float); }

int launch_chunk(hkv_paged_ctx* c, const PagedAttnArgs& t, const void* q, int small, PagedFinishArgs& f, cudaStream_t st) {
    const hkv_paged_geometry& g = c->g;
    const int G = g.num_heads / g.num_kv_heads;
    PagedChunkArgs a{};
    a.t = t;
    a.QT = kCkRows / G;
    a.line.G = G;
    a.line.KVH = g.num_kv_heads;
    a.line.QB = block_queries(g);
    a.line.keys = wide(g) ? kWdKeys : kCkKeys;
    a.line.shift = line_shift((double)g.max_pages * g.page_size, g.max_tokens, g.max_requests, g.num_kv_heads, a.line.QB);
    a.part = c->chunk_part;
    a.cuts = c->chunk_cuts;
    a.fix = fix_of(c);
    a.box_rows = std::min(g.page_size, a.line.keys);
    a.pieces = a.line.keys / a.box_rows;
    a.small = small;
    CUtensorMap mq, mk, mv;
    int e = encode_tiles(c, t.k_cache, 64, a.box_rows, &mk);
    if (!e) e = encode_tiles(c, t.v_cache, 64, a.box_rows, &mv);
    if (e) return e;
    const size_t smem = chunk_smem(g, t.b.requests);
    // behind a few-token launch this one starts where that one's CTAs leave room (neither reads what the other writes)
    const Launch l((unsigned)c->sm_count, wide(g) ? kWdThreads : kCkThreads, smem, st, small > 0);
    cudaError_t le;
    if (wide(g)) {
        le = g.dtype == HKV_DTYPE_F16 ? cudaLaunchKernelEx(&l.cfg, hkv_paged_wide_kernel<__half>, mk, mv, a)
                                      : cudaLaunchKernelEx(&l.cfg, hkv_paged_wide_kernel<__nv_bfloat16>, mk, mv, a);
    } else {
        const cuuint64_t dims[3] = {(cuuint64_t)g.head_dim, (cuuint64_t)g.num_heads, (cuuint64_t)t.b.tokens};
        const cuuint64_t strides[2] = {(cuuint64_t)g.head_dim * 2, (cuuint64_t)t.q_stride * 2};
        const cuuint32_t box[3] = {64u, (cuuint32_t)G, (cuuint32_t)a.QT}, one[3] = {1u, 1u, 1u};
        const CUresult r = encode_tiled_fn()(
            &mq, g.dtype == HKV_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q),
            dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return fail(c, HKV_ERR_CUDA, "cuTensorMapEncodeTiled failed (queries)");
        le = cudaLaunchKernelEx(&l.cfg, pick_chunk(g.dtype, g.head_dim), mq, mk, mv, a);
    }
    if (le != cudaSuccess) return fail_cuda(c, le, "attention launch");
    f.chunk_part = c->chunk_part;
    f.chunk_cuts = c->chunk_cuts;
    f.ctas = c->sm_count;
    f.tiles = wide(g) ? 1 : 2;
    f.QT = a.QT;
    return HKV_OK;
}

int launch_finish(hkv_paged_ctx* c, const PagedFinishArgs& f, cudaStream_t st) {
    const Launch l((unsigned)finish_blocks(f, c->g.num_kv_heads), 256, 0, st, true);
    const cudaError_t e = c->g.dtype == HKV_DTYPE_F16 ? cudaLaunchKernelEx(&l.cfg, hkv_paged_finish_kernel<__half>, f)
                                                       : cudaLaunchKernelEx(&l.cfg, hkv_paged_finish_kernel<__nv_bfloat16>, f);
    return e == cudaSuccess ? HKV_OK : fail_cuda(c, e, "attention finish launch");
}

template <typename T>
void launch_rope(const MropeArgs& a, int lph, unsigned blocks, cudaStream_t st) {
    switch (lph) {
        case 4: hkv_paged_norm_rope_kernel<T, 4><<<blocks, kMropeThreads, 0, st>>>(a); break;
        case 8: hkv_paged_norm_rope_kernel<T, 8><<<blocks, kMropeThreads, 0, st>>>(a); break;
        case 16: hkv_paged_norm_rope_kernel<T, 16><<<blocks, kMropeThreads, 0, st>>>(a); break;
        case 32: hkv_paged_norm_rope_kernel<T, 32><<<blocks, kMropeThreads, 0, st>>>(a); break;
        default: hkv_paged_norm_rope_any_kernel<T><<<blocks, kMropeThreads, 0, st>>>(a); break;
    }
}

// A token stride: 0 = dense, else at least one token's row.
bool stride_ok(int64_t given, long long row, long long* out) {
    if (given != 0 && given < row) return false;
    *out = given ? given : row;
    return true;
}

int attention(hkv_paged_ctx* c, const void* q, int64_t q_token_stride, const void* k_cache,
              const void* v_cache, void* out, const int32_t* d_block_table, const int32_t* d_q_start,
              const int32_t* d_step_len, const int32_t* d_key_len, int32_t requests, int32_t tokens, int32_t max_step,
              float scale, void* stream, bool causal) {
    PAGED_CHECK(c);
    const hkv_paged_geometry& g = c->g;
    if (g.flags & HKV_FLAG_APPEND_ONLY) return fail(c, HKV_ERR_WORKSPACE, "attention: the context was created append-only");
    if (!q || !k_cache || !v_cache || !out || !d_block_table || !d_q_start || !d_step_len || !d_key_len)
        return fail(c, HKV_ERR_INVALID_ARG, "attention: null argument");
    if (requests < 0 || tokens < 0 || max_step < 0) return fail(c, HKV_ERR_INVALID_ARG, "attention: negative count");
    if (requests > g.max_requests || tokens > g.max_tokens)
        return fail(c, HKV_ERR_TOO_LARGE, "attention: more requests or tokens than the context was created for");
    if (!std::isfinite(scale)) return fail(c, HKV_ERR_INVALID_ARG, "attention: scale is not finite");
    PagedAttnArgs a{};
    if (!stride_ok(q_token_stride, (long long)g.num_heads * g.head_dim, &a.q_stride))
        return fail(c, HKV_ERR_INVALID_ARG, "attention: q_token_stride smaller than one token's row");
    if (!aligned(q, 2) || !aligned(k_cache, 2) || !aligned(v_cache, 2) || !aligned(out, 2) || !aligned(d_block_table, 4) ||
        !aligned(d_q_start, 4) || !aligned(d_step_len, 4) || !aligned(d_key_len, 4))
        return fail(c, HKV_ERR_ALIGNMENT, "attention: a tensor is not aligned to its element size");
    if (requests == 0 || tokens == 0 || max_step == 0) return HKV_OK;
    // (rows that are done again read their queries after others of the call have been written)
    if (out == q) return fail(c, HKV_ERR_INVALID_ARG, "attention: out must not be q");
    a.b.table = d_block_table;
    a.b.q_start = d_q_start;
    a.b.step_len = d_step_len;
    a.b.key_len = d_key_len;
    a.b.status = c->d_status;
    a.b.requests = requests;
    a.b.cols = g.max_pages;
    a.b.page = g.page_size;
    a.b.pages = g.num_pages;
    a.b.tokens = tokens;
    a.b.max_step = max_step;
    a.b.window = causal ? g.window_size : 0;
    a.b.causal = causal ? 1 : 0;
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.out = out;
    a.H = g.num_heads;
    a.KVH = g.num_kv_heads;
    a.HD = g.head_dim;
    a.scale_log2 = scale * 1.4426950408889634f;
    const cudaStream_t st = (cudaStream_t)stream;
    const int G = g.num_heads / g.num_kv_heads;
    const bool tensors_ok = aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16) && a.q_stride % 8 == 0;
    const bool staged = c->staged && tensors_ok;
    if (!staged && g.kernel_select == HKV_KERNEL_TMA)
        return fail(c, HKV_ERR_ALIGNMENT, "attention: the staged kernels need 16-byte aligned tensors and strides");
    const bool only_small = (long long)max_step * G <= kSmallCols;
    // (the prompt kernel takes the row maximum before the scale, which it can for a positive one)
    if (!only_small && !(scale > 0.0f) && g.kernel_select == HKV_KERNEL_TMA)
        return fail(c, HKV_ERR_GEOMETRY, "attention: the staged kernels take chunks with a positive scale only");
    if (staged && (only_small || scale > 0.0f)) {
        // Query rows per KV head of the few-token kernel: all that the call can have, or, beside the prompt kernel, as many
        // tokens as fit one n8 tile (16 rows where a single token has more than 8): with two tiles every request of the
        // launch pays for the registers (head_dim 256: one consumer group instead of two). A call whose requests have 64
        // tokens or more on average leaves it out. (us, without / with, 28 heads of 4, 128 wide: 8 x 448 queries over 4k keys
        // 206 / 212, 2 048 over 32k keys 741 / 794; a prompt of 4 096 beside 63 single tokens over 512 keys each 195 / 217, over 4k
        // keys 299 / 287, over 32k keys 1 120 / 790 — there it loses, but the lengths that would tell are on the device.)
        const int small = only_small ? max_step * G : tokens / 64 >= requests ? 0 : G <= 8 ? 8 / G * G : G <= kSmallCols ? G : 0;
        PagedFinishArgs f{};
        f.t = a;
        f.fix = fix_of(c);
        f.QB = block_queries(g);
        f.may_fix = max_step > 1 ? 1 : 0;                // (nothing is hidden from a single query)
        int e = HKV_OK;
        if (small) e = launch_small(c, a, small, f, st);
        if (!e && !only_small) e = launch_chunk(c, a, q, small, f, st);
        return e ? e : launch_finish(c, f, st);
    }
    const dim3 grid((unsigned)tokens, (unsigned)g.num_heads);
    if (g.dtype == HKV_DTYPE_F16) hkv_paged_generic_kernel<__half><<<grid, kPagedGenWarps * 32, 0, st>>>(a);
    else hkv_paged_generic_kernel<__nv_bfloat16><<<grid, kPagedGenWarps * 32, 0, st>>>(a);
    return launched(c, "attention launch");
}

}  // namespace

extern "C" {

int hkv_paged_create(hkv_paged_ctx** out, const hkv_paged_geometry* geometry) {
    if (!out) return HKV_ERR_INVALID_ARG;
    *out = nullptr;
    hkv_paged_ctx* c = new (std::nothrow) hkv_paged_ctx();
    if (!c) return HKV_ERR_CUDA;
    *out = c;
    const char* why = "";
    const int vst = validate(geometry, &why);
    if (vst) return fail(c, vst, why);
    c->g = *geometry;
    int dev = 0, ndev = 0, major = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
        cudaGetLastError();
        return fail(c, HKV_ERR_NO_DEVICE, "no CUDA device");
    }
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaGetDevice");
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&c->sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (major != 10) return fail(c, HKV_ERR_NO_DEVICE, "device is not compute capability 10.x (built for sm_100a only)");
    c->device = dev;
    e = cudaMalloc(&c->d_status, 2 * sizeof(int32_t));
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(status)");
    c->plan_done = c->d_status + 1;
    e = cudaMemset(c->d_status, 0, 2 * sizeof(int32_t));
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaMemset(status)");
    e = cudaFuncSetAttribute((const void*)hkv_paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)plan_smem_bytes(kPagedMaxRequests));
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaFuncSetAttribute(plan shared memory)");
    int optin = 0, per_sm = 0;
    cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    cudaDeviceGetAttribute(&per_sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev);
    c->smem_optin = (size_t)optin;
    c->smem_sm = (size_t)per_sm;
    c->staged = staged_geometry(*geometry) && geometry->kernel_select != HKV_KERNEL_GENERIC;
    if (geometry->kernel_select == HKV_KERNEL_TMA && !c->staged)
        return fail(c, HKV_ERR_GEOMETRY, "the staged kernels need head_dim in {64,96,128,256}, group <= 128, page_size a power of two >= 8, and max_requests * max_pages * page_size below 1.28e11");
    if (c->staged && !(geometry->flags & HKV_FLAG_APPEND_ONLY)) {
        if (!encode_tiled_fn()) return fail(c, HKV_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
        for (int nt = 1; nt <= 2; ++nt)
            for (int groups = 1; groups <= 2; ++groups) {
                // the attribute belongs to the kernel: always the device maximum, so that contexts never lower it for each other
                e = cudaFuncSetAttribute((const void*)pick_decode(geometry->dtype, geometry->head_dim, nt, groups),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, optin - 2048);
                if (e != cudaSuccess) return fail_cuda(c, e, "cudaFuncSetAttribute(shared memory)");
            }
        c->smem_optin = (size_t)optin - 2048;   // (the kernels hold up to 1.3 KB of their own)
        {
            const size_t need = chunk_smem(*geometry, geometry->max_requests);
            if (need > c->smem_optin) return fail(c, HKV_ERR_TOO_LARGE, "shared memory too small for the request table");
            e = cudaFuncSetAttribute(chunk_kernel(*geometry), cudaFuncAttributeMaxDynamicSharedMemorySize, optin - 2048);
            if (e != cudaSuccess) return fail_cuda(c, e, "cudaFuncSetAttribute(shared memory)");
            const size_t cb = chunk_part_bytes(*geometry, c->sm_count);
            if ((e = cudaMalloc(&c->chunk_part, cb)) != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(partial rows)");
            if ((e = cudaMalloc(&c->chunk_cuts, sizeof(int4) * c->sm_count)) != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(cuts)");
            c->workspace_bytes += cb + sizeof(int4) * c->sm_count;
        }
        const size_t nb = part_bytes(*geometry, c->sm_count);
        if ((e = cudaMalloc(&c->part, nb)) != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(partial rows)");
        if ((e = cudaMalloc(&c->cuts, sizeof(int4) * 2 * c->sm_count)) != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(cuts)");
        if ((e = cudaMalloc(&c->fix, sizeof(int4) * (1 + kFixMax))) != cudaSuccess) return fail_cuda(c, e, "cudaMalloc(list)");
        if ((e = cudaMemset(c->fix, 0, sizeof(int4) * (1 + kFixMax))) != cudaSuccess) return fail_cuda(c, e, "cudaMemset(list)");
        c->workspace_bytes += nb + sizeof(int4) * (2 * c->sm_count + 1 + kFixMax);
    }
    // the memsets above went to the default stream, behind whatever is queued there; the first call may come on a stream
    // that does not wait for it
    if ((e = cudaStreamSynchronize(nullptr)) != cudaSuccess) return fail_cuda(c, e, "cudaStreamSynchronize(create)");
    c->ready = true;
    return HKV_OK;
}

int hkv_paged_destroy(hkv_paged_ctx* c) {
    if (!c) return HKV_OK;
    if (c->part) cudaFree(c->part);
    if (c->cuts) cudaFree(c->cuts);
    if (c->fix) cudaFree(c->fix);
    if (c->chunk_part) cudaFree(c->chunk_part);
    if (c->chunk_cuts) cudaFree(c->chunk_cuts);
    if (c->d_status) cudaFree(c->d_status);
    delete c;
    return HKV_OK;
}

const char* hkv_paged_last_error(const hkv_paged_ctx* c) { return c ? c->err.c_str() : "null context"; }
size_t hkv_paged_workspace_bytes(const hkv_paged_ctx* c) { return c ? c->workspace_bytes : 0; }

int hkv_paged_device_status(hkv_paged_ctx* c, void* stream, int32_t* status_out) {
    if (!c || !status_out) return HKV_ERR_INVALID_ARG;
    PAGED_CHECK(c);
    // read and cleared on the caller's stream, and over when this returns: on the default stream the clearing could come
    // after a kernel of a stream that does not wait for it, and take that kernel's bit
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyAsync(status_out, c->d_status, sizeof(int32_t), cudaMemcpyDeviceToHost, st);
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaMemcpyAsync(status)");
    e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return fail_cuda(c, e, "cudaStreamSynchronize");
    if (*status_out != 0) {
        e = cudaMemsetAsync(c->d_status, 0, sizeof(int32_t), st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
        if (e != cudaSuccess) return fail_cuda(c, e, "cudaMemsetAsync(status)");
        return fail(c, HKV_ERR_DEVICE_FAULT, "device status word is non-zero");
    }
    return HKV_OK;
}

int hkv_paged_plan(hkv_paged_ctx* c, int32_t requests, int32_t tokens, const int32_t* d_past_len,
                   const int32_t* d_new_len, int32_t* d_block_table, const int32_t* d_free_pages,
                   const int32_t* d_free_count, int32_t* d_total_len, int32_t* d_step_len, int32_t* d_q_start,
                   int32_t* d_slots, int32_t* d_positions, int32_t* d_free_left, void* stream) {
    PAGED_CHECK(c);
    if (!d_past_len || !d_new_len || !d_block_table || !d_free_pages || !d_free_count || !d_total_len || !d_step_len ||
        !d_q_start || !d_slots || !d_positions || !d_free_left)
        return fail(c, HKV_ERR_INVALID_ARG, "plan: null argument");
    if (requests < 0 || tokens < 0) return fail(c, HKV_ERR_INVALID_ARG, "plan: negative count");
    if (requests > c->g.max_requests || tokens > c->g.max_tokens)
        return fail(c, HKV_ERR_TOO_LARGE, "plan: more requests or tokens than the context was created for");
    for (const void* p : {(const void*)d_past_len, (const void*)d_new_len, (const void*)d_block_table, (const void*)d_free_pages,
                          (const void*)d_free_count, (const void*)d_total_len, (const void*)d_step_len, (const void*)d_q_start,
                          (const void*)d_slots, (const void*)d_positions, (const void*)d_free_left})
        if (!aligned(p, 4)) return fail(c, HKV_ERR_ALIGNMENT, "plan: an int32 array is not 4-byte aligned");
    PlanArgs a{};
    a.past = d_past_len;
    a.fresh = d_new_len;
    a.free_pages = d_free_pages;
    a.free_count = d_free_count;
    a.table = d_block_table;
    a.total = d_total_len;
    a.step = d_step_len;
    a.q_start = d_q_start;
    a.slots = d_slots;
    a.positions = d_positions;
    a.free_left = d_free_left;
    a.requests = requests;
    a.tokens = tokens;
    a.cols = c->g.max_pages;
    a.page = c->g.page_size;
    a.pages = c->g.num_pages;
    a.by_page = fast_div((uint32_t)c->g.page_size);
    // few requests and tokens: one small block (cheaper barriers); else two tokens per thread
    int threads = kPlanThreads;
    while (threads > 128 && threads / 2 * kPlanPer >= requests && threads >= tokens) threads /= 2;
    const int ctas = std::max(1, std::min((tokens + 2 * threads - 1) / (2 * threads), c->sm_count));
    a.done = ctas > 1 && (d_total_len == d_past_len || d_free_left == d_free_count) ? c->plan_done : nullptr;
    hkv_paged_plan_kernel<<<ctas, threads, plan_smem_bytes(requests), (cudaStream_t)stream>>>(a);
    return launched(c, "plan launch");
}

int hkv_paged_release(hkv_paged_ctx* c, int32_t requests, const int32_t* d_finished, int32_t* d_seq_len,
                      const int32_t* d_block_table, int32_t* d_free_pages, int32_t* d_free_count, void* stream) {
    PAGED_CHECK(c);
    if (!d_finished || !d_seq_len || !d_block_table || !d_free_pages || !d_free_count)
        return fail(c, HKV_ERR_INVALID_ARG, "release: null argument");
    if (requests < 0) return fail(c, HKV_ERR_INVALID_ARG, "release: negative count");
    if (requests > c->g.max_requests) return fail(c, HKV_ERR_TOO_LARGE, "release: more requests than the context was created for");
    for (const void* p : {(const void*)d_finished, (const void*)d_seq_len, (const void*)d_block_table,
                          (const void*)d_free_pages, (const void*)d_free_count})
        if (!aligned(p, 4)) return fail(c, HKV_ERR_ALIGNMENT, "release: an int32 array is not 4-byte aligned");
    if (requests == 0) return HKV_OK;
    ReleaseArgs a{};
    a.finished = d_finished;
    a.table = d_block_table;
    a.seq_len = d_seq_len;
    a.free_pages = d_free_pages;
    a.free_count = d_free_count;
    a.requests = requests;
    a.cols = c->g.max_pages;
    a.page = c->g.page_size;
    a.pages = c->g.num_pages;
    hkv_paged_release_kernel<<<1, kPlanThreads, (size_t)requests * 8, (cudaStream_t)stream>>>(a);
    return launched(c, "release launch");
}

int hkv_paged_append(hkv_paged_ctx* c, const void* k_new, const void* v_new, int64_t kv_token_stride, void* k_cache,
                     void* v_cache, const int32_t* d_slots, int32_t tokens, void* stream) {
    PAGED_CHECK(c);
    if (!k_new || !v_new || !k_cache || !v_cache || !d_slots) return fail(c, HKV_ERR_INVALID_ARG, "append: null argument");
    if (tokens < 0) return fail(c, HKV_ERR_INVALID_ARG, "append: negative tokens");
    if (tokens > c->g.max_tokens) return fail(c, HKV_ERR_TOO_LARGE, "append: more tokens than the context was created for");
    if (!aligned(k_new, 2) || !aligned(v_new, 2) || !aligned(k_cache, 2) || !aligned(v_cache, 2) || !aligned(d_slots, 4))
        return fail(c, HKV_ERR_ALIGNMENT, "append: a tensor is not aligned to its element size");
    PagedAppendArgs a{};
    a.row_elems = c->g.num_kv_heads * c->g.head_dim;
    if (!stride_ok(kv_token_stride, a.row_elems, &a.stride))
        return fail(c, HKV_ERR_INVALID_ARG, "append: kv_token_stride smaller than one token's row");
    if (tokens == 0) return HKV_OK;
    a.k = k_new;
    a.v = v_new;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.slots = d_slots;
    a.status = c->d_status;
    a.rows = (long long)c->g.num_pages * c->g.page_size;
    a.tokens = tokens;
    const bool vec = aligned(k_new, 16) && aligned(v_new, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                     a.row_elems % 8 == 0 && a.stride % 8 == 0;
    const unsigned blocks = (unsigned)std::min<long long>(((long long)tokens + 7) / 8, (long long)c->sm_count * 8);
    if (vec) hkv_paged_append_kernel<uint4><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
    else hkv_paged_append_kernel<uint16_t><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
    return launched(c, "append launch");
}

int hkv_paged_norm_rope(hkv_paged_ctx* c, const hkv_paged_rope* r, void* stream) {
    PAGED_CHECK(c);
    if (!r) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: null arguments");
    const hkv_paged_geometry& g = c->g;
    const bool cached = r->k_cache || r->v_cache;
    if (!r->q || !r->k || !r->q_out || !r->d_positions || (cached && (!r->k_cache || !r->v_cache || !r->v || !r->d_slots)) ||
        (!cached && !r->k_out))
        return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: null tensor (q, k, q_out, positions; v, slots and both planes, or k_out)");
    if (!r->q_norm_w != !r->k_norm_w) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: one norm weight without the other");
    if (r->tokens < 0) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: negative tokens");
    if (r->tokens > g.max_tokens) return fail(c, HKV_ERR_TOO_LARGE, "norm_rope: more tokens than the context was created for");
    for (const void* p : {r->q, r->k, r->v, (const void*)r->q_out, (const void*)r->k_out, r->q_norm_w, r->k_norm_w,
                          (const void*)r->k_cache, (const void*)r->v_cache})
        if (!aligned(p, 2)) return fail(c, HKV_ERR_ALIGNMENT, "norm_rope: a tensor is not 2-byte aligned");
    if (!aligned(r->d_positions, 4) || !aligned(r->d_slots, 4))
        return fail(c, HKV_ERR_ALIGNMENT, "norm_rope: an int32 array is not 4-byte aligned");
    MropeArgs a{};
    const int rot = r->rotary_dim == 0 ? g.head_dim : r->rotary_dim;
    if (rot < 0 || rot > g.head_dim || rot % 2 != 0)
        return fail(c, HKV_ERR_GEOMETRY, "norm_rope: rotary_dim must be even and at most head_dim");
    if (!(r->theta > 0.0) || !std::isfinite(r->theta) || !std::isfinite(r->scaling_factor) || !(r->eps >= 0.0f) || !std::isfinite(r->eps))
        return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: theta must be positive, eps non-negative, all finite");
    const int axes = r->axes == 0 ? 1 : r->axes;
    if (axes < 1 || axes > HKV_ROPE_MAX_AXES) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: axes outside 1..HKV_ROPE_MAX_AXES");
    if (r->interleaved != 0 && r->interleaved != 1) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: interleaved is 0 or 1");
    const int half = rot / 2;
    if (axes > 1) {
        long long sum = 0;
        for (int i = 0; i < axes; ++i) {
            if (r->sections[i] < 0) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: negative section");
            sum += r->sections[i];
        }
        if (sum != half) return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: sections must sum to rotary_dim / 2");
        int at = 0;
        for (int i = 0; i < axes; ++i) {
            if (r->interleaved) {
                // the last pair of axis i is i + axes * (sections[i] - 1)
                if (i > 0 && r->sections[i] > 0 && i + (long long)axes * (r->sections[i] - 1) >= half)
                    return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: an interleaved section reaches past rotary_dim / 2");
                if (i > 0) for (int j = 0; j < r->sections[i]; ++j) a.axis[i + axes * j] = (uint8_t)i;
            } else {
                for (int j = 0; j < r->sections[i]; ++j) a.axis[at++] = (uint8_t)i;
            }
        }
    }
    const long long qrow = (long long)g.num_heads * g.head_dim, krow = (long long)g.num_kv_heads * g.head_dim;
    if (!stride_ok(r->q_token_stride, qrow, &a.q_stride) || !stride_ok(r->q_out_token_stride, qrow, &a.qo_stride) ||
        !stride_ok(r->kv_token_stride, krow, &a.kv_stride) || !stride_ok(r->k_out_token_stride, krow, &a.ko_stride))
        return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: a token stride is smaller than one token's row");
    if ((r->q_out == r->q && a.qo_stride != a.q_stride) || (!cached && r->k_out == r->k && a.ko_stride != a.kv_stride))
        return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: in place needs the same token stride on both sides");
    if (r->position_axis_stride != 0 && r->position_axis_stride < r->tokens)
        return fail(c, HKV_ERR_INVALID_ARG, "norm_rope: position_axis_stride smaller than tokens");
    if (r->tokens == 0) return HKV_OK;
    a.q = r->q; a.k = r->k; a.v = r->v; a.q_w = r->q_norm_w; a.k_w = r->k_norm_w;
    a.q_out = r->q_out; a.k_out = r->k_out; a.k_cache = r->k_cache; a.v_cache = r->v_cache;
    a.slots = r->d_slots; a.pos = r->d_positions;
    a.status = c->d_status;
    a.axis_stride = r->position_axis_stride ? r->position_axis_stride : r->tokens;
    a.rows = (long long)g.num_pages * g.page_size;
    a.tokens = r->tokens; a.H = g.num_heads; a.KVH = g.num_kv_heads; a.HD = g.head_dim; a.rot = rot;
    a.eps = r->eps;
    const double scaling = r->scaling_factor > 0.0 ? r->scaling_factor : 1.0;
    for (int i = 0; i < half; ++i) a.turns[i] = std::pow(r->theta, -2.0 * i / rot) / (scaling * 6.283185307179586476925);
    // 16-byte pieces whose pair partner is a whole piece away; everything else goes element by element
    bool pieces = g.head_dim % 16 == 0 && rot % 16 == 0 && a.q_stride % 8 == 0 && a.kv_stride % 8 == 0 && a.qo_stride % 8 == 0 &&
                  a.ko_stride % 8 == 0;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.q_out, (const void*)a.k_out, a.q_w, a.k_w, (const void*)a.k_cache, (const void*)a.v_cache})
        pieces = pieces && aligned(p, 16);
    int lph = 4;                             // lanes per head
    while (lph * 16 < g.head_dim) lph *= 2;
    // enough warps to fill the machine: a token is shared by several, a round of heads each at least, when there are few
    const int heads = g.num_heads + (cached ? 2 : 1) * g.num_kv_heads, rounds = pieces ? (heads + 32 / lph - 1) / (32 / lph) : heads;
    a.parts = (int)std::max<long long>(1, std::min<long long>(rounds, (long long)c->sm_count * 16 / r->tokens));
    const long long units = (long long)r->tokens * a.parts;
    const unsigned blocks = (unsigned)std::min<long long>((units + kMropeWarps - 1) / kMropeWarps, (long long)c->sm_count * 8);
    const cudaStream_t st = (cudaStream_t)stream;
    if (g.dtype == HKV_DTYPE_F16) launch_rope<__half>(a, pieces ? lph : 0, blocks, st);
    else launch_rope<__nv_bfloat16>(a, pieces ? lph : 0, blocks, st);
    return launched(c, "norm_rope launch");
}

int hkv_paged_attention(hkv_paged_ctx* c, const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache,
                        void* out, const int32_t* d_block_table, const int32_t* d_q_start, const int32_t* d_step_len,
                        const int32_t* d_total_len, int32_t requests, int32_t tokens, int32_t max_step, float scale,
                        void* stream) {
    return attention(c, q, q_token_stride, k_cache, v_cache, out, d_block_table, d_q_start, d_step_len,
                     d_total_len, requests, tokens, max_step, scale, stream, true);
}

int hkv_paged_cross_attention(hkv_paged_ctx* c, const void* q, int64_t q_token_stride, const void* k_cache,
                              const void* v_cache, void* out, const int32_t* d_block_table, const int32_t* d_q_start,
                              const int32_t* d_step_len, const int32_t* d_key_len, int32_t requests, int32_t tokens,
                              int32_t max_step, float scale, void* stream) {
    return attention(c, q, q_token_stride, k_cache, v_cache, out, d_block_table, d_q_start, d_step_len,
                     d_key_len, requests, tokens, max_step, scale, stream, false);
}

}  // extern "C"
