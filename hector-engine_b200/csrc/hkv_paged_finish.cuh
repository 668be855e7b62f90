// hkv_paged_finish.cuh — the second launch of paged attention: joins the partial rows of what the staged kernels had to cut,
//     o = sum 2^(m_c - M) o_c / sum 2^(m_c - M) l_c,   M = max m_c,
// and does again what they left on the list of items with hidden values that are not finite. Blocks of 256 threads:
// first those of the few-token kernel (a block per span, KV head and query row: few rows, up to hundreds of parts, so
// eight warps deal the parts of a row among them), then those of the prompt kernel (many rows of mostly two parts). It is launched while the kernel before it still runs and waits for its end on
// the GPU. Bound: launch latency; the partial rows (39 MB at most) come out of the L2:
// 4 us for a few-token call, 10 to 16 us where every CTA of a prompt launch cut an item.
#pragma once

#include "hkv_paged_chunk.cuh"

namespace hkv {

struct PagedFinishArgs {
    PagedAttnArgs t;
    PagedFix fix;
    const float* small_part;      // [2 * spans][KVH][cols][HD + 2]
    const int4* small_cuts;       // [spans]
    const float* chunk_part;      // [2 * ctas] sets of tiles * 128 rows
    const int4* chunk_cuts;       // [ctas]
    int spans, cols;              // spans 0: no few-token launch
    int ctas, tiles, QT, QB;      // ctas 0: no prompt launch
    int may_fix;                  // 0: a single query per request, nothing can be on the list
};
// (blocks of 32 rows behind those of the few-token kernel)
__host__ __device__ inline int finish_parts(int HD) { return HD > 128 ? 2 : 1; }     // blocks per 32 rows: 128 columns each
__host__ __device__ inline int finish_blocks(const PagedFinishArgs& a, int KVH) { return a.spans * KVH * a.cols + a.ctas * a.tiles * 4 * finish_parts(a.t.HD); }

template <typename T>
__device__ __forceinline__ void finish_small(const PagedFinishArgs& a, const int block, const int fix_count) {
    const int c = block % a.cols, kvh = block / a.cols % a.t.KVH, span = block / (a.cols * a.t.KVH);
    const int4 cut = a.small_cuts[span];
    const int G = a.t.H / a.t.KVH, HD = a.t.HD, parts = cut.y;
    if (parts <= 1 || c >= cut.w * G) return;
    if (fix_count && paged_to_fix(a.fix, fix_count, cut.x, -1, kvh)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ float s_o[8][256];
    __shared__ float s_m[8], s_l[8];
    float M = kLow, L = 0.0f;
    float2 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = make_float2(0.0f, 0.0f);
    for (int p0 = warp; p0 < parts; p0 += 16) {
        float2 ml[2], x[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // part 0 sits in this span's second slot, the others in the first slots of the spans behind it
            const int p = p0 + 8 * u, slot = 2 * (span + p) + (p == 0 ? 1 : 0);
            const float* row = a.small_part + (((long long)slot * a.t.KVH + kvh) * a.cols + c) * (HD + 2);
            ml[u] = p < parts ? *reinterpret_cast<const float2*>(row + HD) : make_float2(kLow, 0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 2 * lane + 64 * i;
                x[u][i] = p < parts && d < HD ? *reinterpret_cast<const float2*>(row + d) : make_float2(0.0f, 0.0f);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float Mn = fmaxf(M, ml[u].x), keep = exp2f(M - Mn), w = exp2f(ml[u].x - Mn);
            L = fmaf(ml[u].y, w, L * keep);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i].x = fmaf(x[u][i].x, w, acc[i].x * keep);
                acc[i].y = fmaf(x[u][i].y, w, acc[i].y * keep);
            }
            M = Mn;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 2 * lane + 64 * i;
        if (d < HD) *reinterpret_cast<float2*>(&s_o[warp][d]) = acc[i];
    }
    if (lane == 0) { s_m[warp] = M; s_l[warp] = L; }
    __syncthreads();
    float Mx = s_m[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) Mx = fmaxf(Mx, s_m[w]);
    float f[8], Lx = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        f[w] = exp2f(s_m[w] - Mx);
        Lx = fmaf(s_l[w], f[w], Lx);
    }
    const float inv = Lx > 0.0f ? 1.0f / Lx : 0.0f;
    T* op = (T*)a.t.out + ((long long)(cut.z + c / G) * a.t.H + (long long)kvh * G + c % G) * HD;
    for (int d = threadIdx.x; d < HD; d += 256) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) o = fmaf(s_o[w][d], f[w], o);
        op[d] = from_f32<T>(o * inv);
    }
}

// 32 rows and 128 columns per block (80 registers, three blocks per SM; with whole rows of head_dim 256 two blocks, and calls that cut
// much took 2 to 5 us longer). A warp takes 8 rows and every eighth group of 4 x 4 columns, so that it reads whole lines of
// a set and writes whole sectors of a row; the loads of two parts are in flight together, nothing in front of them but the entry.
template <typename T>
__device__ __forceinline__ void finish_chunk(const PagedFinishArgs& a, const int block, const int fix_count) {
    const int rows = a.tiles * 128, wide = finish_parts(a.t.HD), shares = rows / 32 * wide;
    const int cta = block / shares, share = block % shares / wide;
    const int4 cut = a.chunk_cuts[cta];
    const int parts = cut.w;
    if (parts <= 1) return;
    if (fix_count && paged_to_fix(a.fix, fix_count, cut.x, cut.z, cut.y)) return;
    const int G = a.t.H / a.t.KVH, HD = a.t.HD, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cols = HD < 128 ? HD : 128;
    const int row = share * 32 + (warp & 3) * 8 + (lane & 7), cb = block % wide * 32 + (warp >> 2) * 4 + (lane >> 3);
    const int ql = row % 128 / G, i = cut.z * a.QB + row / 128 * a.QT + ql;
    const PagedRequest q = paged_request(a.t.b, cut.x);
    if (ql >= a.QT || i >= q.n) return;
    const long long set = partial_floats(rows, HD);
    // part 0 sits in this CTA's second slot, the others in the first slots of the CTAs behind it
    const float* base = a.chunk_part + 2ll * cta * set;
    float M = kLow, L = 0.0f;
    float4 acc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p0 = 0; p0 < parts; p0 += 2) {
        float2 ml[2];
        float4 x[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int p = p0 + u;
            const float* s = base + (2ll * p + (p == 0 ? 1 : 0)) * set;
            ml[u] = p < parts ? *reinterpret_cast<const float2*>(s + (long long)rows * HD + 2 * row) : make_float2(kLow, 0.0f);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[u][e] = p < parts && 32 * e < cols ? *reinterpret_cast<const float4*>(s + ((long long)(cb + 8 * e) * rows + row) * 4)
                                                   : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float Mn = fmaxf(M, ml[u].x), keep = exp2f(M - Mn), w = exp2f(ml[u].x - Mn);
            L = fmaf(ml[u].y, w, L * keep);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e].x = fmaf(x[u][e].x, w, acc[e].x * keep); acc[e].y = fmaf(x[u][e].y, w, acc[e].y * keep);
                acc[e].z = fmaf(x[u][e].z, w, acc[e].z * keep); acc[e].w = fmaf(x[u][e].w, w, acc[e].w * keep);
            }
            M = Mn;
        }
    }
    const float inv = L == 0.0f ? 0.0f : (L < kSumLimit ? 1.0f / L : NAN);
    T* op = (T*)a.t.out + ((long long)(q.start + i) * a.t.H + (long long)cut.y * G + row % 128 % G) * HD + 4 * cb;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (32 * e < cols) *reinterpret_cast<uint2*>(op + 32 * e) = make_uint2(pack2<T>(acc[e].x * inv, acc[e].y * inv), pack2<T>(acc[e].z * inv, acc[e].w * inv));
}

template <typename T>
__global__ void __launch_bounds__(256, 3) hkv_paged_finish_kernel(const __grid_constant__ PagedFinishArgs a) {
    wait_for_previous();
    const int count = a.may_fix ? *reinterpret_cast<volatile int*>(a.fix.head) : 0;
    const int small = a.spans * a.t.KVH * a.cols;
    if ((int)blockIdx.x < small) finish_small<T>(a, blockIdx.x, count);
    else finish_chunk<T>(a, blockIdx.x - small, count);
    if (count > 0) {
        __syncthreads();
        paged_fix_rows<T, 8>(a.t, a.fix, count, a.QB);
    }
}

}  // namespace hkv
