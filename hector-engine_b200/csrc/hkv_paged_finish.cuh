// hkv_paged_finish.cuh — the second launch of paged attention: joins the partial rows of what the staged kernels had to cut,
//     o = sum 2^(m_c - M) o_c / sum 2^(m_c - M) l_c,   M = max m_c,
// and does again what they left on the list of items with hidden values that are not finite. Blocks of 256 threads:
// first those of the few-token kernel (a block per span, KV head and query row: few rows, up to hundreds of parts, so
// eight warps deal the parts of a row among them), then those of the prompt kernel (eight per CTA of that launch: many
// rows of mostly two parts, a warp each). It is launched while the kernel before it still runs and waits for its end on
// the GPU. Bound: launch latency; the partial rows (39 MB at most) come out of the L2.
#pragma once

#include "hkv_paged.cuh"

namespace hkv {

struct PagedFinishArgs {
    PagedAttnArgs t;
    PagedFix fix;
    const float* small_part;      // [2 * spans][KVH][cols][HD + 2]
    const int4* small_cuts;       // [spans]
    const float* chunk_part;      // [2 * ctas][tiles * 128][HD + 4]
    const int4* chunk_cuts;       // [ctas]
    int spans, cols;              // spans 0: no few-token launch
    int ctas, tiles, QT, QB;      // ctas 0: no prompt launch
    int may_fix;                  // 0: a single query per request, nothing can be on the list
};
constexpr int kFinishPerCta = 8;  // blocks per CTA of the prompt launch
__host__ __device__ inline int finish_blocks(const PagedFinishArgs& a, int KVH) { return a.spans * KVH * a.cols + a.ctas * kFinishPerCta; }

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

template <typename T>
__device__ __forceinline__ void finish_chunk(const PagedFinishArgs& a, const int block, const int fix_count) {
    const int cta = block / kFinishPerCta, share = block % kFinishPerCta;
    const int4 cut = a.chunk_cuts[cta];
    const int parts = cut.w;
    if (parts <= 1) return;
    if (fix_count && paged_to_fix(a.fix, fix_count, cut.x, cut.z, cut.y)) return;
    const PagedRequest q = paged_request(a.t.b, cut.x);
    const int G = a.t.H / a.t.KVH, HD = a.t.HD, PW = HD + 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long set = (long long)a.tiles * 128 * PW;
    // part 0 sits in this CTA's second slot, the others in the first slots of the CTAs behind it
    const float* first = a.chunk_part + (2ll * cta + 1) * set;
    const float* rest = a.chunk_part + 2ll * (cta + 1) * set;
    for (int row = share * 8 + warp; row < a.tiles * 128; row += kFinishPerCta * 8) {
        const int ql = row % 128 / G, i = cut.z * a.QB + row / 128 * a.QT + ql;
        if (ql >= a.QT || i >= q.n) continue;
        auto at = [&](int p) { return (p == 0 ? first : rest + 2ll * (p - 1) * set) + (long long)row * PW; };
        // maxima and sums of up to 32 parts at a time, one per lane; then the rows, four floats per lane
        float M = kLow, L = 0.0f;
        float4 acc[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
        for (int p0 = 0; p0 < parts; p0 += 32) {
            const int n = parts - p0 < 32 ? parts - p0 : 32;
            const float2 ml = lane < n ? *reinterpret_cast<const float2*>(at(p0 + lane) + HD) : make_float2(kLow, 0.0f);
            float Mn = ml.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, o));
            Mn = fmaxf(Mn, M);
            const float keep = exp2f(M - Mn), w = lane < n ? exp2f(ml.x - Mn) : 0.0f;
            float l = ml.y * w;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            L = fmaf(L, keep, l);
#pragma unroll
            for (int e = 0; e < 2; ++e) { acc[e].x *= keep; acc[e].y *= keep; acc[e].z *= keep; acc[e].w *= keep; }
#pragma unroll 4
            for (int p = 0; p < n; ++p) {
                const float wp = __shfl_sync(0xffffffffu, w, p);
                const float* r = at(p0 + p);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 4 * lane + 128 * e;
                    if (d < HD) {
                        const float4 x = *reinterpret_cast<const float4*>(r + d);
                        acc[e].x = fmaf(x.x, wp, acc[e].x); acc[e].y = fmaf(x.y, wp, acc[e].y);
                        acc[e].z = fmaf(x.z, wp, acc[e].z); acc[e].w = fmaf(x.w, wp, acc[e].w);
                    }
                }
            }
            M = Mn;
        }
        const float inv = L == 0.0f ? 0.0f : (L < kSumLimit ? 1.0f / L : NAN);
        T* op = (T*)a.t.out + ((long long)(q.start + i) * a.t.H + (long long)cut.y * G + row % 128 % G) * HD;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 4 * lane + 128 * e;
            if (d < HD) *reinterpret_cast<uint2*>(op + d) = make_uint2(pack2<T>(acc[e].x * inv, acc[e].y * inv), pack2<T>(acc[e].z * inv, acc[e].w * inv));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) hkv_paged_finish_kernel(const __grid_constant__ PagedFinishArgs a) {
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
