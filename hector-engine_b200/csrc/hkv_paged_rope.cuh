// hkv_paged_rope.cuh — per-head RMSNorm + rotary embedding with several position axes for packed tokens, K and V rows
// written through a slot map (the front of the paged append path).
//
//   x_n[i] = x[i] * rsqrt(mean(x^2) + eps) * w[i]            (x[i] without weights)
//   pair i = elements (i, i + rot/2), turned by  pos[axis(i)] / scaling * theta^(-2i/rot);  dims >= rot pass through
#pragma once

#include "hkv_paged.cuh"

namespace hkv {

constexpr int kMropeThreads = 256;
constexpr int kMropeWarps = kMropeThreads / 32;
constexpr int kMropeMaxPairs = 256;    // head_dim <= 512

struct MropeArgs {
    const void *q, *k, *v, *q_w, *k_w;
    void *q_out, *k_out, *k_cache, *v_cache;
    const int32_t *slots, *pos;
    int32_t* status;
    long long q_stride, kv_stride, qo_stride, ko_stride, axis_stride;
    long long rows;                    // pages * page
    int tokens, H, KVH, HD, rot;
    int parts;                         // warps that share a token (each takes a range of its heads)
    float eps;
    // turns per unit of position of each pair, theta^(-2i/rot) / (scaling * 2 pi), and the pair's axis. In 64 bits: a
    // position of 10^6 times a 32-bit frequency is off by 0.06 radians.
    double turns[kMropeMaxPairs];
    uint8_t axis[kMropeMaxPairs];
};

// cos and sin of pair i of token t: the turn is reduced to [-1/2, 1/2] in 64 bits, the rest in 32.
__device__ __forceinline__ float2 mrope_angle(const MropeArgs& a, const double turns, const int axis, const long long t) {
    const double x = (double)a.pos[axis * a.axis_stride + t] * turns;
    float s, c;
    sincospif(2.0f * (float)(x - rint(x)), &s, &c);
    return make_float2(c, s);
}

// Element by element: any head_dim <= 512, rotary span and alignment. A warp per (token, part of its heads).
template <typename T>
__global__ void __launch_bounds__(kMropeThreads) hkv_paged_norm_rope_any_kernel(const __grid_constant__ MropeArgs a) {
    __shared__ float s_x[kMropeWarps][512];
    __shared__ float2 s_cs[kMropeWarps][kMropeMaxPairs];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.rot / 2;
    const int heads = a.H + a.KVH + (a.k_cache ? a.KVH : 0);
    const long long units = (long long)a.tokens * a.parts;
    for (long long u = blockIdx.x * (long long)kMropeWarps + warp; u < units; u += gridDim.x * (long long)kMropeWarps) {
        const long long t = u / a.parts;
        const int part = (int)(u % a.parts);
        for (int i = lane; i < half; i += 32) s_cs[warp][i] = mrope_angle(a, a.turns[i], a.axis[i], t);
        const int slot = a.k_cache ? a.slots[t] : 0;
        if (slot >= a.rows && a.k_cache && lane == 0) atomicOr(a.status, kStatusBoundCheck);
        const bool store = slot >= 0 && (!a.k_cache || slot < a.rows);
        __syncwarp();
        for (int j = (int)((long long)heads * part / a.parts); j < (int)((long long)heads * (part + 1) / a.parts); ++j) {
            const bool is_q = j < a.H, is_k = !is_q && j < a.H + a.KVH;
            const int kvh = is_k ? j - a.H : j - a.H - a.KVH;
            if (!is_q && !store) continue;
            const T* src = is_q ? (const T*)a.q + t * a.q_stride + (long long)j * a.HD
                                : (const T*)(is_k ? a.k : a.v) + t * a.kv_stride + (long long)kvh * a.HD;
            T* dst = is_q ? (T*)a.q_out + t * a.qo_stride + (long long)j * a.HD
                   : a.k_cache ? (T*)(is_k ? a.k_cache : a.v_cache) + ((long long)slot * a.KVH + kvh) * a.HD
                               : (T*)a.k_out + t * a.ko_stride + (long long)kvh * a.HD;
            if (!is_q && !is_k) {
                for (int i = lane; i < a.HD; i += 32) dst[i] = src[i];
                continue;
            }
            const T* w = (const T*)(is_q ? a.q_w : a.k_w);
            float ssq = 0.0f;
            for (int i = lane; i < a.HD; i += 32) {
                const float x = to_f32(src[i]);
                ssq = fmaf(x, x, ssq);
                s_x[warp][i] = w ? x * to_f32(w[i]) : x;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
            const float inv = w ? 1.0f / sqrtf(ssq / (float)a.HD + a.eps) : 1.0f;
            __syncwarp();
            const float* x = s_x[warp];
            for (int i = lane; i < a.HD; i += 32) {
                float r = x[i];
                if (i < half) r = x[i] * s_cs[warp][i].x - x[i + half] * s_cs[warp][i].y;
                else if (i < a.rot) r = x[i - half] * s_cs[warp][i - half].y + x[i] * s_cs[warp][i - half].x;
                dst[i] = from_f32<T>(r * inv);
            }
            __syncwarp();
        }
        __syncwarp();
    }
}

// The register path (host: rows 16-byte aligned, head_dim and rotary_dim multiples of 16).
//
// Bound: HBM for prompts (each row read once, written once); latency for a decode step. A warp works on one token at a
// time, or on a part of its heads when there are few tokens, and needs nothing from other warps: no block barrier.
//   * LPH lanes hold a head, each a 16-byte piece of the first half of the rotated span and the piece rotary_dim/2 behind
//     it, so that both elements of a pair sit in one lane (lanes past rotary_dim/16 hold two pieces that pass through):
//     8 lanes for head_dim 128, four heads per warp and round.
//   * cos and sin of a token's pairs are computed once, two pairs per lane at head_dim 128, and shared through the warp's
//     table in shared memory: 64-bit turns reduced to [-1/2, 1/2], then sincospi in 32 bits.
//   * U rounds' loads are issued together, in front of the angles.
constexpr int kMropeRounds = 4;

template <typename T, int LPH>
__global__ void __launch_bounds__(kMropeThreads) hkv_paged_norm_rope_kernel(const __grid_constant__ MropeArgs a) {
    constexpr int HPW = 32 / LPH;                      // heads per warp and round
    constexpr int U = kMropeRounds;
    __shared__ float2 s_cs[kMropeWarps][LPH * 8];      // pairs of one token: rot/2 <= LPH * 8
    __shared__ double s_turns[LPH * 8];
    __shared__ uint8_t s_axis[LPH * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.rot / 2;
    const int sub = lane / LPH, p = lane % LPH;
    const int heads = a.H + a.KVH + (a.k_cache ? a.KVH : 0);
    for (int i = threadIdx.x; i < half; i += kMropeThreads) { s_turns[i] = a.turns[i]; s_axis[i] = a.axis[i]; }
    const bool live = 16 * p < a.HD, turns = 16 * p < a.rot;
    // elements of this lane's two pieces
    const int e0 = turns ? 8 * p : 16 * p, e1 = turns ? half + 8 * p : 16 * p + 8;
    const float inv_hd = 1.0f / (float)a.HD;
    __syncthreads();
    const long long units = (long long)a.tokens * a.parts;
    for (long long unit = blockIdx.x * (long long)kMropeWarps + warp; unit < units; unit += gridDim.x * (long long)kMropeWarps) {
        const long long t = unit / a.parts;
        const int part = (int)(unit - t * a.parts);
        // this unit's heads, in whole rounds
        const int rounds = (heads + HPW - 1) / HPW;
        const int j0 = rounds * part / a.parts * HPW, j1 = rounds * (part + 1) / a.parts * HPW;
        const T* qt = (const T*)a.q + t * a.q_stride;
        const T* kt = (const T*)a.k + t * a.kv_stride;
        const T* vt = (const T*)a.v + t * a.kv_stride;
        const int slot = a.k_cache ? a.slots[t] : 0;
        uint4 x0[U], x1[U];
        auto load = [&](int jb) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = jb + u * HPW + sub;
                x0[u] = x1[u] = make_uint4(0, 0, 0, 0);
                if (live && j < j1 && j < heads) {
                    const T* src = j < a.H ? qt + (long long)j * a.HD
                                 : j < a.H + a.KVH ? kt + (long long)(j - a.H) * a.HD : vt + (long long)(j - a.H - a.KVH) * a.HD;
                    x0[u] = *reinterpret_cast<const uint4*>(src + e0);
                    x1[u] = *reinterpret_cast<const uint4*>(src + e1);
                }
            }
        };
        load(j0);
        for (int i = lane; i < half; i += 32) s_cs[warp][i] = mrope_angle(a, s_turns[i], s_axis[i], t);
        const bool store = slot >= 0 && (!a.k_cache || slot < a.rows);
        if (a.k_cache && slot >= a.rows && lane == 0) atomicOr(a.status, kStatusBoundCheck);
        __syncwarp();
        float c[8], s[8];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float4 w = turns ? *reinterpret_cast<const float4*>(&s_cs[warp][8 * p + e]) : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
            c[e] = w.x; s[e] = w.y; c[e + 1] = w.z; s[e + 1] = w.w;
        }
        for (int jb = j0; jb < j1; jb += U * HPW) {
            if (jb != j0) load(jb);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = jb + u * HPW + sub;
                if (jb + u * HPW >= j1) break;         // warp-uniform
                const bool is_q = j < a.H, is_v = j >= a.H + a.KVH;
                float x[8], y[8];
                const uint32_t w0[4] = {x0[u].x, x0[u].y, x0[u].z, x0[u].w}, w1[4] = {x1[u].x, x1[u].y, x1[u].z, x1[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack2<T>(w0[e]), g = unpack2<T>(w1[e]);
                    x[2 * e] = f.x; x[2 * e + 1] = f.y;
                    y[2 * e] = g.x; y[2 * e + 1] = g.y;
                }
                if (a.q_w) {
                    float ssq = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ssq = fmaf(x[e], x[e], fmaf(y[e], y[e], ssq));
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
                    const float inv = rsqrtf(fmaf(ssq, inv_hd, a.eps));
                    const T* w = (const T*)(is_q ? a.q_w : a.k_w);
                    if (live) {
                        const uint4 a0 = *reinterpret_cast<const uint4*>(w + e0), a1 = *reinterpret_cast<const uint4*>(w + e1);
                        const uint32_t u0[4] = {a0.x, a0.y, a0.z, a0.w}, u1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = unpack2<T>(u0[e]), g = unpack2<T>(u1[e]);
                            x[2 * e] *= inv * f.x; x[2 * e + 1] *= inv * f.y;
                            y[2 * e] *= inv * g.x; y[2 * e + 1] *= inv * g.y;
                        }
                    }
                }
                uint32_t r0[4], r1[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    r0[e] = pack2<T>(x[2 * e] * c[2 * e] - y[2 * e] * s[2 * e], x[2 * e + 1] * c[2 * e + 1] - y[2 * e + 1] * s[2 * e + 1]);
                    r1[e] = pack2<T>(x[2 * e] * s[2 * e] + y[2 * e] * c[2 * e], x[2 * e + 1] * s[2 * e + 1] + y[2 * e + 1] * c[2 * e + 1]);
                }
                if (!live || j >= heads || (!is_q && !store)) continue;
                T* dst = is_q ? (T*)a.q_out + t * a.qo_stride + (long long)j * a.HD
                       : is_v ? (T*)a.v_cache + ((long long)slot * a.KVH + (j - a.H - a.KVH)) * a.HD
                       : a.k_cache ? (T*)a.k_cache + ((long long)slot * a.KVH + (j - a.H)) * a.HD
                                   : (T*)a.k_out + t * a.ko_stride + (long long)(j - a.H) * a.HD;
                *reinterpret_cast<uint4*>(dst + e0) = is_v ? x0[u] : make_uint4(r0[0], r0[1], r0[2], r0[3]);
                *reinterpret_cast<uint4*>(dst + e1) = is_v ? x1[u] : make_uint4(r1[0], r1[1], r1[2], r1[3]);
            }
        }
        __syncwarp();                                  // the table is read before the next token's is written
    }
}

}  // namespace hkv
