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

}  // namespace hkv
