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

// Two 32-bit values in one 64-bit register: sm_100 multiplies and adds them in one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack_f2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack_f2(f32x2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <typename T>
__device__ __forceinline__ f32x2 widen2(uint32_t w) {
    const float2 f = unpack2<T>(w);
    return pack_f2(f.x, f.y);
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
//   * The norm weights are folded into them, per token and kind of head: with x, y the halves of a pair,
//         x' = inv (x A + y B)   y' = inv (x C + y D)    A = w_x cos   B = -w_y sin   C = w_x sin   D = w_y cos
//     so that an element costs three packed instructions of two elements each beside its conversions. (Unfolded and
//     unpacked the kernel was bound by instruction issue: 245 instructions a round, 40 us for 8 192 tokens.)
//   * U rounds' loads are issued together, in front of the angles.
constexpr int kMropeRounds = 4;

template <typename T, int LPH>
__global__ void __launch_bounds__(kMropeThreads, 2) hkv_paged_norm_rope_kernel(const __grid_constant__ MropeArgs a) {
    constexpr int HPW = 32 / LPH;                      // heads per warp and round
    constexpr int U = kMropeRounds;
    __shared__ float2 s_cs[kMropeWarps][LPH * 8];      // pairs of one token: rot/2 <= LPH * 8
    __shared__ double s_turns[LPH * 8];
    __shared__ uint8_t s_axis[LPH * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.rot / 2;
    const int sub = lane / LPH, p = lane % LPH;
    const int heads = a.H + a.KVH + (a.k_cache ? a.KVH : 0), HK = a.H + a.KVH;
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
                    const T* src = j < a.H ? qt + j * a.HD : j < HK ? kt + (j - a.H) * a.HD : vt + (j - HK) * a.HD;
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
        f32x2 A[4], B[4], C[4], D[4];                  // of this lane's 8 pairs, for the kind of head it is at
        int kind = -1;                                 // 0 query, 1 key, 2 value (copied)
        // rows of this token that are written: query rows, and key / value rows in the planes or in k_out
        T* const q_row = (T*)a.q_out + t * a.qo_stride;
        T* const k_row = a.k_cache ? (T*)a.k_cache + (long long)slot * a.KVH * a.HD : (T*)a.k_out + t * a.ko_stride;
        T* const v_row = (T*)a.v_cache + (long long)slot * a.KVH * a.HD;
        for (int jb = j0; jb < j1; jb += U * HPW) {
            if (jb != j0) load(jb);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = jb + u * HPW + sub;
                if (jb + u * HPW >= j1) break;         // warp-uniform
                const int is = j < a.H ? 0 : j < HK ? 1 : 2;
                if (is != kind && is < 2) {
                    const T* w = (const T*)(is == 0 ? a.q_w : a.k_w);
                    uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
                    if (w && live) { w0 = *reinterpret_cast<const uint4*>(w + e0); w1 = *reinterpret_cast<const uint4*>(w + e1); }
                    const uint32_t v0[4] = {w0.x, w0.y, w0.z, w0.w}, v1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 cs = turns ? *reinterpret_cast<const float4*>(&s_cs[warp][8 * p + 2 * e]) : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
                        const f32x2 c = pack_f2(cs.x, cs.z), s = pack_f2(cs.y, cs.w), n = pack_f2(-cs.y, -cs.w);
                        const f32x2 wx = w ? widen2<T>(v0[e]) : pack_f2(1.0f, 1.0f), wy = w ? widen2<T>(v1[e]) : pack_f2(1.0f, 1.0f);
                        A[e] = mul2(wx, c); B[e] = mul2(wy, n); C[e] = mul2(wx, s); D[e] = mul2(wy, c);
                    }
                }
                kind = is;
                uint32_t r0[4] = {x0[u].x, x0[u].y, x0[u].z, x0[u].w}, r1[4] = {x1[u].x, x1[u].y, x1[u].z, x1[u].w};
                f32x2 x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) { x[e] = widen2<T>(r0[e]); y[e] = widen2<T>(r1[e]); }
                float inv = 1.0f;
                if (a.q_w) {
                    f32x2 q = mul2(x[0], x[0]);
#pragma unroll
                    for (int e = 1; e < 4; ++e) q = fma2(x[e], x[e], q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) q = fma2(y[e], y[e], q);
                    const float2 h = unpack_f2(q);
                    float ssq = h.x + h.y;
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
                    inv = rsqrtf(fmaf(ssq, inv_hd, a.eps));
                }
                if (!live || j >= heads || (is > 0 && !store)) continue;
                if (is < 2) {
                    const f32x2 i2 = pack_f2(inv, inv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = unpack_f2(mul2(i2, fma2(x[e], A[e], mul2(y[e], B[e]))));
                        const float2 g = unpack_f2(mul2(i2, fma2(x[e], C[e], mul2(y[e], D[e]))));
                        r0[e] = pack2<T>(f.x, f.y);
                        r1[e] = pack2<T>(g.x, g.y);
                    }
                }
                T* dst = is == 0 ? q_row + j * a.HD : is == 1 ? k_row + (j - a.H) * a.HD : v_row + (j - HK) * a.HD;
                *reinterpret_cast<uint4*>(dst + e0) = make_uint4(r0[0], r0[1], r0[2], r0[3]);
                *reinterpret_cast<uint4*>(dst + e1) = make_uint4(r1[0], r1[1], r1[2], r1[3]);
            }
        }
        __syncwarp();                                  // the table is read before the next token's is written
    }
}

}  // namespace hkv
