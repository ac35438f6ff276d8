// KV cache in 4 bits: writing it (with rotation and per-head norm) and reading it back.  Attention over it: kv4_attend.cuh.
//
// A group is 64 neighbouring channels of one slot of one KV head: x = (c - z) * s, codes c in 0..15, from the group's minimum and
// maximum: s = bf16((max - min) / 15), z = fp16(-min / s), c = clamp(rint(x / s + z), 0, 15).  bf16 inputs keep |z| below 2^13 (max - min is at
// least one of their steps); a constant group takes s = bf16(|min| / 256), so that it reads as itself.  A group with a value that is
// not finite, or whose range leaves fp32, reads as NaN.
//
// A tile is 32 slots of one KV head in one piece of 36 * D bytes (G = D / 64), which one bulk copy brings into shared memory:
//   K codes  [G][32 slots][32 B]                            channel 2b in the low half of byte b
//   V codes  [G][16 slot pairs][8 chunks][2 slots][4 B]     chunk = 8 channels; chunk g of pair p at place g ^ ((p & 2) << 1)
//   K        [32 slots][G] { fp16 zero, bf16 scale }
//   V scale  [32 slots][G] bf16,  V zero [G][32 slots] fp16
// Attention wants values of two slots side by side as a tensor-core operand, hence the pairs of V; the places of the chunks keep its
// shared-memory reads free of bank conflicts.
#pragma once
#include <cuda_fp16.h>
#include <type_traits>
#include "common.cuh"
#include "staged_input.cuh"

namespace cb {

constexpr int KV4_GROUP = 64;
constexpr int KV4_TILE = 32;                                           // slots
constexpr int KV4_MAX_GROUPS = 4;
constexpr int KV4_THREADS = 256;

__host__ __device__ constexpr int kv4_tile_bytes(int G) { return 36 * 64 * G; }
__device__ __forceinline__ int kv4_k_row(int G, int g, int slot) { return g * 1024 + slot * 32; }
__device__ __forceinline__ int kv4_v_chunk(int G, int g, int slot, int chunk) {
    const int pair = slot >> 1;
    return 1024 * G + g * 1024 + pair * 64 + ((chunk ^ ((pair & 2) << 1)) << 3) + ((slot & 1) << 2);
}
__device__ __forceinline__ int kv4_k_meta(int G, int g, int slot) { return 2048 * G + (slot * G + g) * 4; }
__device__ __forceinline__ int kv4_v_scale(int G, int g, int slot) { return 2176 * G + (slot * G + g) * 2; }
__device__ __forceinline__ int kv4_v_zero(int G, int g, int slot) { return 2240 * G + (g * KV4_TILE + slot) * 2; }

__device__ uint32_t g_kv4_status;                                      // first bounded wait that gave up, on this device

struct Kv4Cache {
    uint8_t* tiles;
    long long seq_stride;                                              // bytes
    int n_kv, n_tiles, n_slots;
    __device__ __forceinline__ uint8_t* tile(int seq, int kvh, int slot, int G) const {
        return tiles + (long long)seq * seq_stride + ((long long)kvh * n_tiles + slot / KV4_TILE) * kv4_tile_bytes(G);
    }
};

// monotone map of fp32 to signed integers (its own inverse)
__device__ __forceinline__ int ordered_int(float f) {
    const int b = __float_as_int(f);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float ordered_float(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7FFFFFFF)); }

// ----------------------------------------------------------------------------- writing
struct Kv4AppendParams {
    const uint16_t *k, *v, *q;                                         // q may be null
    uint16_t* q_out;
    long long ld_k, ld_v, ld_q, ld_qo;                                 // elements from row to row
    const long long* positions;
    long long pos_stride;                                              // from sequence to sequence (0: the same positions)
    Kv4Cache cache;
    int T, n_heads;
    const float* inv_freq;                                             // may be null: no rotation
    const uint16_t *q_norm, *k_norm;                                   // may be null
    float eps;
};

// Codes, scale and zero of one group held by a warp (lane l: channels 2l and 2l + 1).
__device__ __forceinline__ void kv4_quantise(float a, float b, uint32_t& byte, uint16_t& scale, uint16_t& zero) {
    const uint32_t full = 0xFFFFFFFFu;
    const int ka = ordered_int(a), kb = ordered_int(b);
    const float lo = ordered_float(__reduce_min_sync(full, min(ka, kb))), hi = ordered_float(__reduce_max_sync(full, max(ka, kb)));
    float s = bf16_round(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    // a NaN is above or below everything as an integer, so it is one of the two bounds; so is an infinity
    if (!(fabsf(s) < INFINITY)) {
        byte = 0u; scale = 0x7FC0u; zero = 0u;
        return;
    }
    if (s == 0.0f) s = bf16_round(__fmul_rn(fabsf(lo), 0.00390625f));
    const bool empty = s == 0.0f;                                      // all zero
    const __half z = __float2half_rn(empty ? 0.0f : __fdiv_rn(-lo, s));
    const float zf = __half2float(z);
    auto code = [&](float x) {
        return empty ? 0u : (uint32_t)fminf(fmaxf(rintf(__fadd_rn(__fdiv_rn(x, s), zf)), 0.0f), 15.0f);
    };
    byte = code(a) | code(b) << 4;
    scale = (uint16_t)(__float_as_uint(s) >> 16);
    zero = __half_as_ushort(z);
}

// One block per row (token of a sequence) and share of the heads: a warp takes whole heads, lane l holds channels 2l, 2l + 1 of every
// group.  The cosines and sines of the position are the same for every head and computed once per block.
template <int G>
__global__ void __launch_bounds__(KV4_THREADS) kv4_append_kernel(const Kv4AppendParams P) {
    constexpr int D = 64 * G, HALF = D / 2;
    __shared__ float cs[HALF], sn[HALF];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.x, seq = row / P.T, t = row - seq * P.T;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long pos = P.positions[seq * P.pos_stride + t];
    const bool stored = pos >= 0 && pos < P.cache.n_slots;              // a position outside the cache is never stored
    if (P.inv_freq) {
        for (int d = threadIdx.x; d < HALF; d += KV4_THREADS) {
            const float ang = (float)pos * P.inv_freq[d];
            cs[d] = bf16_round(cosf(ang));
            sn[d] = bf16_round(sinf(ang));
        }
        __syncthreads();
    }
    const int n_kv = P.cache.n_kv, items = 2 * n_kv + (P.q ? P.n_heads : 0);
    for (int item = blockIdx.y * (KV4_THREADS / 32) + warp; item < items; item += gridDim.y * (KV4_THREADS / 32)) {
        const int kind = item < n_kv ? 0 : item < 2 * n_kv ? 1 : 2;     // key, value, query
        const int head = item - kind * n_kv;
        if (kind < 2 && !stored) continue;
        const uint16_t* src = (kind == 0 ? P.k + row * P.ld_k : kind == 1 ? P.v + row * P.ld_v : P.q + row * P.ld_q) + head * D;
        float x[G][2];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(src + 64 * g + 2 * lane);
            x[g][0] = __uint_as_float(w << 16);
            x[g][1] = __uint_as_float(w & 0xFFFF0000u);
        }
        const uint16_t* nw = kind == 0 ? P.k_norm : kind == 2 ? P.q_norm : nullptr;
        if (nw) {                                                      // x' = bf16( x * rsqrt(mean(x^2) + eps) * (1 + w) )
            float ss = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) ss += x[g][0] * x[g][0] + x[g][1] * x[g][1];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
            const float r = rsqrtf(ss / (float)D + P.eps);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(nw + 64 * g + 2 * lane);
                x[g][0] = bf16_round(__fmul_rn(__fmul_rn(x[g][0], r), __fadd_rn(1.0f, __uint_as_float(w << 16))));
                x[g][1] = bf16_round(__fmul_rn(__fmul_rn(x[g][1], r), __fadd_rn(1.0f, __uint_as_float(w & 0xFFFF0000u))));
            }
        }
        if (P.inv_freq && kind != 1) {
            float y[G][2];                                             // the other half's channel of each of mine
            if (G % 2 == 0) {
#pragma unroll
                for (int g = 0; g < G; ++g) { y[g][0] = x[(g + G / 2) % G][0]; y[g][1] = x[(g + G / 2) % G][1]; }
            } else {
                float o[G][2];
#pragma unroll
                for (int g = 0; g < G; ++g)
                    for (int e = 0; e < 2; ++e) o[g][e] = __shfl_xor_sync(0xFFFFFFFFu, x[g][e], 16);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int d = 64 * g + 2 * lane, pg = (d < HALF ? d + HALF : d - HALF) >> 6;
#pragma unroll
                    for (int j = 0; j < G; ++j)
                        if (j == pg) { y[g][0] = o[j][0]; y[g][1] = o[j][1]; }
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 64 * g + 2 * lane + e;
                    const float c = cs[d < HALF ? d : d - HALF], s = sn[d < HALF ? d : d - HALF];
                    x[g][e] = bf16_round(bf16_round(x[g][e] * c) + bf16_round((d < HALF ? -y[g][e] : y[g][e]) * s));
                }
        }
        if (kind == 2) {
            uint16_t* dst = P.q_out + row * P.ld_qo + head * D;
#pragma unroll
            for (int g = 0; g < G; ++g) *reinterpret_cast<uint32_t*>(dst + 64 * g + 2 * lane) = pack_bf16x2(x[g][0], x[g][1]);
            continue;
        }
        uint8_t* tile = P.cache.tile(seq, head, (int)pos, G);
        const int slot = (int)pos % KV4_TILE;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t byte;
            uint16_t scale, zero;
            kv4_quantise(x[g][0], x[g][1], byte, scale, zero);
            if (kind == 0) {
                tile[kv4_k_row(G, g, slot) + lane] = (uint8_t)byte;
                if (lane == 0) *reinterpret_cast<uint32_t*>(tile + kv4_k_meta(G, g, slot)) = (uint32_t)zero | (uint32_t)scale << 16;
            } else {
                tile[kv4_v_chunk(G, g, slot, lane >> 2) + (lane & 3)] = (uint8_t)byte;
                if (lane == 0) *reinterpret_cast<uint16_t*>(tile + kv4_v_scale(G, g, slot)) = scale;
                if (lane == 1) *reinterpret_cast<uint16_t*>(tile + kv4_v_zero(G, g, slot)) = zero;
            }
        }
    }
}

// ----------------------------------------------------------------------------- reading back
// the two channels (2l, 2l + 1) of group g that lane l of a warp holds
__device__ __forceinline__ float2 kv4_pair(uint32_t byte, uint32_t scale, uint32_t zero) {
    const float s = __uint_as_float(scale << 16), z = __half2float(__ushort_as_half((uint16_t)zero));
    return make_float2(((float)(byte & 15u) - z) * s, ((float)(byte >> 4) - z) * s);
}
__device__ __forceinline__ float2 kv4_key(const uint8_t* tile, int G, int g, int slot, int lane) {
    const uint32_t m = *reinterpret_cast<const uint32_t*>(tile + kv4_k_meta(G, g, slot));
    return kv4_pair(tile[kv4_k_row(G, g, slot) + lane], m >> 16, m & 0xFFFFu);
}
__device__ __forceinline__ float2 kv4_value(const uint8_t* tile, int G, int g, int slot, int lane) {
    return kv4_pair(tile[kv4_v_chunk(G, g, slot, lane >> 2) + (lane & 3)], *reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, g, slot)),
                    *reinterpret_cast<const uint16_t*>(tile + kv4_v_zero(G, g, slot)));
}

// k, v [rows][n_kv][D] bf16 of the slots at positions; a position outside the cache reads as zeros.  One warp per row and head.
template <int G>
__global__ void __launch_bounds__(KV4_THREADS) kv4_read_kernel(const Kv4Cache C, const long long* positions, long long pos_stride, int T,
                                                               long long items, uint16_t* k, uint16_t* v) {
    constexpr int D = 64 * G;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long item = (long long)blockIdx.x * (KV4_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= items) return;
    const long long row = item / C.n_kv;
    const int head = (int)(item - row * C.n_kv), seq = (int)(row / T), t = (int)(row - (long long)seq * T);
    const long long pos = positions[seq * pos_stride + t];
    const bool held = pos >= 0 && pos < C.n_slots;
    const uint8_t* tile = C.tile(seq, head, held ? (int)pos : 0, G);
    const int slot = held ? (int)pos % KV4_TILE : 0;
    float2 a[G], b[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        a[g] = kv4_key(tile, G, g, slot, lane);
        b[g] = kv4_value(tile, G, g, slot, lane);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const size_t at = (size_t)item * D + 64 * g + 2 * lane;
        *reinterpret_cast<uint32_t*>(k + at) = held ? pack_bf16x2(a[g].x, a[g].y) : 0u;
        *reinterpret_cast<uint32_t*>(v + at) = held ? pack_bf16x2(b[g].x, b[g].y) : 0u;
    }
}

}  // namespace cb
