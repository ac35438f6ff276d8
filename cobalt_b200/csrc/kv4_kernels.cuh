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
constexpr int KV4_THREADS = 128;

__host__ __device__ constexpr int kv4_tile_bytes(int G) { return 36 * 64 * G; }
__device__ __forceinline__ int kv4_k_row(int G, int g, int slot) { return g * 1024 + slot * 32; }
__device__ __forceinline__ int kv4_v_chunk(int G, int g, int slot, int chunk) {
    const int pair = slot >> 1;
    return 1024 * G + g * 1024 + pair * 64 + ((chunk ^ ((pair & 2) << 1)) << 3) + ((slot & 1) << 2);
}
__device__ __forceinline__ int kv4_k_meta(int G, int g, int slot) { return 2048 * G + (slot * G + g) * 4; }
__device__ __forceinline__ int kv4_v_scale(int G, int g, int slot) { return 2176 * G + (slot * G + g) * 2; }
__device__ __forceinline__ int kv4_v_zero(int G, int g, int slot) { return 2240 * G + (g * KV4_TILE + slot) * 2; }

__device__ uint32_t g_kv4_status;                                      // first bounded wait that gave up, on this device, of calls without a word of their own

struct Kv4Cache {
    uint8_t* tiles;
    long long seq_stride;                                              // bytes
    int n_kv, n_tiles, n_slots;
    __device__ __forceinline__ uint8_t* tile(int seq, int kvh, int slot, int G) const {
        return tiles + (long long)seq * seq_stride + ((long long)kvh * n_tiles + slot / KV4_TILE) * kv4_tile_bytes(G);
    }
};

// x / d for 0 <= x < 2^31 (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994)
struct Kv4Div {
    uint32_t mul, shift;
    __device__ __forceinline__ int operator()(int x) const { return (int)((__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift); }
};
inline Kv4Div kv4_div(int d) {
    Kv4Div v = {0, 0};
    while ((1ll << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)((((1ull << v.shift) - (uint64_t)d) << 32) / (uint64_t)d + 1);
    return v;
}

// How a warp takes the channels of a row: lane l has eight neighbouring ones, 8 G lanes a head (4, 2, 1, 1 heads at a time for G = 1 .. 4;
// with G = 3 the last eight lanes idle), eight lanes a group.
template <int G>
struct Kv4Lane {
    static constexpr int LANES = 8 * G, HEADS = 32 / LANES;
    int sub, at, g, chunk;                                             // head of the item, lane in the head, group, chunk of the group
    bool live;
    __device__ __forceinline__ explicit Kv4Lane(int lane) {
        sub = lane / LANES;
        at = lane - sub * LANES;
        g = at >> 3;
        chunk = at & 7;
        live = sub < HEADS;
    }
};

// ----------------------------------------------------------------------------- writing
struct Kv4AppendParams {
    const uint16_t *k, *v, *q;                                         // q may be null
    uint16_t* q_out;
    long long ld_k, ld_v, ld_q, ld_qo;                                 // elements from row to row
    const long long* positions;
    long long pos_stride;                                              // from sequence to sequence (0: the same positions)
    Kv4Cache cache;
    int T, n_heads;
    Kv4Div by_T;
    const float* inv_freq;                                             // may be null: no rotation
    const uint16_t *q_norm, *k_norm;                                   // may be null
    float eps;
};

__device__ __forceinline__ uint32_t bf16x2_min(uint32_t a, uint32_t b) { uint32_t d; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ uint32_t bf16x2_max(uint32_t a, uint32_t b) { uint32_t d; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }

// The rotation's products and sums, each rounded to bf16 as the bf16 cache's kernel rounds them from fp32: a product of two bf16 values is exact there, and a
// sum that is not exact in fp32 lies too near its larger term for the second rounding to differ.
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) { uint32_t d; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ uint32_t bf16x2_add(uint32_t a, uint32_t b) { uint32_t d; asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }

// clamp, then round to nearest even in the low bits of 1.5 * 2^23 + code; the constants of eight such words are taken out at once
__device__ __forceinline__ uint32_t kv4_codes(const float (&c)[8], float zero) {
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 7; i >= 0; --i) codes = codes * 16u + __float_as_uint(__fadd_rn(fminf(fmaxf(__fadd_rn(c[i], zero), 0.0f), 15.0f), 12582912.0f));
    return codes - 0x4B400000u * 0x11111111u;
}
// { codes, zero and scale } by divisions: groups that are constant, not finite, very small or very large
__device__ __noinline__ uint2 kv4_quantise_any(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, float lo, float range) {
    float s = bf16_round(__fdiv_rn(range, 15.0f));
    if (!(s < INFINITY)) return make_uint2(0u, 0x7FC00000u);           // a value that is not finite, or a range beyond fp32
    if (s == 0.0f) s = bf16_round(__fmul_rn(fabsf(lo), 0.00390625f));  // constant
    if (s == 0.0f) return make_uint2(0u, 0u);                          // all zero
    const __half z = __float2half_rn(__fdiv_rn(-lo, s));
    const uint32_t w[4] = {w0, w1, w2, w3};
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __fdiv_rn(__uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16), s);
    return make_uint2(kv4_codes(c, __half2float(z)), (__float_as_uint(s) & 0xFFFF0000u) | __half_as_ushort(z));
}
// Codes (eight channels of this lane), zero (low half) and scale of a group held by eight lanes; w: the channels as bf16 pairs.
__device__ __forceinline__ uint2 kv4_quantise(const uint32_t (&w)[4]) {
    uint32_t lo2 = bf16x2_min(bf16x2_min(w[0], w[1]), bf16x2_min(w[2], w[3])), hi2 = bf16x2_max(bf16x2_max(w[0], w[1]), bf16x2_max(w[2], w[3]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo2 = bf16x2_min(lo2, __shfl_xor_sync(0xFFFFFFFFu, lo2, o));
        hi2 = bf16x2_max(hi2, __shfl_xor_sync(0xFFFFFFFFu, hi2, o));
    }
    const float lo = __uint_as_float(bf16x2_min(lo2, lo2 << 16) & 0xFFFF0000u), hi = __uint_as_float(bf16x2_max(hi2, hi2 << 16) & 0xFFFF0000u);
    const float range = __fsub_rn(hi, lo);
    if (__builtin_expect(!(range > 0x1p-80f && range < 0x1p80f), 0)) return kv4_quantise_any(w[0], w[1], w[2], w[3], lo, range);
    // quotients by the reciprocal, put right by their remainders: the correctly rounded ones while nothing leaves the range of normal
    // numbers (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  One that does is far
    // below a code and a zero point: it rounds to nothing either way
    auto quotient = [](float x, float d, float inv) {
        const float q = __fmul_rn(x, inv);
        return fmaf(fmaf(-q, d, x), inv, q);
    };
    const float s = bf16_round(quotient(range, 15.0f, 1.0f / 15.0f)), inv = __frcp_rn(s);
    const __half z = __float2half_rn(quotient(-lo, s, inv));
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = quotient(__uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16), s, inv);
    return make_uint2(kv4_codes(c, __half2float(z)), (__float_as_uint(s) & 0xFFFF0000u) | __half_as_ushort(z));
}

// A block takes a row (token of a sequence), or a share of its heads; a warp takes Kv4Lane::HEADS heads at a time, keys, then values, then queries.
// The cosines and sines of a position are the same for every head and computed once per block.
// Bound: instruction issue (2.8 a cycle; ~150 per item of keys or values, ~50 per item of queries) until the last third of the time, then the
// loads of 45 % of the warps an SM can hold (64 registers; 48 and 40 spilled and were no faster).  8191 tokens, 32 / 8 heads of 128, rotated: 40.6 us
// for 177 MB (4.4 TB/s); 8 x 200 tokens of 16 heads, not rotated 8.0 us; one token 2.2 us.  What it took from the first form, a warp
// per head with two channels a lane: eight channels a lane (one scale per group and lane, not per 32), rotation in pairs of bf16,
// divisions by one reciprocal (108 - 12 -> 53 us), no index arithmetic per item and blocks of four warps (-> 41 us).
template <int G>
__global__ void __launch_bounds__(KV4_THREADS) kv4_append_kernel(const Kv4AppendParams P) {
    constexpr int D = 64 * G, HALF = D / 2, WARPS = KV4_THREADS / 32, HEADS = Kv4Lane<G>::HEADS;
    __shared__ __align__(16) uint16_t table[2][HALF];                  // cosines, sines
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Kv4Lane<G> L(lane);
    const int row = blockIdx.x, seq = P.by_T(row);
    const long long pos = P.positions[seq * P.pos_stride + (row - seq * P.T)];
    const int n_kv = P.cache.n_kv, kv_items = (n_kv + HEADS - 1) / HEADS, q_items = (P.n_heads + HEADS - 1) / HEADS;       // (no queries: no heads)
    const int begin = blockIdx.y * WARPS + warp, step = gridDim.y * WARPS;
    // this warp's items, as if keys, values and queries were one list
    const int k0 = begin, v0 = k0 + max(0, (kv_items - k0 + step - 1) / step) * step - kv_items;
    const int q0 = v0 + max(0, (kv_items - v0 + step - 1) / step) * step - kv_items;
    const uint16_t* src[3] = {P.k + row * P.ld_k, P.v + row * P.ld_v, P.q + (P.q ? row * P.ld_q : 0)};
    auto request = [&](const uint16_t* p, int item, int heads) {
        const int head = item * HEADS + L.sub;
        return L.live && head < heads ? *reinterpret_cast<const uint4*>(p + head * D + 8 * L.at) : make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 raw_k = request(src[0], k0, n_kv), raw_v = request(src[1], v0, n_kv), raw_q = request(src[2], q0, P.n_heads);
    // cosines and sines of this lane's channels; those of the first half of a head are rotated by the negated sine
    const bool first = L.at < 4 * G;
    const int other = (lane + (first ? 4 * G : -4 * G)) & 31;          // lane of the channels that this lane's are rotated with
    uint32_t cs[4] = {}, sn[4] = {};
    if (P.inv_freq) {
        for (int i = threadIdx.x; i < 2 * HALF; i += KV4_THREADS) {
            const int d = i < HALF ? i : i - HALF;
            const float ang = (float)pos * P.inv_freq[d];
            table[i < HALF ? 0 : 1][d] = float_to_bf16(i < HALF ? cosf(ang) : sinf(ang));
        }
        __syncthreads();
        const int d0 = 8 * (first || !L.live ? L.at % (4 * G) : L.at - 4 * G);
        const uint4 c = *reinterpret_cast<const uint4*>(&table[0][d0]), s = *reinterpret_cast<const uint4*>(&table[1][d0]);
        const uint32_t sign = first ? 0x80008000u : 0u;
        cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
        sn[0] = s.x ^ sign; sn[1] = s.y ^ sign; sn[2] = s.z ^ sign; sn[3] = s.w ^ sign;
    }
    auto turn = [&](uint32_t (&w)[4], const uint16_t* nw) {            // norm: x' = bf16( x * rsqrt(mean(x^2) + eps) * (1 + w) ), and rotation
        if (nw) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = __uint_as_float(w[i] << 16), b = __uint_as_float(w[i] & 0xFFFF0000u);
                ss += a * a + b * b;
            }
#pragma unroll
            for (int o = 1; o < (G == 3 ? 32 : 8 * G); o <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
            const float r = rsqrtf(ss / (float)D + P.eps);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = L.live ? *reinterpret_cast<const uint32_t*>(nw + 8 * L.at + 2 * i) : 0u;
                w[i] = pack_bf16x2(__fmul_rn(__fmul_rn(__uint_as_float(w[i] << 16), r), __fadd_rn(1.0f, __uint_as_float(v << 16))),
                                   __fmul_rn(__fmul_rn(__uint_as_float(w[i] & 0xFFFF0000u), r), __fadd_rn(1.0f, __uint_as_float(v & 0xFFFF0000u))));
            }
        }
        if (P.inv_freq) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = bf16x2_add(bf16x2_mul(w[i], cs[i]), bf16x2_mul(__shfl_sync(0xFFFFFFFFu, w[i], other), sn[i]));
        }
    };
    if (pos >= 0 && pos < P.cache.n_slots) {                           // a position outside the cache is never stored
        const long long head_bytes = (long long)P.cache.n_tiles * kv4_tile_bytes(G);
        const int slot = (int)pos % KV4_TILE;
        uint8_t* tile = P.cache.tile(seq, 0, (int)pos, G);
#pragma unroll 1
        for (int i = k0; i < kv_items; i += step) {
            uint32_t w[4] = {raw_k.x, raw_k.y, raw_k.z, raw_k.w};
            if (i + step < kv_items) raw_k = request(src[0], i + step, n_kv);
            turn(w, P.k_norm);
            const uint2 qz = kv4_quantise(w);
            const int head = i * HEADS + L.sub;
            if (!L.live || head >= n_kv) continue;
            uint8_t* at = tile + head * head_bytes;
            *reinterpret_cast<uint32_t*>(at + kv4_k_row(G, L.g, slot) + 4 * L.chunk) = qz.x;
            if (L.chunk == 0) *reinterpret_cast<uint32_t*>(at + kv4_k_meta(G, L.g, slot)) = qz.y;
        }
#pragma unroll 1
        for (int i = v0; i < kv_items; i += step) {
            const uint32_t w[4] = {raw_v.x, raw_v.y, raw_v.z, raw_v.w};
            if (i + step < kv_items) raw_v = request(src[1], i + step, n_kv);
            const uint2 qz = kv4_quantise(w);
            const int head = i * HEADS + L.sub;
            if (!L.live || head >= n_kv) continue;
            uint8_t* at = tile + head * head_bytes;
            *reinterpret_cast<uint32_t*>(at + kv4_v_chunk(G, L.g, slot, L.chunk)) = qz.x;
            if (L.chunk == 0) *reinterpret_cast<uint16_t*>(at + kv4_v_scale(G, L.g, slot)) = (uint16_t)(qz.y >> 16);
            if (L.chunk == 1) *reinterpret_cast<uint16_t*>(at + kv4_v_zero(G, L.g, slot)) = (uint16_t)qz.y;
        }
    }
    uint16_t* dst = P.q_out + row * P.ld_qo;
#pragma unroll 1
    for (int i = q0; i < q_items; i += step) {
        uint32_t w[4] = {raw_q.x, raw_q.y, raw_q.z, raw_q.w};
        if (i + step < q_items) raw_q = request(src[2], i + step, P.n_heads);
        turn(w, P.q_norm);
        const int head = i * HEADS + L.sub;
        if (L.live && head < P.n_heads) *reinterpret_cast<uint4*>(dst + head * D + 8 * L.at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ----------------------------------------------------------------------------- reading back
// (c - z) * s of eight channels, rounded to bf16
__device__ __forceinline__ uint4 kv4_values(uint32_t codes, uint32_t scale, uint32_t zero) {
    const float s = __uint_as_float(scale << 16), z = __half2float(__ushort_as_half((uint16_t)zero));
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)                                        // 2^23 + c, exactly
        x[i] = __fmul_rn(__fsub_rn(__fsub_rn(__uint_as_float(0x4B000000u | (codes >> (4 * i) & 15u)), 8388608.0f), z), s);
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// k, v [rows][n_kv][D] bf16 of the slots at positions; a position outside the cache reads as zeros.  A warp per row and Kv4Lane::HEADS heads.
// Bound: one chain of loads a warp (position, tile words), which only other warps hide: 8191 tokens, 8 heads of 128, 11.7 us for 43 MB (3.7 TB/s, 57 % of
// the copy rate); 8 x 200 tokens of 16 heads 5.8 us; one token 1.7 us.
template <int G>
__global__ void __launch_bounds__(KV4_THREADS) kv4_read_kernel(const Kv4Cache C, const long long* positions, long long pos_stride, int T,
                                                               long long items, int per_row, uint16_t* k, uint16_t* v) {
    constexpr int D = 64 * G, HEADS = Kv4Lane<G>::HEADS;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long item = (long long)blockIdx.x * (KV4_THREADS / 32) + (threadIdx.x >> 5);
    if (item >= items) return;
    const Kv4Lane<G> L(threadIdx.x & 31);
    const int row = (int)(item / per_row), head = (int)(item - (long long)row * per_row) * HEADS + L.sub, seq = row / T, t = row - seq * T;
    if (!L.live || head >= C.n_kv) return;
    const long long pos = positions[seq * pos_stride + t];
    const bool held = pos >= 0 && pos < C.n_slots;
    uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
    if (held) {
        const uint8_t* tile = C.tile(seq, head, (int)pos, G);
        const int slot = (int)pos % KV4_TILE;
        const uint32_t kc = *reinterpret_cast<const uint32_t*>(tile + kv4_k_row(G, L.g, slot) + 4 * L.chunk);
        const uint32_t vc = *reinterpret_cast<const uint32_t*>(tile + kv4_v_chunk(G, L.g, slot, L.chunk));
        const uint32_t km = *reinterpret_cast<const uint32_t*>(tile + kv4_k_meta(G, L.g, slot));
        const uint32_t vs = *reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, L.g, slot));
        const uint32_t vz = *reinterpret_cast<const uint16_t*>(tile + kv4_v_zero(G, L.g, slot));
        a = kv4_values(kc, km >> 16, km & 0xFFFFu);
        b = kv4_values(vc, vs, vz);
    }
    const size_t at = ((size_t)row * C.n_kv + head) * D + 8 * L.at;
    *reinterpret_cast<uint4*>(k + at) = a;
    *reinterpret_cast<uint4*>(v + at) = b;
}

}  // namespace cb
