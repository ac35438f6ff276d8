// Attention of many rows per KV head (prompts) over the 4-bit cache, tcgen05.mma for both contractions; heads of 64 or 128.  The format is in
// kv4_kernels.cuh.
//
// One CTA = 128 query rows of one KV head: (token, head) pairs, 128 / rep tokens of the rep query heads that share it.  One pass over the
// keys, 128 at a time, with running maxima and sums:
//   warps 0-7   softmax: warp w owns TMEM lanes 32*(w%4).. (a thread = a row) and key columns 64*(w/4).. of every tile.  The two halves of a
//               row's keys keep a maximum, a sum and a context of their own - nothing is exchanged between threads until the end,
//               where the two are joined.  A maximum moves only when a score exceeds it by 2^8 (the probabilities are fp16, times 2^6,
//               which have the room); then the warp rescales its part of the context in tensor memory, after the product before it.
//   warps 8-14  expand: a unit is 32 slots of a group of keys, or of values; codes to fp16 in K-major (values: N-major), 128-byte-swizzled
//               operands.  Units go round the seven warps, each with its next unit requested ahead
//   warp 15     MMA: scores into one of two TMEM buffers, the two contexts into two others; the scores of tile j+1 are issued before
//               the context of tile j
// Key tiles that no row of the CTA sees are skipped (between the first slots and the window, too); only tiles on a border are masked.
// Operands are fp16 (2^-11): in bf16 the roundings of keys, values and probabilities doubled the result's error (3.3e-3 against 1.7e-3, which
// is that of its own rounding).  So that any bf16 range fits, queries are scaled by a power of two per row, keys and values by one each
// per CTA, from the largest magnitude that the scales and zeros of its visible slots allow (looked through once at the start: 4 G + 4 G
// bytes a slot); scores, maxima, sums and contexts are fp32.  fp16 holds 2^-39 of that largest magnitude, so groups down to 2^-20 of it keep
// 2^-19 of their own.  Where groups lie further apart, a slot that only some rows see would cost the others their bits: such a CTA's
// queries and keys, or probabilities and values, are bf16, which holds any of them to 2^-8.
//
// A slot that only some rows see has to stay out of the others' products even where its values are not numbers: such groups are
// expanded to zeros and marked, and marked CTAs look through the scales of their rows' slots once at the end.
//
// Bound: the latency of instructions at 16 warps an SM (1.9 a clock; ALU 47 %, tensor and XU 15 to 18 %).  A unit of expansion takes 1440 clocks, so the
// 16 units of a tile of 128 channels 3300 on seven warps; softmax takes 2000 a tile beside it, the tensor pipe 1000.  2048 tokens, 32 / 8 heads
// of 128: 102.7 us; 2 x 500 tokens with a window of 1024 over 6000 slots, 32 / 16 heads: 70.6 us (the kernel of few rows: 248 and 138 us).
// Steps: a lane per eight channels with scale, zero and visibility for each word 166 us; whole rows per lane, ten operations a word, maxima of raw
// scores 113 us; no branch per word, so that words overlap 97 us; fp16 operands 102 us, two codes per fused multiply-add 101 us, loads of the start
// together 100 us.  Codes at bits that keep a constant's rounding below 2^-12 of a step, two shifts a word more, 100.6 us; a second copy of the roles
// for large scores 101.6 us, for magnitudes far apart 102.4 us.  Eleven expanding warps at 72 registers (softmax 128) slowed the softmax by
// 30 % and gained nothing.
#pragma once
#include "kv4_attend.cuh"
#include "tcgen05.cuh"

namespace cb {

constexpr int KP_ROWS = 128, KP_KEYS = 128;
constexpr int KP_SOFTMAX = 256, KP_EXPAND = 7, KP_THREADS = KP_SOFTMAX + 32 * KP_EXPAND + 32;
constexpr uint32_t KP_SUB = 128 * 128;                                 // bytes of 128 rows x 64 fp16: one swizzled sub-tile
constexpr uint32_t kp_smem_bytes(int G) { return KP_SUB * (uint32_t)(5 * G + 4) + 256 + 1024; }      // Q, 2 K, 2 V, 2 P of two halves; barriers
static_assert(kp_smem_bytes(2) <= 227 * 1024, "the 128-wide head fills the shared memory of one SM");

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
          "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
          "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
          "r"(v[31]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Eight codes of a word as fp16 or bf16 values (c - z) * s.  A code anywhere in the mantissa of an fp32 number is that power of two plus c; at bits 12 and
// 16 (2^11, 2^7) one "and-or" per code makes the number, and the constant -(2^k + z) * s is good to 2^-12 of a step.  (At bit 8, which would save
// two shifts of twelve operations a word, the constant of 2^15 is off by up to 2^-8 of a step: as much as fp16 rounds the largest values of a group,
// but of every value, those next to zero among them.)
struct Kv4Step {
    uint64_t s2, b2;                                                   // pairs: fma.rn.f32x2 takes two codes at a time
    __device__ __forceinline__ static uint64_t two(float lo, float hi) {
        uint64_t d;
        asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
        return d;
    }
    __device__ __forceinline__ Kv4Step(float s, float z) : s2(two(s, s)), b2(two(-(2048.0f + z) * s, -(128.0f + z) * s)) {}
    // the codes at bits 12 and 16
    __device__ __forceinline__ uint32_t pair(uint32_t w, bool bf16) const {
        const uint64_t x = two(__uint_as_float((w & 0xF000u) | 0x45000000u), __uint_as_float((w & 0xF0000u) | 0x43000000u));
        float lo, hi;
        asm("{\n\t.reg .b64 x;\n\tfma.rn.f32x2 x, %2, %3, %4;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(lo), "=f"(hi) : "l"(x), "l"(s2), "l"(b2));
        return bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
    }
    __device__ __forceinline__ uint4 values(uint32_t w, bool bf16) const {
        return make_uint4(pair(w << 12, bf16), pair(w << 4, bf16), pair(w >> 4, bf16), pair(w >> 12, bf16));
    }
};
// largest magnitude that a group's codes could stand for (a constant group near the end of fp32 would leave it); 0 for one that is no number
__device__ __forceinline__ float kv4_largest(uint32_t scale, uint32_t zero) {
    const float s = __uint_as_float(scale << 16), z = f16_to_float(zero), m = s * fmaxf(fabsf(z), fabsf(15.0f - z));
    return (scale & 0x7F80u) == 0x7F80u ? 0.0f : fminf(m, 0x1.fffffep127f);
}

// The same with tiles of 128 slots
__device__ __forceinline__ Kv4Tiles kv4_key_tiles(const Kv4Span& s, int sinks) {
    Kv4Tiles e;
    const int tiles = (s.hi_max + KP_KEYS) / KP_KEYS;
    e.n_sink = (min(sinks, s.hi_max + 1) + KP_KEYS - 1) / KP_KEYS;
    e.first = min(tiles, s.lo_min / KP_KEYS);
    if (e.first <= e.n_sink) e.first = e.n_sink = 0;
    e.n = e.n_sink + tiles - e.first;
    if (e.n == 0) { e.n = 1; e.first = 0; }
    return e;
}

template <int G>
__global__ void __launch_bounds__(KP_THREADS, 1) kv4_prompt_kernel(const Kv4AttendParams P, const int tok_per_cta) {
    constexpr int D = 64 * G, TILE = kv4_tile_bytes(G), SUBTILES = KP_KEYS / KV4_TILE;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t no_number;                                     // a group of values that is not a number was seen
    __shared__ uint32_t largest[2], smallest[2];                       // magnitude (bits) of a group among the visible keys, values; but for groups of zeros
    __shared__ int q_exp[KP_ROWS];                                     // queries of a row were divided by 2^(this - 14); 128: one is not finite
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full_mask = 0xFFFFFFFFu;
    const uint32_t s_raw = smem_u32(smem), s0 = (s_raw + 1023u) & ~1023u;
    const uint32_t q_base = s0, k_base = q_base + G * KP_SUB, v_base = k_base + 2 * G * KP_SUB, p_base = v_base + 2 * G * KP_SUB;
    const uint32_t bars = p_base + 4 * KP_SUB, tmem_slot = bars + 8u * 20u, bar_end = bars + 8u * 21u;
    auto bar_kfull = [&](int s) { return bars + 8u * s; };
    auto bar_kempty = [&](int s) { return bars + 16u + 8u * s; };
    auto bar_vfull = [&](int s) { return bars + 32u + 8u * s; };
    auto bar_vempty = [&](int s) { return bars + 48u + 8u * s; };
    auto bar_sfull = [&](int s) { return bars + 64u + 8u * s; };
    auto bar_sempty = [&](int s) { return bars + 80u + 8u * s; };
    auto bar_pfull = [&](int h, int s) { return bars + 96u + 16u * h + 8u * s; };
    auto bar_pempty = [&](int h, int s) { return bars + 128u + 16u * h + 8u * s; };
    float* stat = reinterpret_cast<float*>(smem + (p_base - s_raw));   // (at the end) [half][row] maximum, then [half][row] sum
    uint32_t* status = P.status;

    // the longest rows (last tokens of the prompt) first, so that the short ones fill the end of the grid
    const int n_kv = P.cache.n_kv, order = (int)(gridDim.x - 1 - blockIdx.x);
    const int block = P.by_kv(order), kvh = order - block * n_kv, seq = blockIdx.y, tok0 = block * tok_per_cta;
    // queries (rows that are none are zero): requested at once, worked on below
    constexpr int CHUNKS = KP_ROWS * D / 8 / KP_THREADS;
    static_assert(CHUNKS * KP_THREADS * 8 == KP_ROWS * D, "whole rounds");
    uint4 queries[CHUNKS];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        const int i = threadIdx.x + k * KP_THREADS, r = i / (D / 8), c = i % (D / 8), tok = P.by_rep(r), row_tok = tok0 + tok;
        queries[k] = make_uint4(0u, 0u, 0u, 0u);
        if (tok < tok_per_cta && row_tok < P.T)
            queries[k] = __ldg(reinterpret_cast<const uint4*>(P.q + ((long long)seq * P.T + row_tok) * P.ld_q + (kvh * P.rep + r - tok * P.rep) * D) + c);
    }
    Kv4Span span = {-1, 0x7FFFFFFF, 0x7FFFFFFF, 0};
    for (int i = lane; i < tok_per_cta && tok0 + i < P.T; i += 32) {
        const Kv4Range r = kv4_range(P, seq, tok0 + i);
        span.hi_max = max(span.hi_max, r.hi);
        span.hi_min = min(span.hi_min, r.hi);
        span.lo_max = max(span.lo_max, r.lo);
        if (r.lo <= r.hi) span.lo_min = min(span.lo_min, r.lo);
    }
    span.hi_max = __reduce_max_sync(full_mask, span.hi_max);
    span.hi_min = __reduce_min_sync(full_mask, span.hi_min);
    span.lo_max = __reduce_max_sync(full_mask, span.lo_max);
    span.lo_min = __reduce_min_sync(full_mask, span.lo_min);
    const Kv4Tiles tiles = kv4_key_tiles(span, P.sinks);
    const int n = tiles.n;
    auto nobody = [&](int j) { return j > span.hi_max || (j < span.lo_min && j >= P.sinks); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar_kfull(s), SUBTILES * G); mbar_init(bar_kempty(s), 1);
            mbar_init(bar_vfull(s), SUBTILES * G); mbar_init(bar_vempty(s), 1);
            mbar_init(bar_sfull(s), 1); mbar_init(bar_sempty(s), KP_SOFTMAX);
            for (int h = 0; h < 2; ++h) { mbar_init(bar_pfull(h, s), 128); mbar_init(bar_pempty(h, s), 1); }
        }
        mbar_init(bar_end, 1);
        mbar_fence_init();
        no_number = largest[0] = largest[1] = 0u;
        smallest[0] = smallest[1] = 0x7F800000u;
    }
    __syncthreads();
    const uint8_t* base = P.cache.tiles + (long long)seq * P.cache.seq_stride + (long long)kvh * P.cache.n_tiles * TILE;
    {                                                                  // the largest and smallest groups of keys and values that some row sees
        float top_k = 0.0f, top_v = 0.0f, low_k = INFINITY, low_v = INFINITY;
        const int slots = n * KP_KEYS;
#pragma unroll 1
        for (int i0 = threadIdx.x; i0 < slots; i0 += 4 * KP_THREADS) {
            uint32_t mk[4][G], vs[4][G], vz[4][G];                     // four slots in flight
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = min(i0 + k * KP_THREADS, slots - 1), j = tiles.tile(i / KP_KEYS) * KP_KEYS + i % KP_KEYS, slot = j % KV4_TILE;
                const bool seen = !nobody(j);                          // (slots beyond the cache are not)
                const uint8_t* tile = base + (long long)(j / KV4_TILE) * TILE;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    mk[k][g] = seen ? __ldg(reinterpret_cast<const uint32_t*>(tile + kv4_k_meta(G, g, slot))) : 0u;
                    vs[k][g] = seen ? __ldg(reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, g, slot))) : 0u;
                    vz[k][g] = seen ? __ldg(reinterpret_cast<const uint16_t*>(tile + kv4_v_zero(G, g, slot))) : 0u;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float key = kv4_largest(mk[k][g] >> 16, mk[k][g] & 0xFFFFu), value = kv4_largest(vs[k][g], vz[k][g]);
                    top_k = fmaxf(top_k, key);
                    top_v = fmaxf(top_v, value);
                    if (key > 0.0f) low_k = fminf(low_k, key);
                    if (value > 0.0f) low_v = fminf(low_v, value);
                }
        }
        const uint32_t bk = __reduce_max_sync(full_mask, __float_as_uint(top_k)), bv = __reduce_max_sync(full_mask, __float_as_uint(top_v));
        const uint32_t ck = __reduce_min_sync(full_mask, __float_as_uint(low_k)), cv = __reduce_min_sync(full_mask, __float_as_uint(low_v));
        if (lane == 0) { atomicMax(&largest[0], bk); atomicMax(&largest[1], bv); atomicMin(&smallest[0], ck); atomicMin(&smallest[1], cv); }
    }
    // The scale is made positive (its sign goes to the queries; none at all: queries of zero), so that maxima can be taken of raw scores
    const uint32_t q_and = P.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu, q_xor = P.scale_log2 < 0.0f ? 0x80008000u : 0u;
    auto store_queries = [&](bool bf16) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int i = threadIdx.x + k * KP_THREADS, r = i / (D / 8), c = i % (D / 8);
            const uint4 v = queries[k];
            const uint32_t w[4] = {(v.x & q_and) ^ q_xor, (v.y & q_and) ^ q_xor, (v.z & q_and) ^ q_xor, (v.w & q_and) ^ q_xor};
            uint32_t top = 0u, o[4];                                   // largest magnitude of the row; a NaN stays on top
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7FFF0000u, (w[e] & 0x7FFFu) << 16));
#pragma unroll
            for (int x = 1; x < D / 8; x <<= 1) top = max(top, __shfl_xor_sync(full_mask, top, x));
            const int ex = max(-112, (int)(top >> 23) - 127);          // in [2^ex, 2^(ex + 1)), to [2^14, 2^15)
            const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float lo = __uint_as_float(w[e] << 16) * up, hi = __uint_as_float(w[e] & 0xFFFF0000u) * up;
                o[e] = bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
            }
            if (c == 0) q_exp[r] = ex;
            sts128(q_base + (uint32_t)(c >> 3) * KP_SUB + (uint32_t)r * 128u + ((((uint32_t)c & 7u) ^ ((uint32_t)r & 7u)) << 4), o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async();
    };
    store_queries(false);
    if (warp == KP_THREADS / 32 - 1) { tmem_alloc<false>(tmem_slot, 512); tmem_relinquish<false>(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // keys and values times a power of two that brings the largest into [2^14, 2^15)
    const int ex_k = max(-110, (int)(largest[0] >> 23) - 127), ex_v = max(-110, (int)(largest[1] >> 23) - 127);
    const float up_k = __uint_as_float((uint32_t)(14 - ex_k + 127) << 23), up_v = __uint_as_float((uint32_t)(14 - ex_v + 127) << 23);
    auto apart = [&](int i) { return __uint_as_float(smallest[i]) * 0x1p20f < __uint_as_float(largest[i]); };
    const bool wide_k = apart(0), wide_v = apart(1);                   // bf16 operands
    if (wide_k) {
        store_queries(true);
        __syncthreads();
    }
    // Scores that may pass 2^24 (times log2(e)) are rounded before the maximum is taken off: it was rounded, too, and what an exact product would leave
    // of the two is no longer small
    int ex_q = -1000;
#pragma unroll
    for (int r = lane; r < KP_ROWS; r += 32) ex_q = max(ex_q, q_exp[r] < 128 ? q_exp[r] : -1000);
    ex_q = __reduce_max_sync(full_mask, ex_q);
    const bool big = ldexpf(fabsf(P.scale_log2), ex_q + ex_k + 2 + 7) > 0x1p24f;
    const uint32_t tmem = lds32(tmem_slot), tmem_o = tmem + 2 * KP_KEYS;              // scores 2 x 128 columns, contexts 2 x D

    // (PLAIN: fp16 operands, scores below 2^24.  The rest, which asks at every step, has a copy of its own: asked in one, 100.6 -> 106.6 us)
    auto roles = [&](auto plain) {
        constexpr bool PLAIN = decltype(plain)::value;
        if (warp < 8) {
            // =========================================================== softmax, epilogue
            const int half = warp >> 2, r = threadIdx.x & 127;
            const int sub = P.by_rep(r), tok = tok0 + sub, head = r - sub * P.rep;
            const bool valid = sub < tok_per_cta && tok < P.T;
            const Kv4Range range = valid ? kv4_range(P, seq, tok) : Kv4Range{0, -1};
            const uint32_t my_lanes = (uint32_t)((warp & 3) * 32) << 16, my_o = tmem_o + my_lanes + (uint32_t)(half * D);
            bool healthy = true;
            // What a raw score is times.  Positive: a masked score is -inf before it, and must stay so.  Raw scores are below 2^38, so those that are held to
            // the smallest normal number here are nothing (below 2^-88) either way; the exponents are added as whole numbers, as a
            // product of two of the three factors may leave fp32 where that of all three does not
            float scale = q_exp[r] < 128 ? ldexpf(P.scale_log2 == 0.0f ? 1.0f : fabsf(P.scale_log2), q_exp[r] + ex_k - 28) : __uint_as_float(0x7FC00000u);
            if (scale < 0x1p-126f) scale = 0x1p-126f;
            float m = -INFINITY, l = 0.0f;                                  // reference and sum of this row's half, scores times log2(e)
            for (int j = 0; j < n; ++j) {
                healthy = __all_sync(full_mask, mbar_wait_bounded(bar_sfull(j & 1), (uint32_t)(j >> 1) & 1u, status, DEV_TIMEOUT_ACC));
                if (!healthy) break;
                tc_fence_after();
                uint32_t v[2][32];
                tmem_ld32(tmem + my_lanes + (uint32_t)((j & 1) * KP_KEYS + half * 64), v[0]);
                tmem_ld32(tmem + my_lanes + (uint32_t)((j & 1) * KP_KEYS + half * 64 + 32), v[1]);
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(bar_sempty(j & 1));
                float x[64];
#pragma unroll
                for (int i = 0; i < 64; ++i) x[i] = __uint_as_float(v[i >> 5][i & 31]);
                const int k0 = tiles.tile(j) * KP_KEYS;
                if (k0 + KP_KEYS - 1 > span.hi_min || (k0 < span.lo_max && k0 + KP_KEYS > P.sinks)) {                      // a border crosses this tile
                    const int hi = range.hi - k0 - half * 64, lo = range.lo - k0 - half * 64, sinks = P.sinks - k0 - half * 64;
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (i > hi || (i < lo && i >= sinks)) x[i] = -INFINITY;
                }
                float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int i = 4; i < 60; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) t[k] = fmaxf(fmaxf(t[k], x[i + k]), x[i + 4 + k]);
                const float top = scale * fmaxf(fmaxf(fmaxf(t[0], x[60]), fmaxf(t[1], x[61])), fmaxf(fmaxf(t[2], x[62]), fmaxf(t[3], x[63])));
                const bool move = top > m + 8.0f;
                if (__any_sync(full_mask, move)) {
                    // (a row without a reference has a context of zeros: nothing to rescale)
                    const float f = move && m != -INFINITY ? ex2(m - top) : 1.0f;
                    if (move) { m = top; l *= f; }
                    if (j > 0 && __any_sync(full_mask, f != 1.0f)) {
                        healthy = __all_sync(full_mask, mbar_wait_bounded(bar_pempty(half, (j - 1) & 1), (uint32_t)((j - 1) >> 1) & 1u, status, DEV_TIMEOUT_EMPTY));
                        if (!healthy) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(my_o + (uint32_t)c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st32(my_o + (uint32_t)c, o);
                            tmem_st_wait();
                        }
                        tc_fence_before();
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m, base = m == -INFINITY ? 0.0f : 6.0f - m;            // probabilities times 2^6
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float a = ex2(PLAIN ? fmaf(x[2 * i], scale, base) : __fmul_rn(x[2 * i], scale) - ref + 6.0f);
                    const float b = ex2(PLAIN ? fmaf(x[2 * i + 1], scale, base) : __fmul_rn(x[2 * i + 1], scale) - ref + 6.0f);
                    p[i] = !PLAIN && wide_v ? pack_bf16x2(a, b) : pack_f16x2(a, b);
                    s[i & 3] += a + b;
                }
                l += (s[0] + s[1]) + (s[2] + s[3]);
                healthy = __all_sync(full_mask, mbar_wait_bounded(bar_pempty(half, j & 1), ((uint32_t)(j >> 1) & 1u) ^ 1u, status, DEV_TIMEOUT_EMPTY));
                if (!healthy) break;
                const uint32_t row = p_base + (uint32_t)(j & 1) * 2u * KP_SUB + (uint32_t)half * KP_SUB + (uint32_t)r * 128u;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    sts128(row + (((uint32_t)c ^ (uint32_t)(r & 7)) << 4), p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
                fence_proxy_async();
                mbar_arrive(bar_pfull(half, j & 1));
            }
            if (healthy)                                                   // the last products of both halves
                for (int h = 0; h < 2; ++h)
                    healthy = __all_sync(full_mask, healthy && mbar_wait_bounded(bar_pempty(h, (n - 1) & 1), (uint32_t)((n - 1) >> 1) & 1u, status, DEV_TIMEOUT_ACC));
            tc_fence_after();
            stat[half * KP_ROWS + r] = m;
            if (!healthy) l = __uint_as_float(0x7FC00000u);            // (a wait gave up: no number, in the channels of both halves)
            stat[(2 + half) * KP_ROWS + r] = l;
            asm volatile("bar.sync 1, 480;" ::: "memory");                  // the softmax warps; those that expand have arrived (no_number)
            const float om = stat[(half ^ 1) * KP_ROWS + r], ol = stat[(2 + (half ^ 1)) * KP_ROWS + r];
            const float gm = fmaxf(m, om), base = gm == -INFINITY ? 0.0f : gm;
            const float mine = ex2(m - base), other = ex2(om - base);
            const float inv = __uint_as_float((uint32_t)(ex_v - 14 + 127) << 23) / (l * mine + ol * other);
            const float w0 = (half ? other : mine) * inv, w1 = (half ? mine : other) * inv;        // of the contexts of halves 0 and 1
            const bool any = range.hi >= 0 && (range.lo <= range.hi || P.sinks > 0);
            bool nan = !healthy;
            if (no_number && any && healthy) {                         // a marked group: does this row see one?
                const int g = half * (D / 2) / 64;
                for (int j = 0; j <= range.hi; ++j) {
                    if (j < range.lo && j >= P.sinks) { j = range.lo - 1; continue; }
                    const uint8_t* tile = P.cache.tile(seq, kvh, j, G);
                    const uint32_t sc = *reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, g, j % KV4_TILE));
                    nan |= (sc & 0x7F80u) == 0x7F80u;
                }
            }
#pragma unroll 1
            for (int c0 = 0; c0 < D / 2; c0 += 32) {
                uint32_t a[32], b[32];
                const uint32_t col = (uint32_t)(half * (D / 2) + c0);
                tmem_ld32(tmem_o + my_lanes + col, a);
                tmem_ld32(tmem_o + my_lanes + (uint32_t)D + col, b);
                tmem_ld_wait();
                if (valid) {
                    uint4* dst = reinterpret_cast<uint4*>(P.out + (((long long)seq * P.T + tok) * P.n_heads + kvh * P.rep + head) * D + col);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = 8 * c + 2 * e;
                            o[e] = pack_bf16x2(fmaf(__uint_as_float(a[i]), w0, __uint_as_float(b[i]) * w1),
                                               fmaf(__uint_as_float(a[i + 1]), w0, __uint_as_float(b[i + 1]) * w1));
                            o[e] = !any ? 0u : nan ? 0x7FC07FC0u : o[e];
                        }
                        dst[c] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            tc_fence_before();
        } else if (warp < 8 + KP_EXPAND) {
            // =========================================================== expansion: units (tile, keys or values, group, 32 slots) in this order
            // (seven warps: after keys of a tile a warp comes to keys of the same or the next one or to values of the same, so that what it last waited
            // for puts every slot at most one turn of its barrier behind; with a step of more than a tile's units it could pass a turn unseen)
            static_assert(KP_EXPAND < 2 * SUBTILES, "units of a tile of the narrowest head");
            const int units = n * 2 * G * SUBTILES;
            // Keys: a lane has a slot, all 64 channels.  Values: a lane has half the chunks of a pair of slots; every other two pairs swap neighbouring
            // chunks, so that eight lanes store to eight places of a row
            const int pair = lane >> 1, swap = (pair >> 1) & 1;
            uint4 raw[2];
            uint32_t meta[3];                                              // keys: { zero, scale }; values: the scales, both zeros.  Nothing is done
            bool hidden[2];                                                // with them before they are used: the request would wait for its loads
            auto request = [&](int u) {
                const int sub = u % SUBTILES, g = u / SUBTILES % G, at = tiles.tile(u / (2 * G * SUBTILES)) * SUBTILES + sub;
                const bool keys = u / (G * SUBTILES) % 2 == 0, held = at < P.cache.n_tiles;              // (the last tile may reach beyond the cache)
                const uint8_t* tile = base + (long long)(held ? at : 0) * TILE;
                const uint4* p = reinterpret_cast<const uint4*>(tile + (keys ? 0 : 1024 * G) + 1024 * g + 32 * lane);       // 32 slots, or 16 pairs of 2 halves
                raw[0] = __ldg(p);
                raw[1] = __ldg(p + 1);
                const int j = KV4_TILE * at + (keys ? lane : 2 * pair);
                hidden[0] = !held || nobody(j);                            // zeros: nobody sees the slot, it may hold anything
                hidden[1] = !held || nobody(j + 1);
                if (keys) {
                    meta[0] = __ldg(reinterpret_cast<const uint32_t*>(tile + kv4_k_meta(G, g, lane)));
                } else {
                    meta[0] = __ldg(reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, g, 2 * pair)));
                    meta[1] = __ldg(reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, g, 2 * pair + 1)));
                    meta[2] = __ldg(reinterpret_cast<const uint32_t*>(tile + kv4_v_zero(G, g, 2 * pair)));
                }
            };
            int u = warp - 8;
            if (u < units) request(u);
#pragma unroll 1
            for (; u < units; u += KP_EXPAND) {
                const int sub = u % SUBTILES, g = u / SUBTILES % G, j = u / (2 * G * SUBTILES), s = j & 1;
                const bool keys = u / (G * SUBTILES) % 2 == 0;
                if (!__all_sync(full_mask, mbar_wait_bounded(keys ? bar_kempty(s) : bar_vempty(s), ((uint32_t)(j >> 1) & 1u) ^ 1u, status, DEV_TIMEOUT_EMPTY))) break;
                const uint32_t dst = (keys ? k_base : v_base) + (uint32_t)(s * G + g) * KP_SUB + (uint32_t)(32 * sub) * 128u;
                const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
                if (keys) {
                    const uint32_t m = hidden[0] ? 0u : meta[0];
                    const Kv4Step st(__uint_as_float(m & 0xFFFF0000u) * up_k, f16_to_float(m & 0xFFFFu));
                    if (u + KP_EXPAND < units) request(u + KP_EXPAND);
                    auto store = [&](int c, const uint4 x) { sts128(dst + (uint32_t)lane * 128u + (((uint32_t)c ^ ((uint32_t)lane & 7u)) << 4), x.x, x.y, x.z, x.w); };
#pragma unroll
                    for (int c = 0; c < 8; ++c) store(c, st.values(w[c], !PLAIN && wide_k));
                } else {
                    uint32_t s0v = hidden[0] ? 0u : meta[0], s1v = hidden[1] ? 0u : meta[1];
                    uint32_t z0 = hidden[0] ? 0u : meta[2] & 0xFFFFu, z1 = hidden[1] ? 0u : meta[2] >> 16;
                    if ((s0v & 0x7F80u) == 0x7F80u) { s0v = z0 = 0u; no_number = 1u; }
                    if ((s1v & 0x7F80u) == 0x7F80u) { s1v = z1 = 0u; no_number = 1u; }
                    const Kv4Step even(__uint_as_float(s0v << 16) * up_v, f16_to_float(z0)), odd(__uint_as_float(s1v << 16) * up_v, f16_to_float(z1));
                    if (u + KP_EXPAND < units) request(u + KP_EXPAND);
                    const uint32_t row = 2u * (uint32_t)pair;
                    uint32_t we[4], wo[4], at[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {                          // words 2k, 2k + 1: place 4 h + k of both slots
                        const int k1 = i ^ 1;
                        we[i] = swap ? w[2 * k1] : w[2 * i];
                        wo[i] = swap ? w[2 * k1 + 1] : w[2 * i + 1];
                        const uint32_t place = 4u * ((uint32_t)lane & 1u) + (uint32_t)(swap ? k1 : i);
                        at[i] = place ^ (((uint32_t)pair & 2u) << 1);      // its chunk
                    }
                    auto store = [&](uint32_t r, uint32_t chunk, const uint4 x) { sts128(dst + r * 128u + ((chunk ^ (r & 7u)) << 4), x.x, x.y, x.z, x.w); };
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        store(row, at[i], even.values(we[i], !PLAIN && wide_v));
                        store(row + 1u, at[i], odd.values(wo[i], !PLAIN && wide_v));
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(keys ? bar_kfull(s) : bar_vfull(s));
            }
            asm volatile("bar.arrive 1, 480;" ::: "memory");
        } else {
            // =========================================================== MMA
            constexpr uint32_t BF16 = (1u << 7) | (1u << 10);           // (both operands fp16 without)
            const uint32_t idesc_s = umma_idesc(KP_KEYS) & ~(!PLAIN && wide_k ? 0u : BF16);
            const uint32_t idesc_o = (umma_idesc(D) & ~(!PLAIN && wide_v ? 0u : BF16)) | (1u << 16);        // B (= V) is N-major
            const uint64_t qd = umma_smem_desc(q_base);
            bool healthy = true;
            auto issue_scores = [&](int j) {
                const int s = j & 1;
                healthy = healthy && mbar_wait_bounded(bar_kfull(s), (uint32_t)(j >> 1) & 1u, status, DEV_TIMEOUT_STAGE);
                healthy = __all_sync(full_mask, healthy && mbar_wait_bounded(bar_sempty(s), ((uint32_t)(j >> 1) & 1u) ^ 1u, status, DEV_TIMEOUT_EMPTY));
                if (!healthy) return;
                tc_fence_after();
                const uint64_t kd = umma_smem_desc(k_base + (uint32_t)s * G * KP_SUB);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t off = (uint64_t)((k / 4) * (KP_SUB >> 4) + (k % 4) * 2);
                        umma_bf16<false>(tmem + (uint32_t)(s * KP_KEYS), qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
                    }
                    umma_commit<false>(bar_kempty(s));
                    umma_commit<false>(bar_sfull(s));
                }
                __syncwarp();
            };
            auto issue_context = [&](int j) {
                const int s = j & 1;
                healthy = __all_sync(full_mask, healthy && mbar_wait_bounded(bar_vfull(s), (uint32_t)(j >> 1) & 1u, status, DEV_TIMEOUT_STAGE));
                for (int h = 0; h < 2; ++h) {
                    healthy = __all_sync(full_mask, healthy && mbar_wait_bounded(bar_pfull(h, s), (uint32_t)(j >> 1) & 1u, status, DEV_TIMEOUT_FULL));
                    if (!healthy) return;
                    tc_fence_after();
                    const uint64_t pd = umma_smem_desc(p_base + (uint32_t)(2 * s + h) * KP_SUB);
                    const uint64_t vd = umma_smem_desc_mn(v_base + (uint32_t)s * G * KP_SUB, KP_SUB);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_bf16<false>(tmem_o + (uint32_t)(h * D), pd + (uint64_t)(k * 2), vd + (uint64_t)((4 * h + k) * (2048 >> 4)), idesc_o,
                                             (j > 0 || k > 0) ? 1u : 0u);
                        umma_commit<false>(bar_pempty(h, s));
                        if (h == 1) umma_commit<false>(bar_vempty(s));
                    }
                    __syncwarp();
                }
            };
            issue_scores(0);
            for (int j = 0; j < n && healthy; ++j) {
                if (j + 1 < n) issue_scores(j + 1);
                issue_context(j);
            }
            if (!healthy) {                                            // nothing issued may run behind the CTA's end
                if (elect_one()) umma_commit<false>(bar_end);
                __syncwarp();
                mbar_wait_bounded(bar_end, 0u, status, DEV_TIMEOUT_ACC);
            }
        }
    };
    if (__builtin_expect(big || wide_k || wide_v, 0)) roles(std::false_type());
    else roles(std::true_type());
    tc_fence_before();
    __syncthreads();
    if (warp == KP_THREADS / 32 - 1) { tc_fence_after(); tmem_dealloc<false>(tmem, 512); }
}

}  // namespace cb
