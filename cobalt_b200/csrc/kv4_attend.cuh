// Attention of few rows per KV head (decode, proposed tokens; prompts of head widths without a kernel of their own) over the 4-bit cache.
// The format is in kv4_kernels.cuh.
//
// The columns of a tile product are (token, query head) pairs of one KV head, eight to an n of mma.m16n8k16, and both contractions have
// the cache as their A operand, so no row of the tensor core is wasted:
//     S^T [slots x 8] = K [slots x D] Q^T,        O^T [D x 8] += V^T [D x slots] P^T.
// A code is an operand as it is: a nibble in the low bits of a 16-bit float is the subnormal c * 2^-24, exactly, one nibble further up it is
// 16 times that (the queries' channels, or the result's rows, take the 1/16).  Expanding eight codes is one shift and four ands;
// scales and zeros never touch a code:
//     S = sum_g s_g ( sum_{d in g} q c  -  z_g sum_{d in g} q ),        O_g = sum_j (P_j s_jg) c_j  -  sum_j (P_j s_jg) z_jg,
// the last sum through the tensor core too (z is an fp16 operand), so that both sums carry the same rounded weights: with many
// slots of nearly equal weight they cancel down to the mean, and a rounding of one alone would show.
// Queries are scaled by a power of two into the upper range of fp16, which holds every bf16 significand; so are the weights P s, by
// the largest scale seen so far: fp16 weights (2^-11).  Everything else is fp32 as the tensor core adds it, which cuts each product of a step of 16
// at a quarter of the last place of its running sum: over 80 steps of nearly equal weight (16 sequences of 15000 to 32768 slots) the result's error
// is 1.81e-3 where its own rounding gives 1.65e-3, over a few steps 1.65e-3 to 1.70e-3.  With several tokens (MANY) every column has a power of its own per
// group, as a slot that one token sees and another does not would else cost the other its bits (five tokens, 16 / 4 heads of 64, 8 sequences of
// 700 to 6000 slots 14.1 -> 14.5 us; 40 tokens, 4 of 300 to 2000 18.0 -> 19.4 us).  A running maximum per column, moved only when a score
// exceeds it by 2^8 (fp16 weights have that room), keeps the rescaling of O out of the loop.
//
// A warp owns a ring of tiles, one bulk copy each, and walks every 4th tile of its CTA's share alone; the states of a head are joined
// at its end.  Two ways to share the work:
//   heads  a cluster of 1 to 16 CTAs per head (sequence, tile of columns, KV head); it joins its states over shared memory.  For heads
//          that are short or many.
//   list   the list of all (head, tile) is cut into equal ranges, one per resident CTA, whatever the lengths of the sequences are; heads
//          that lie in several CTAs are joined by kv4_combine_kernel.  For few and long heads.
#pragma once
#include "kv4_kernels.cuh"

namespace cb {

struct Kv4AttendParams {
    const uint16_t* q;                                                 // [n_seq * T] rows of n_heads * D
    long long ld_q;
    Kv4Cache cache;
    const long long* positions;
    long long pos_stride;
    uint16_t* out;                                                     // [n_seq * T][n_heads * D]
    int n_seq, T, n_heads, rep;
    int window, sinks;
    float scale_log2;                                                  // scale * log2(e)
    int cols, col_tiles;                                               // rep * T columns per KV head, in tiles of 8 * NB
    Kv4Div by_rep, by_tiles, by_kv;
    uint32_t* status;                                                  // first bounded wait that gave up
};

// The slots that a token sees: j <= hi and (j >= lo or j < sinks); hi = -1: none.
struct Kv4Range { int lo, hi; };
__device__ __forceinline__ Kv4Range kv4_range(const Kv4AttendParams& P, int seq, int tok) {
    const long long pos = P.positions[seq * P.pos_stride + tok];
    Kv4Range r;
    r.hi = pos < 0 ? -1 : (int)min(pos, (long long)P.cache.n_slots - 1);
    r.lo = P.window > 0 && pos > 0 ? (int)max(0ll, min(pos - P.window + 1, (long long)P.cache.n_slots)) : 0;
    return r;
}
// What a range of tokens sees: the slots between the bounds of all of them, and those between the bounds that bind every one.
struct Kv4Span { int hi_max, lo_min, hi_min, lo_max; };
__device__ __forceinline__ Kv4Span kv4_span(const Kv4AttendParams& P, int seq, int tok0, int tok1) {
    Kv4Span s = {-1, 0x7FFFFFFF, 0x7FFFFFFF, 0};
    for (int t = tok0; t <= tok1; ++t) {
        const Kv4Range r = kv4_range(P, seq, t);
        s.hi_max = max(s.hi_max, r.hi);
        s.hi_min = min(s.hi_min, r.hi);
        s.lo_max = max(s.lo_max, r.lo);
        if (r.lo <= r.hi) s.lo_min = min(s.lo_min, r.lo);
    }
    return s;
}
// The tiles that hold a slot some token sees, in order: i < n_sink: tile i, else first + i - n_sink.  At least one, so that a row
// that sees nothing gets its zeros.
struct Kv4Tiles {
    int n, n_sink, first;
    __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
__device__ __forceinline__ Kv4Tiles kv4_tiles(const Kv4Span& s, int sinks) {
    Kv4Tiles e;
    const int tiles = (s.hi_max + KV4_TILE) / KV4_TILE;                // of slots 0 .. hi_max
    e.n_sink = (min(sinks, s.hi_max + 1) + KV4_TILE - 1) / KV4_TILE;
    e.first = min(tiles, s.lo_min / KV4_TILE);
    if (e.first <= e.n_sink) e.first = e.n_sink = 0;
    e.n = e.n_sink + tiles - e.first;
    if (e.n == 0) { e.n = 1; e.first = 0; }
    return e;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {       // d = a b
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float f16_to_float(uint32_t bits) { return __half2float(__ushort_as_half((uint16_t)bits)); }
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
// the words, and the bf16 values, of a slot's G groups (aligned to their own size where G is a power of two)
template <int G>
__device__ __forceinline__ void kv4_words(const uint8_t* p, uint32_t (&w)[G]) {
    if (G == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[G - 1] = v.y; }
    else if (G == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1 % G] = v.y; w[2 % G] = v.z; w[3 % G] = v.w; }
    else {
#pragma unroll
        for (int gr = 0; gr < G; ++gr) w[gr] = reinterpret_cast<const uint32_t*>(p)[gr];
    }
}
template <int G>
__device__ __forceinline__ void kv4_halves(const uint8_t* p, float (&f)[G]) {
    if (G % 2 == 0) {
#pragma unroll
        for (int k = 0; k < G / 2; ++k) {
            const uint32_t v = reinterpret_cast<const uint32_t*>(p)[k];
            f[(2 * k) % G] = __uint_as_float(v << 16);
            f[(2 * k + 1) % G] = __uint_as_float(v & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int gr = 0; gr < G; ++gr) f[gr] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[gr] << 16);
    }
}

constexpr int KA_WARPS = 4, KA_THREADS = 32 * KA_WARPS;
constexpr int KA_STAGES = 2;
constexpr int KA_MIN_TILES = 4;                                        // per CTA: one per warp
constexpr int KA_ENTRIES = 256;                                        // (sequence, tile of columns) pairs of a list
constexpr int KA_MAX_CLUSTER = 8;                                      // (sixteen are slow to place: 32 heads of 128 tiles took 20.1 us against 12.0)
constexpr int KA_WIDE_HEADS = 8;                                       // of so few heads, with more than four tiles a warp, sixteen all the same
constexpr int ka_max_nb(int G) { return G == 1 ? 4 : G == 2 ? 2 : 1; } // groups of eight columns a warp holds
constexpr int ka_ctas_per_sm(int G, int NB) { return NB == 1 ? (G <= 2 ? 4 : G == 3 ? 3 : 2) : G * NB <= 2 ? 3 : 2; }
constexpr int ka_state_floats(int G, int NB) { return NB * (16 * G + 4); }      // per lane: O, reference and sum of two columns
constexpr size_t ka_ring_bytes(int G) { return (size_t)KA_WARPS * KA_STAGES * (kv4_tile_bytes(G) + 8); }
constexpr size_t ka_list_smem(int G, int NB) { return ka_ring_bytes(G) + 2 * (size_t)ka_state_floats(G, NB) * 128 + KA_ENTRIES * 20 + 64; }
constexpr size_t ka_heads_smem(int G, int NB) { return ka_ring_bytes(G) + 4 * (size_t)ka_state_floats(G, NB) * 128 + NB * 512; }
static_assert(ka_list_smem(4, 1) * 2 <= 226 * 1024 && ka_heads_smem(4, 1) * 2 <= 226 * 1024 && ka_heads_smem(2, 1) * 4 <= 224 * 1024, "CTAs per SM");

// ----------------------------------------------------------------------------- one warp, one head, one tile of columns
// Lane (g, t) = (lane / 4, lane % 4): query column g of every eight; scores of slots g and g + 8 of every sixteen, columns 2t and 2t + 1;
// results of columns 2t, 2t + 1, channels 8g .. 8g + 7 of every group of 64.
template <int G, int NB, bool MANY>
struct Kv4Columns {
    static constexpr int UPS = MANY ? 2 * NB : 1;
    uint32_t qf[NB][G][8];                                             // queries as B operands
    float qs[NB][G][2], fac[NB][2];                                    // their sums per group, what makes a score of a sum
    Kv4Range range[NB][2];
    // scores are taken relative to a reference per column (base: its negative); one above `room` moves it.  up_v: power of two that the
    // weights of a group are scaled by (MANY: of columns nb, c at 2 nb + c; 0 for a column that sees nothing); up_top: the largest
    float o[NB][G][4][4], zero[NB][G][4], base[NB][2], room[NB][2], sum[NB][2], up_v[UPS][G], up_top[G];
    __device__ __forceinline__ float up(int nb, int c, int gr) const { return up_v[MANY ? 2 * nb + c : 0][gr]; }

    __device__ __forceinline__ static void load_queries(const Kv4AttendParams& P, int seq, int kvh, int col0, int lane, uint4 (&raw)[NB][G][2]) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int col = col0 + 8 * nb + (lane >> 2), tok = P.by_rep(col);
            const uint4* src = reinterpret_cast<const uint4*>(P.q + ((long long)seq * P.T + tok) * P.ld_q + (kvh * P.rep + col - tok * P.rep) * (64 * G) + 16 * (lane & 3));
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int k = 0; k < 2; ++k) raw[nb][gr][k] = col < P.cols ? __ldg(src + 8 * gr + k) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ void begin(const Kv4AttendParams& P, int seq, int col0, int lane, const uint4 (&raw)[NB][G][2]) {
        const int t = lane & 3;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            uint32_t top = 0u;                                         // largest magnitude; a NaN stays on top
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t v[4] = {raw[nb][gr][k].x, raw[nb][gr][k].y, raw[nb][gr][k].z, raw[nb][gr][k].w};
#pragma unroll
                    for (int d = 0; d < 4; ++d) top = max(top, max(v[d] & 0x7FFF0000u, (v[d] & 0x7FFFu) << 16));
                }
#pragma unroll
            for (int s = 1; s < 4; s <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
            const int ex = max(-112, (int)(top >> 23) - 127);          // largest magnitude in [2^ex, 2^(ex + 1))
            const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);     // exact: a power of two
            // (queries that are not finite, or beyond 2^117, give no number)
            const float my_fac = ex <= 117 ? P.scale_log2 * __uint_as_float((uint32_t)(ex + 10 + 127) << 23) : __uint_as_float(0x7FC00000u);
            float my_sum[G];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t v[4] = {raw[nb][gr][j].x, raw[nb][gr][j].y, raw[nb][gr][j].z, raw[nb][gr][j].w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {                      // channels 2h, 2h + 1 and 2h + 4, 2h + 5 of the eight
                        const float a = __uint_as_float(v[h] << 16) * up, b = __uint_as_float(v[h] & 0xFFFF0000u) * up;
                        const float c = __uint_as_float(v[h + 2] << 16) * up, d = __uint_as_float(v[h + 2] & 0xFFFF0000u) * up;
                        s += (a + b) + (c + d);
                        qf[nb][gr][4 * j + 2 * h] = pack_f16x2(a, c);
                        qf[nb][gr][4 * j + 2 * h + 1] = pack_f16x2(b * 0.0625f, d * 0.0625f);
                    }
                }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
                my_sum[gr] = s * 0x1p-24f;
            }
            // what the scores of columns 2t, 2t + 1 need
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                fac[nb][c] = __shfl_sync(0xFFFFFFFFu, my_fac, 4 * (2 * t + c));
#pragma unroll
                for (int gr = 0; gr < G; ++gr) qs[nb][gr][c] = __shfl_sync(0xFFFFFFFFu, my_sum[gr], 4 * (2 * t + c));
                const int cc = col0 + 8 * nb + 2 * t + c;
                range[nb][c] = cc < P.cols ? kv4_range(P, seq, P.by_rep(cc)) : Kv4Range{0, MANY ? -1 : 0x7FFFFFFF};
                if (MANY)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr)
                        up_v[(2 * nb + c) % UPS][gr] = range[nb][c].hi >= 0 && (range[nb][c].lo <= range[nb][c].hi || P.sinks > 0) ? 0x1p126f : 0.0f;
                base[nb][c] = sum[nb][c] = 0.0f;
                room[nb][c] = -INFINITY;
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                up_top[gr] = 0x1p126f;
                if (!MANY) up_v[0][gr] = 0x1p126f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    zero[nb][gr][r] = 0.0f;
#pragma unroll
                    for (int m = 0; m < 4; ++m) o[nb][gr][m][r] = 0.0f;
                }
            }
        }
    }

    // sixteen slots of a tile; MASKED: some column does not see all of them
    template <bool MASKED>
    __device__ __forceinline__ void sixteen(const uint8_t* tile, int j0, int b, const Kv4Span& span, int sinks, int lane) {
        const int g = lane >> 2, t = lane & 3;
        auto nobody = [&](int j) { return j > span.hi_max || (j < span.lo_min && j >= sinks); };           // such a slot may hold anything
        // ---- scores of slots g and g + 8, columns 2t, 2t + 1, relative to the reference; value scales of the same slots, times up_v (MANY: not yet)
        float x[NB][4], vs[G][2], acc[NB][G][4];
        const uint8_t* keys = tile + 512 * b + 32 * g + 8 * t;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            const uint2 ka = *reinterpret_cast<const uint2*>(keys + kv4_k_row(G, gr, 0));
            const uint2 kb = *reinterpret_cast<const uint2*>(keys + kv4_k_row(G, gr, 8));
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t wa = (j ? ka.y : ka.x) >> (8 * h), wb = (j ? kb.y : kb.x) >> (8 * h);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint32_t* q = &qf[nb][gr][4 * j + 2 * h];
                        if (j + h == 0)
                            mma_f16_first(acc[nb][gr], wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u, q[0], q[1]);
                        else
                            mma_f16(acc[nb][gr], wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u, q[0], q[1]);
                    }
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            uint32_t m[G];
            float sv[G];
            kv4_words<G>(tile + kv4_k_meta(G, 0, 16 * b + g + 8 * r), m);
            kv4_halves<G>(tile + kv4_v_scale(G, 0, 16 * b + g + 8 * r), sv);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float v = 0.0f;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        const float in = fmaf(-f16_to_float(m[gr] & 0xFFFFu), qs[nb][gr][c], acc[nb][gr][2 * r + c]);
                        v = gr == 0 ? __uint_as_float(m[gr] & 0xFFFF0000u) * in : fmaf(__uint_as_float(m[gr] & 0xFFFF0000u), in, v);
                    }
                    x[nb][2 * r + c] = fmaf(v, fac[nb][c], base[nb][c]);
                }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) vs[gr][r] = MANY ? sv[gr] : sv[gr] * up_v[0][gr];
            if (MASKED) {
                const int j = j0 + 16 * b + g + 8 * r;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        if (j > range[nb][c].hi || (j < range[nb][c].lo && j >= sinks)) x[nb][2 * r + c] = -INFINITY;
#pragma unroll
                for (int gr = 0; gr < G; ++gr)
                    if (nobody(j)) vs[gr][r] = 0.0f;
            }
        }
        bool move = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) move |= fmaxf(x[nb][c], x[nb][c + 2]) > room[nb][c];
        if (__builtin_expect(__any_sync(0xFFFFFFFFu, move), 0)) {      // new references
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(x[nb][c], x[nb][c + 2]);
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
                    const bool first = room[nb][c] == -INFINITY;       // (no number so far: nothing to rescale)
                    if (!first) top = fmaxf(top, 0.0f);
                    const bool set = top != -INFINITY;
                    f[c] = first ? 1.0f : ex2(-top);
                    if (set) {
                        base[nb][c] -= top;
                        room[nb][c] = 8.0f;
                        x[nb][c] -= top;
                        x[nb][c + 2] -= top;
                    }
                    sum[nb][c] *= f[c];
                }
#pragma unroll
                for (int gr = 0; gr < G; ++gr)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        zero[nb][gr][r] *= f[r & 1];
#pragma unroll
                        for (int m = 0; m < 4; ++m) o[nb][gr][m][r] *= f[r & 1];
                    }
            }
        }
        // ---- weights, and weights times scales as B operands (columns by slots: the transpose of how the scores lie)
        uint32_t pf[NB][G][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = ex2(x[nb][2 * r]), p1 = ex2(x[nb][2 * r + 1]);
                sum[nb][0] += p0;
                sum[nb][1] += p1;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    uint32_t w = MANY ? pack_f16x2(p0 * (vs[gr][r] * up(nb, 0, gr)), p1 * (vs[gr][r] * up(nb, 1, gr))) : pack_f16x2(p0 * vs[gr][r], p1 * vs[gr][r]);
                    if (MASKED)                                        // a slot that only some columns see: no NaN of its scale for the others
                        w &= (x[nb][2 * r] == -INFINITY ? 0u : 0xFFFFu) | (x[nb][2 * r + 1] == -INFINITY ? 0u : 0xFFFF0000u);
                    pf[nb][gr][r] = transpose_8x8(w);
                }
            }
        // ---- values: slots 2t, 2t + 1 of each eight, channels 8g .. 8g + 7 of every group
        const uint8_t* vals = tile + kv4_v_chunk(G, 0, 2 * t, g) + 512 * b;
        const uint8_t* zeros = tile + kv4_v_zero(G, 0, 16 * b + 2 * t);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            uint32_t w[2][2], z[2];                                    // [eight slots][channels 0..3, 4..7] of the even (low half) and odd slot
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint2 v = *reinterpret_cast<const uint2*>(vals + 1024 * gr + 256 * r);
                w[r][0] = __byte_perm(v.x, v.y, 0x5410);
                w[r][1] = __byte_perm(v.x, v.y, 0x7632);
                z[r] = *reinterpret_cast<const uint32_t*>(zeros + 64 * gr + 16 * r);
                if (MASKED) {
                    const int j = j0 + 16 * b + 8 * r + 2 * t;
                    if (nobody(j)) z[r] &= 0xFFFF0000u;
                    if (nobody(j + 1)) z[r] &= 0x0000FFFFu;
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                mma_f16(zero[nb][gr], z[0], z[0], z[1], z[1], pf[nb][gr][0], pf[nb][gr][1]);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const uint32_t wa = w[0][m >> 1] >> (8 * (m & 1)), wb = w[1][m >> 1] >> (8 * (m & 1));
                    mma_f16(o[nb][gr][m], wa & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x000F000Fu, wb & 0x00F000F0u, pf[nb][gr][0], pf[nb][gr][1]);
                }
            }
        }
    }

    // The power of two that a scale (its bits) leaves; returns what makes values scaled by `up` so before ones scaled so now
    __device__ __forceinline__ static float lower(float& up, uint32_t scale) {
        const int ex = max(-120, (int)(scale >> 23) - 127);
        const float was = up;
        up = fminf(was, __uint_as_float((uint32_t)(6 - ex + 127) << 23));
        return up * __uint_as_float((254u - (__float_as_uint(was) >> 23)) << 23);
    }
    // The same for every column, by the scales of the slots that it sees itself (here a lane has slots g, g + 8, g + 16, g + 24).  A column whose first
    // visible slot is still to come keeps `up_top` high, and every tile until then comes here
    __device__ __forceinline__ void rescale_columns(const uint8_t* tile, int j0, int sinks, int lane) {
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float sv[4], most = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                sv[k] = fmaxf(__uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(tile + kv4_v_scale(G, gr, (lane >> 2) + 8 * k)) << 16), 0.0f);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = j0 + (lane >> 2) + 8 * k;
                        if (j <= range[nb][c].hi && (j >= range[nb][c].lo || j < sinks)) top = fmaxf(top, sv[k]);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                    float& mine = up_v[(2 * nb + c) % UPS][gr];
                    const float down = lower(mine, __float_as_uint(top));
                    most = fmaxf(most, mine);
                    zero[nb][gr][c] *= down;
                    zero[nb][gr][c + 2] *= down;
#pragma unroll
                    for (int m = 0; m < 4; ++m) { o[nb][gr][m][c] *= down; o[nb][gr][m][c + 2] *= down; }
                }
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            up_top[gr] = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
        }
    }

    // the 32 slots from j0 on
    __device__ __forceinline__ void tile(const uint8_t* tile, int j0, const Kv4Span& span, int sinks, int lane) {
        // a value scale that is too large for the weights' range moves the power of two that they are scaled by
        float sv[G];
        kv4_halves<G>(tile + kv4_v_scale(G, 0, lane), sv);
        bool grow = false;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) grow |= sv[gr] * (MANY ? up_top[gr] : up_v[0][gr]) >= 128.0f;
        const bool whole = j0 + KV4_TILE - 1 <= span.hi_min && (j0 >= span.lo_max || j0 + KV4_TILE <= sinks);
        if (__builtin_expect(__any_sync(0xFFFFFFFFu, grow), 0)) {
            if (MANY && !whole) {
                rescale_columns(tile, j0, sinks, lane);
            } else {                                                   // every column sees the same slots
                const int j = j0 + lane;
                const bool nobody = j > span.hi_max || (j < span.lo_min && j >= sinks);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const float top = nobody ? 0.0f : fmaxf(sv[gr], 0.0f);                         // a NaN stays out
                    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top));
                    if (MANY) lower(up_top[gr], bits);
                    float down[UPS];
#pragma unroll
                    for (int i = 0; i < UPS; ++i) down[i] = lower(up_v[i][gr], bits);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float d = down[MANY ? 2 * nb + (r & 1) : 0];
                            zero[nb][gr][r] *= d;
#pragma unroll
                            for (int m = 0; m < 4; ++m) o[nb][gr][m][r] *= d;
                        }
                }
            }
        }
        // sixteen slots at a time: unrolled to 32 the loop's code no longer fits where four warps per scheduler fetch it from
        if (__builtin_expect(whole, 1)) {
#pragma unroll 1
            for (int b = 0; b < 2; ++b) sixteen<false>(tile, j0, b, span, sinks, lane);
        } else {
#pragma unroll 1
            for (int b = 0; b < 2; ++b) sixteen<true>(tile, j0, b, span, sinks, lane);
        }
    }
};

// The state of a warp's columns in plain fp32 values.  o[16 G]: group, channel pair m, { channel 2m col 0, 2m col 1, 2m + 1 col 0, 2m + 1 col 1 };
// reference and sum of both columns.  In memory [4 + 16 G][32 lanes]: references, sums, o.
template <int G>
struct Kv4State {
    float o[16 * G], ref[2], sum[2];
    template <int NB, bool MANY>
    __device__ __forceinline__ void take(const Kv4Columns<G, NB, MANY>& C, int nb) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float v = C.sum[nb][c];
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, s);
            sum[c] = v;
            ref[c] = C.room[nb][c] == -INFINITY ? -INFINITY : -C.base[nb][c];
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float down[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) down[c] = __uint_as_float((254u - (__float_as_uint(C.up(nb, c, gr)) >> 23)) << 23);
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    o[16 * gr + 4 * m + r] = fmaf(C.o[nb][gr][m][r], r < 2 ? 0x1p24f : 0x1p20f, -C.zero[nb][gr][r & 1]) * down[r & 1];
        }
    }
    __device__ __forceinline__ void store(float* p, int lane) const {
#pragma unroll
        for (int c = 0; c < 2; ++c) { p[c * 32 + lane] = ref[c]; p[(2 + c) * 32 + lane] = sum[c]; }
#pragma unroll
        for (int i = 0; i < 16 * G; ++i) p[(4 + i) * 32 + lane] = o[i];
    }
    __device__ __forceinline__ void join(const float* p, int lane) {
        float mine[2], other[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float r = p[c * 32 + lane], top = fmaxf(ref[c], r), base = top == -INFINITY ? 0.0f : top;
            mine[c] = ex2(ref[c] - base);
            other[c] = ex2(r - base);
            ref[c] = top;
            sum[c] = sum[c] * mine[c] + p[(2 + c) * 32 + lane] * other[c];
        }
#pragma unroll
        for (int i = 0; i < 16 * G; ++i) o[i] = o[i] * mine[i & 1] + p[(4 + i) * 32 + lane] * other[i & 1];
    }
};
// where the result of a column goes, and whether it sees any slot
__device__ __forceinline__ uint16_t* kv4_out(const Kv4AttendParams& P, int seq, int kvh, int col, int D, bool& any) {
    const int tok = P.by_rep(col);
    const Kv4Range r = kv4_range(P, seq, tok);
    any = r.hi >= 0 && (r.lo <= r.hi || P.sinks > 0);
    return P.out + (((long long)seq * P.T + tok) * P.n_heads + kvh * P.rep + col - tok * P.rep) * D;
}
template <int G>
__device__ __forceinline__ void kv4_write_out(const Kv4AttendParams& P, const Kv4State<G>& st, int seq, int kvh, int col0, int D, int first_group, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int col = col0 + 2 * t + c;
        if (col >= P.cols) continue;
        bool any;
        uint16_t* dst = kv4_out(P, seq, kvh, col, D, any) + 64 * first_group + 8 * g;
        const float inv = 1.0f / st.sum[c];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            uint32_t w[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) w[m] = any ? pack_bf16x2(st.o[16 * gr + 4 * m + c] * inv, st.o[16 * gr + 4 * m + 2 + c] * inv) : 0u;
            *reinterpret_cast<uint4*>(dst + 64 * gr) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ----------------------------------------------------------------------------- a cluster per head
// Four values (one channel pair of a group, two columns) of several states
struct Kv4Quad {
    float v[4] = {}, ref[2] = {-INFINITY, -INFINITY}, sum[2] = {};
    __device__ __forceinline__ void join(const float (&r)[2], const float (&s)[2], const float (&o)[4]) {
        float mine[2], other[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float top = fmaxf(ref[c], r[c]), base = top == -INFINITY ? 0.0f : top;
            mine[c] = ex2(ref[c] - base);
            other[c] = ex2(r[c] - base);
            ref[c] = top;
            sum[c] = sum[c] * mine[c] + s[c] * other[c];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] * mine[i & 1] + o[i] * other[i & 1];
    }
    __device__ __forceinline__ void write(const Kv4AttendParams& P, int seq, int kvh, int col0, int D, int channel, int lane) const {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = col0 + 2 * (lane & 3) + c;
            if (col >= P.cols) continue;
            bool any;
            uint16_t* dst = kv4_out(P, seq, kvh, col, D, any) + channel + 8 * (lane >> 2);
            const float inv = 1.0f / sum[c];
            *reinterpret_cast<uint32_t*>(dst) = any ? pack_bf16x2(v[c] * inv, v[2 + c] * inv) : 0u;
        }
    }
};

// grid: heads x `share` CTAs (a cluster).  Nothing is looked up: queries and positions are requested at once, then the tiles.
template <int G, int NB, bool MANY>
__global__ void __launch_bounds__(KA_THREADS, ka_ctas_per_sm(G, NB)) kv4_attend_heads_kernel(const Kv4AttendParams P, const int share) {
    constexpr int D = 64 * G, TILE = kv4_tile_bytes(G), STATE = (16 * G + 4) * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = smem + warp * (KA_STAGES * TILE);
    const uint32_t bar0 = smem_u32(smem + KA_WARPS * KA_STAGES * TILE) + warp * KA_STAGES * 8;
    float* region = reinterpret_cast<float*>(smem + ka_ring_bytes(G));
    float* heads = region + 4 * NB * STATE;                            // [NB][4][32]: references and sums of the CTA's joined states
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (last tokens first: their rows are the longest)
    const int rank = share > 1 ? (int)cluster_rank() : 0, head = (share > 1 ? (int)((gridDim.x - 1 - blockIdx.x) / (unsigned)share) : (int)(gridDim.x - 1 - blockIdx.x));
    const int entry = P.by_kv(head), kvh = head - entry * P.cache.n_kv, seq = P.by_tiles(entry), col0 = (entry - seq * P.col_tiles) * 8 * NB;
    uint4 raw[NB][G][2];
    Kv4Columns<G, NB, MANY>::load_queries(P, seq, kvh, col0, lane, raw);
    const Kv4Span span = kv4_span(P, seq, P.by_rep(col0), P.by_rep(min(col0 + 8 * NB, P.cols) - 1));
    if (lane == 0) {
        for (int s = 0; s < KA_STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        mbar_fence_init();
        fence_proxy_async();
    }
    __syncwarp();
    const Kv4Tiles tiles = kv4_tiles(span, P.sinks);
    const int end = (int)((long long)tiles.n * (rank + 1) / share);
    int next = (int)((long long)tiles.n * rank / share) + warp, fetched = 0, used = 0;
    const uint8_t* base = P.cache.tiles + (long long)seq * P.cache.seq_stride + (long long)kvh * P.cache.n_tiles * TILE;
    auto fetch = [&]() {
        if (next >= end) return;
        if (lane == 0) {
            const int s = fetched % KA_STAGES;
            mbar_arrive_expect_tx(bar0 + 8 * s, TILE);
            bulk_g2s(smem_u32(ring + s * TILE), base + (long long)tiles.tile(next) * TILE, TILE, bar0 + 8 * s);
        }
        ++fetched;
        next += KA_WARPS;
    };
    int i = next;
#pragma unroll 1
    for (int s = 0; s < KA_STAGES; ++s) fetch();
    Kv4Columns<G, NB, MANY> C;
    C.begin(P, seq, col0, lane, raw);
    bool healthy = true;
#pragma unroll 1
    for (; i < end; i += KA_WARPS) {
        const int s = used % KA_STAGES;
        if (__builtin_expect(!__all_sync(0xFFFFFFFFu, mbar_try_wait(bar0 + 8 * s, (uint32_t)(used / KA_STAGES) & 1u)), 0)) {
            healthy = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar0 + 8 * s, (uint32_t)(used / KA_STAGES) & 1u, P.status, DEV_TIMEOUT_TILE));
            if (!healthy) break;
        }
        ++used;
        C.tile(ring + s * TILE, tiles.tile(i) * KV4_TILE, span, P.sinks, lane);
        __syncwarp();
        fetch();
    }
    for (; used < fetched; ++used)                                     // (after a wait that gave up) no copy may land behind the CTA's end
        mbar_wait_bounded(bar0 + 8 * (used % KA_STAGES), (uint32_t)(used / KA_STAGES) & 1u, P.status, DEV_TIMEOUT_TILE);
    // ---- join: the warps' states over shared memory, warp w the channel pair w of every group; then the CTAs' over the cluster
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        Kv4State<G> st;
        st.take(C, nb);
        if (!healthy) st.sum[0] = st.sum[1] = __uint_as_float(0x7FC00000u);            // every value that it would touch: no number
        st.store(region + (warp * NB + nb) * STATE, lane);
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        float ref[4][2], sum[4][2];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float* p = region + (w * NB + nb) * STATE + c * 32 + lane;
                ref[w][c] = p[0];
                sum[w][c] = p[64];
            }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            Kv4Quad q;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float* p = region + (w * NB + nb) * STATE + (4 + 16 * gr + 4 * warp) * 32 + lane;
                const float o[4] = {p[0], p[32], p[64], p[96]};
                q.join(ref[w], sum[w], o);
            }
            if (share == 1) {
                q.write(P, seq, kvh, col0 + 8 * nb, D, 64 * gr + 2 * warp, lane);
            } else {                                                   // (only this lane reads these places of the first state)
                float* p = region + nb * STATE + (4 + 16 * gr + 4 * warp) * 32 + lane;
#pragma unroll
                for (int k = 0; k < 4; ++k) p[32 * k] = q.v[k];
                if (gr == 0 && warp == 0) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) { heads[(nb * 4 + c) * 32 + lane] = q.ref[c]; heads[(nb * 4 + 2 + c) * 32 + lane] = q.sum[c]; }
                }
            }
        }
    }
    if (share == 1) return;
    cluster_sync_all();
    const uint32_t region_at = smem_u32(region) + 4 * lane, heads_at = smem_u32(heads) + 4 * lane;
#pragma unroll 1
    for (int k = rank; k < G * NB; k += share) {                       // (eight columns, group) k: its channel pair `warp`
        const int nb = k / G, gr = k - nb * G;
        Kv4Quad q;
#pragma unroll 4
        for (int r = 0; r < share; ++r) {
            const uint32_t h = map_to_rank(heads_at + nb * 512, r), v = map_to_rank(region_at + (nb * STATE + (4 + 16 * gr + 4 * warp) * 32) * 4, r);
            const float ref[2] = {ld_cluster_f32(h), ld_cluster_f32(h + 128)}, sum[2] = {ld_cluster_f32(h + 256), ld_cluster_f32(h + 384)};
            const float o[4] = {ld_cluster_f32(v), ld_cluster_f32(v + 128), ld_cluster_f32(v + 256), ld_cluster_f32(v + 384)};
            q.join(ref, sum, o);
        }
        q.write(P, seq, kvh, col0 + 8 * nb, D, 64 * gr + 2 * warp, lane);
    }
    cluster_sync_all();                                                // nobody leaves while a neighbour still reads
}

// ----------------------------------------------------------------------------- the list of all heads' tiles, in equal ranges
struct Kv4Work {
    float* partial;                                                    // [CTA][2][floats][32 lanes]
    int4* joins;                                                       // [CTA]: head that begins in this CTA and ends in a later one
};

template <int G, int NB, bool MANY>
__global__ void __launch_bounds__(KA_THREADS, ka_ctas_per_sm(G, NB)) kv4_attend_list_kernel(const Kv4AttendParams P, const Kv4Work W) {
    constexpr int D = 64 * G, TILE = kv4_tile_bytes(G), STATE = (16 * G + 4) * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = smem + warp * (KA_STAGES * TILE);
    const uint32_t bar0 = smem_u32(smem + KA_WARPS * KA_STAGES * TILE) + warp * KA_STAGES * 8;
    float* region = reinterpret_cast<float*>(smem + ka_ring_bytes(G));
    int4* spans = reinterpret_cast<int4*>(region + 2 * NB * STATE);
    int* before = reinterpret_cast<int*>(spans + KA_ENTRIES);          // tiles (of one head) of the entries before
    int* scan = before + KA_ENTRIES;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0) {
        for (int s = 0; s < KA_STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        mbar_fence_init();
        fence_proxy_async();
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- the entries (sequence, tile of columns) and their tiles; this CTA's range of the list: every entry is n_kv heads of n tiles
    const int n_kv = P.cache.n_kv, entries = P.n_seq * P.col_tiles;
    int total = 0;
#pragma unroll 1
    for (int c0 = 0; c0 < entries; c0 += KA_THREADS) {
        const int e = c0 + threadIdx.x;
        int n = 0;
        if (e < entries) {
            const int seq = P.by_tiles(e), col = (e - seq * P.col_tiles) * 8 * NB;
            const Kv4Span sp = kv4_span(P, seq, P.by_rep(col), P.by_rep(min(col + 8 * NB, P.cols) - 1));
            spans[e] = make_int4(sp.hi_max, sp.lo_min, sp.hi_min, sp.lo_max);
            n = kv4_tiles(sp, P.sinks).n;
        }
        int up = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, up, o);
            if (lane >= o) up += v;
        }
        if (lane == 31) scan[warp] = up;
        __syncthreads();
        int at = total + up - n;
#pragma unroll
        for (int w = 0; w < KA_WARPS; ++w) {
            if (w < warp) at += scan[w];
            total += scan[w];
        }
        if (e < entries) before[e] = at;
        __syncthreads();
    }
    total *= n_kv;
    const int per = max(KA_MIN_TILES, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int start = min(total, (int)blockIdx.x * per), end = min(total, start + per);
    if (threadIdx.x == 0) W.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (start >= end) return;

    struct Cursor { int e, kvh, i; Kv4Tiles k; };
    auto load = [&](int e) {
        const int4 v = spans[e];
        return kv4_tiles(Kv4Span{v.x, v.y, v.z, v.w}, P.sinks);
    };
    auto forward = [&](Cursor& c, int by) {                            // the caller stays inside the range
        c.i += by;
        while (c.i >= c.k.n) {
            c.i -= c.k.n;
            if (++c.kvh == n_kv) {
                c.kvh = 0;
                c.k = load(++c.e);
            }
        }
    };
    Cursor at;
    at.e = 0;
    for (int step = KA_ENTRIES / 2; step > 0; step >>= 1)              // the last entry that begins at or before `start`
        if (at.e + step < entries && before[at.e + step] * n_kv <= start) at.e += step;
    at.k = load(at.e);
    at.kvh = (start - before[at.e] * n_kv) / at.k.n;
    at.i = (start - before[at.e] * n_kv) - at.kvh * at.k.n;
    // what the warp fetches next: `run` more of its tiles from `src` on, four tiles apart; then the run that `ahead` stands at
    Cursor ahead = at;
    const int to_fetch = (end - start - warp + KA_WARPS - 1) / KA_WARPS;
    int fetched = 0, used = 0, run = 0, step = warp;
    const uint8_t* src = nullptr;
    auto fetch = [&]() {
        if (fetched >= to_fetch) return;
        if (run == 0) {
            forward(ahead, step);
            const int left = (ahead.i < ahead.k.n_sink ? ahead.k.n_sink : ahead.k.n) - ahead.i;
            run = (left + KA_WARPS - 1) / KA_WARPS;
            step = run * KA_WARPS;
            src = P.cache.tiles + (long long)P.by_tiles(ahead.e) * P.cache.seq_stride +
                  ((long long)ahead.kvh * P.cache.n_tiles + ahead.k.tile(ahead.i)) * TILE;
        }
        if (lane == 0) {
            const int s = fetched % KA_STAGES;
            mbar_arrive_expect_tx(bar0 + 8 * s, TILE);
            bulk_g2s(smem_u32(ring + s * TILE), src, TILE, bar0 + 8 * s);
        }
        ++fetched;
        --run;
        src += KA_WARPS * TILE;
    };
#pragma unroll 1
    for (int s = 0; s < KA_STAGES; ++s) fetch();

    bool healthy = true;
#pragma unroll 1
    for (int i = start; i < end;) {
        const int here = min(at.k.n - at.i, end - i);                  // tiles of this head in this CTA
        const int seq = P.by_tiles(at.e), col0 = (at.e - seq * P.col_tiles) * 8 * NB;
        const Kv4Span span = {spans[at.e].x, spans[at.e].y, spans[at.e].z, spans[at.e].w};
        Kv4Columns<G, NB, MANY> C;
        {
            uint4 raw[NB][G][2];
            Kv4Columns<G, NB, MANY>::load_queries(P, seq, at.kvh, col0, lane, raw);
            C.begin(P, seq, col0, lane, raw);
        }
#pragma unroll 1
        for (int k = (warp - (i - start)) & (KA_WARPS - 1); k < here && healthy; k += KA_WARPS) {
            const int s = used % KA_STAGES;
            if (__builtin_expect(!__all_sync(0xFFFFFFFFu, mbar_try_wait(bar0 + 8 * s, (uint32_t)(used / KA_STAGES) & 1u)), 0)) {
                healthy = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar0 + 8 * s, (uint32_t)(used / KA_STAGES) & 1u, P.status, DEV_TIMEOUT_TILE));
                if (!healthy) break;
            }
            ++used;
            C.tile(ring + s * TILE, at.k.tile(at.i + k) * KV4_TILE, span, P.sinks, lane);
            __syncwarp();
            fetch();
        }
        // ---- join the warps' states
        const bool complete = at.i == 0 && here == at.k.n;
        Kv4State<G> st[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) st[nb].take(C, nb);
        healthy = __syncthreads_and(healthy);                          // (after a wait that gave up: no number, to the end of the range)
        if (!healthy)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) st[nb].sum[0] = st[nb].sum[1] = __uint_as_float(0x7FC00000u);
        // in two rounds (rolled: the code of one): warps 2, 3 into 0, 1, then warp 1 into 0
#pragma unroll 1
        for (int half = KA_WARPS / 2; half > 0; half >>= 1) {
            if (warp >= half && warp < 2 * half)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) st[nb].store(region + ((warp - half) * NB + nb) * STATE, lane);
            __syncthreads();
            if (warp < half)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) st[nb].join(region + (warp * NB + nb) * STATE, lane);
            __syncthreads();
        }
        if (warp == 0) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                if (complete) kv4_write_out<G>(P, st[nb], seq, at.kvh, col0 + 8 * nb, D, 0, lane);
                else st[nb].store(W.partial + ((blockIdx.x * 2ll + (i > start ? 1 : 0)) * NB + nb) * STATE, lane);
            }
            if (at.i == 0 && here < at.k.n && lane == 0)               // it begins here and goes on
                W.joins[blockIdx.x] = make_int4(at.e, at.kvh, i > start ? 1 : 0, (at.k.n - here + per - 1) / per);
        }
        i += here;
        if (i < end) forward(at, here);
    }
    for (; used < fetched; ++used)                                     // (after a wait that gave up) no copy may land behind the CTA's end
        mbar_wait_bounded(bar0 + 8 * (used % KA_STAGES), (uint32_t)(used / KA_STAGES) & 1u, P.status, DEV_TIMEOUT_TILE);
}

// Heads that lie in several CTAs of kv4_attend_list_kernel: block (b, y, z) joins eight columns and a group of channels of the head that begins in
// CTA b.  Its states are slot 1 (or 0: the CTA began with it) of CTA b and slot 0 of the CTAs behind.  First the weight of every state
// (one load round for all of them), then the weighted sums: four warps share the states, a lane has four values of each, four states
// in flight.  State by state with rescaling, one chain of loads per warp, 71 states of a head of 256 took 51 us.
constexpr int KC_THREADS = 512, KC_SHARE = 4;                          // KC_SHARE warps of the same four values
constexpr int KC_MAX_STATES = 1024;                                    // of one head: the CTAs that a launch has at most
template <int G, int NB>
__global__ void __launch_bounds__(KC_THREADS) kv4_combine_kernel(const Kv4AttendParams P, const Kv4Work W) {
    constexpr int STATE = (16 * G + 4) * 32;
    __shared__ float weight[8][KC_MAX_STATES + 1];
    __shared__ float total[8];
    __shared__ float part[KC_SHARE][16][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 j = W.joins[blockIdx.x];
    if (j.x < 0) return;
    const int n = j.w + 1, nb = blockIdx.y, gr = blockIdx.z, seq = P.by_tiles(j.x), col0 = (j.x - seq * P.col_tiles) * 8 * NB + 8 * nb;
    auto state = [&](int k) { return W.partial + (((long long)(blockIdx.x + k) * 2 + (k == 0 ? j.z : 0)) * NB + nb) * STATE; };
    // references and sums of the eight columns: lane t of a state's first four has columns 2t, 2t + 1
    const int c = warp & 7, at = (c & 1) * 32 + (c >> 1);
    float top = -INFINITY;
    if (warp < 8)
        for (int k = lane; k < n; k += 32) top = fmaxf(top, weight[c][k] = state(k)[at]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (top == -INFINITY) top = 0.0f;
    if (warp < 8) {
        float sum = 0.0f;
        for (int k = lane; k < n; k += 32) {
            const float w = ex2(weight[c][k] - top);
            weight[c][k] = w;
            sum = fmaf(w, state(k)[at + 64], sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (lane == 0) total[c] = sum;
    }
    __syncthreads();
    const int quad = warp & 3, share = warp >> 2, t = lane & 3;
    float acc[4] = {};
    const float *w0 = weight[2 * t], *w1 = weight[2 * t + 1];
#pragma unroll 4
    for (int k = share; k < n; k += KC_SHARE) {
        const float* p = state(k) + (4 + 16 * gr + 4 * quad) * 32 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(p[32 * i], i & 1 ? w1[k] : w0[k], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[share][4 * quad + i][lane] = acc[i];
    __syncthreads();
    if (warp == 0) {
        Kv4State<1> st;
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[i] = (part[0][i][lane] + part[1][i][lane]) + (part[2][i][lane] + part[3][i][lane]);
        st.sum[0] = total[2 * t];
        st.sum[1] = total[2 * t + 1];
        kv4_write_out<1>(P, st, seq, j.y, col0, 64 * G, gr, lane);
    }
}

}  // namespace cb
