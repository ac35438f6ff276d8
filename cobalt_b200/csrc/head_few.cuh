// The products of head_loss.cuh for few tokens (up to 128), which are bound by reading W once: the other way round.  W is the M side, 256 rows (or hidden
// columns) a stage of 32 KB, and the tokens are the N side, 32 to 128 columns.
//
// In the pair kernel's tile the tokens are the 256 rows of A, most of them zeros that take half of every stage: with the five stages that it had at the time
// it held 70 KB of W in flight, and 32000 x 4096 took 68 us for one token (3.9 TB/s).  Here six stages hold up to 192 KB: 46 us (5.7 TB/s; the loss with the
// kernel that joins its statistics 49), of which 39 stream W and the rest is the start, the last unit's epilogue and the launch.  With gradients (16 tokens):
// logits again 40 us, 40 % of them from the L2, dx 45, dw (head_loss.cuh) 58, 27 tiles a pair of 1 us each behind 9 us of first passes through code; the loss
// itself then takes 61, as dw's last writes leave the L2 meanwhile.
//
//   stats, dlogits   A = W, two blocks of up to 128 of its rows; B = x.  A unit of work is `rows` rows, so many that the units go round the CTAs evenly.
//                    TMEM lane = row of W, column = token: a warp's statistics are reductions over its lanes, 32 tokens at a time.
//                    Tokens stay where they are (none are packed): what a row without a target holds reaches its own column alone, which is not used.
//                    dlogits leaves d in rows 0 .. n - 1 of the piece's scratch (a second bf16 value of it in rows n .. 2n - 1), and what dw takes beside
//                    it: x with zeros for those rows, as often, and the factor of the sums.
//   dx               A = W with hidden columns as M (M-major as it lies), K = rows of W; B = d, both values of a stage one after the other on the same A.  A
//                    unit is 256 hidden columns and a range of rows.
//   warps 0-7  epilogue: warp w owns lanes 32 * (w % 4).. of block w / 4        warp 8  TMA        warp 9  MMA
#pragma once
#include "head_loss.cuh"

namespace cb {

constexpr int HF_TOKENS = 128;             // at most
constexpr int HF_EPI_WARPS = 8;
// Stages of logits that are summed in tensor memory: half of what the pair kernel takes, as the epilogue has the time here, and a quarter where it has least to do.
// Error of a loss (32000 x 4096, in 2-norm; median of 40 draws for one token) with 1, 2, 4 stages: one token 3.6e-8, 3.9e-8, 7.3e-8, where fp32 products summed
// in fp32 have 3.2e-8; 64 tokens 7.8e-8, 6.9e-8, 9.7e-8, fp32 3.6e-7.  Time: 16 tokens 50.9, 50.7, 50.1 us, 64 tokens of 8000 x 1024 22.3,
// 20.0, 18.4; 128 tokens with 2, 4, 8 stages 62.7, 59.0, 58.0.
__host__ __device__ constexpr int hf_sum_stages(int n_pad) { return n_pad <= 32 ? 2 : 4; }
constexpr int HF_THREADS = HF_EPI_WARPS * 32 + 64;
constexpr uint32_t HF_A_BYTES = 4 * HL_BOX;
// Up to 64 tokens d goes out as hi + lo, each rounded to bf16: 2^-16 of d is lost where one value loses 2^-8, as much as the result's own rounding (dw of one
// token is d times its row of x).  W is read once all the same, and the tensor pipe has the time: gradients of 16 tokens of 32000 x 4096, error in 2-norm 1.9e-3 -> 1.7e-3,
// with the shorter code of the kernel for 64 tokens 219 -> 212 us.  More tokens than that are bound by reading d for every 256 hidden columns: 128 tokens would
// take 313 us instead of 273, 100 of 262144 x 5376 2.55 ms instead of 2.07, and have one value.
constexpr int hf_parts(int n) { return n <= HF_TOKENS / 2 ? 2 : 1; }
// A stage holds W and `parts` operands of the tokens' side (dx: hi and lo; logits: x)
constexpr int hf_stages(int n_pad, int parts) { return n_pad * parts <= 32 ? 6 : n_pad * parts <= 64 ? 5 : 4; }
constexpr uint32_t hf_stage_bytes(int n_pad, int parts) { return HF_A_BYTES + (uint32_t)(n_pad * parts) * 128u; }
// stages, barriers, what belongs to a token (16 bytes), the warps' statistics of it (8 bytes each), room for the alignment
constexpr uint32_t hf_smem(int n_pad, int parts) {
    return (uint32_t)hf_stages(n_pad, parts) * hf_stage_bytes(n_pad, parts) + 256 + (uint32_t)n_pad * (16 + 8 * HF_EPI_WARPS) + 1024;
}
static_assert(hf_smem(32, 1) <= 227 * 1024 && hf_smem(64, 1) <= 227 * 1024 && hf_smem(96, 1) <= 227 * 1024 && hf_smem(128, 1) <= 227 * 1024 &&
              hf_smem(32, 2) <= 227 * 1024 && hf_smem(64, 2) <= 227 * 1024, "stages of every size fit");

struct HfParams {
    int kind;                              // HL_STATS, HL_DLOGITS or HL_DX
    int n, n_pad;                          // tokens; the N of the products, a multiple of 32
    int v0, cols;                          // piece of the vocabulary: its first row, and its rows inside the vocabulary
    int units, rows;                       // stats, dlogits: rows of W a unit, a multiple of 16
    int h_tiles, splits, add;              // dx: tiles of 256 hidden columns; ranges of the piece; the slabs hold the sums of earlier pieces
    int hidden;
    const long long* targets;              // stats, dlogits: of every token; one outside the vocabulary does not count
    long long vocab;
    int* counted;                          // stats: [0] tokens that count, [1] zero, for the kernel that joins; dlogits: [0] rows of d, for dw
    float2* part;                          // stats: [units][n_pad]
    float* at;
    const float2* stats;                   // dlogits: maximum and log2 of the sum
    const float* grad;                     // gradient of the loss, of every token (grad_step 1) or of the sum or mean (0)
    int grad_step, mean;
    float* factor;
    const uint16_t* x;
    long long ldx;
    uint16_t* packed;                      // [values of d][n][hidden]
    uint16_t* d;                           // [values of d][n][ld_d]
    int ld_d;
    float* slab;                           // [split][n][hidden]
    uint32_t* status;
};

// Over the lanes of a warp and 32 values a lane: lane c gets the reduction of every lane's value c.  31 exchanges, each step halves the values.
template <typename F>
__device__ __forceinline__ float reduce_columns(float (&v)[32], int lane, F f) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        const bool up = (lane & s) != 0;
#pragma unroll
        for (int i = 0; i < s; ++i) {
            const float got = __shfl_xor_sync(0xFFFFFFFFu, up ? v[i] : v[i + s], s);
            v[i] = f(up ? v[i + s] : v[i], got);
        }
    }
    return v[0];
}

// The warp that issues the MMAs, as HlIssue does: eight of them and a commit a stage, the next stage's barrier asked ahead (barriers lie where the pair kernel has them)
struct HfIssue {
    uint32_t s0, bars, tmem, stage_bytes, depth, n_pad;
    uint32_t* status;
    uint32_t s, ph, buf, aph, uses;
    bool ready;

    // PARTS operands B of a stage go onto the same sums
    template <bool A_MN, int PARTS>
    __device__ __forceinline__ bool unit(int stages, int per) {
        const uint32_t full_mask = 0xFFFFFFFFu;
        const uint32_t idesc = umma_idesc(n_pad) | (A_MN ? 1u << 15 : 0u);
        constexpr uint32_t A_STEP = A_MN ? 2048 >> 4 : 32 >> 4;
        for (int k0 = 0; k0 < stages; k0 += per) {
            if (!__all_sync(full_mask, mbar_wait_bounded(hl_free(bars, buf), aph ^ 1u, status, DEV_TIMEOUT_EMPTY))) return false;
            tc_fence_after();
            const uint32_t d = tmem + buf * 2u * n_pad;
            for (int k = k0; k < min(stages, k0 + per); ++k) {
                if (!ready && !__all_sync(full_mask, mbar_wait_bounded(hl_full(bars, s), ph, status, DEV_TIMEOUT_FULL))) return false;
                tc_fence_after();
                const uint32_t next = s + 1 == depth ? 0 : s + 1, next_ph = next ? ph : ph ^ 1u;
                const bool seen = mbar_test(hl_full(bars, next), next_ph);
                const uint32_t at = (s0 + s * stage_bytes) >> 4, b = (at + (HF_A_BYTES >> 4)) | 1u << 16;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t block = 0; block < 2; ++block) {
                        const uint32_t a = (at + block * (2 * HL_BOX >> 4)) | (A_MN ? (HL_BOX >> 4) << 16 : 1u << 16);
#pragma unroll
                        for (int q = 0; q < HL_KS / 16; ++q) umma_low<false>(d + block * n_pad, a + A_STEP * q, b + 2u * q, idesc, (k > k0 || q > 0) ? 1u : 0u);
                        if constexpr (PARTS > 1) {
#pragma unroll
                            for (int q = 0; q < HL_KS / 16; ++q) umma_low<false>(d + block * n_pad, a + A_STEP * q, b + (n_pad * 128u >> 4) + 2u * q, idesc, 1u);
                        }
                    }
                    umma_commit<false>(hl_empty(bars, s));
                }
                __syncwarp();
                ++uses;
                ready = __all_sync(full_mask, seen);
                s = next;
                ph = next_ph;
            }
            if (elect_one()) umma_commit<false>(hl_acc(bars, buf));
            __syncwarp();
            buf ^= 1u;
            if (buf == 0) aph ^= 1u;
        }
        return true;
    }
};

// TOKENS: at most.  A CTA passes most of the code once, so its length is time: that for 64 tokens takes 206 us for the gradients of one token, that for 128 216.
template <int TOKENS>
__global__ void __launch_bounds__(HF_THREADS, 1) head_few_kernel(const __grid_constant__ HfParams P, const __grid_constant__ CUtensorMap amap,
                                                                 const __grid_constant__ CUtensorMap bmap) {
    constexpr int PARTS = hf_parts(TOKENS);
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full_mask = 0xFFFFFFFFu;
    const uint32_t s0 = (smem_u32(smem) + 1023u) & ~1023u;
    const bool logits = P.kind != HL_DX;
    const int sum_stages = logits ? hf_sum_stages(P.n_pad) : HL_GRAD_STAGES;
    const int parts = logits ? 1 : PARTS;                  // operands of a stage's tokens' side
    const uint32_t stages = (uint32_t)hf_stages(P.n_pad, parts), stage_bytes = hf_stage_bytes(P.n_pad, parts);
    const uint32_t bars = s0 + stages * stage_bytes;
    const uint32_t tmem_slot = bars + 160u;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < stages; ++s) { mbar_init(hl_full(bars, s), 1); mbar_init(hl_empty(bars, s), 1); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(hl_acc(bars, b), 1); mbar_init(hl_free(bars, b), HF_EPI_WARPS); }
        mbar_fence_init();
        fence_proxy_async();
    }
    if (warp == HF_EPI_WARPS + 1) { tmem_alloc<false>(tmem_slot, 512); tmem_relinquish<false>(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);
    pdl_next();
    pdl_wait();
    const int k_all = ((logits ? P.hidden : P.cols) + HL_KS - 1) / HL_KS;
    auto k_range = [&](int u, int* k0, int* k1) {
        const int split = logits ? 0 : u / P.h_tiles;
        *k0 = logits ? 0 : (int)((long long)k_all * split / P.splits);
        *k1 = logits ? k_all : (int)((long long)k_all * (split + 1) / P.splits);
    };

    if (warp < HF_EPI_WARPS) {
        // =========================================================== epilogue
        const int block = warp >> 2, in_block = (warp & 3) * 32 + lane;
        const uint32_t my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(block * P.n_pad);
        float4* const token_s = reinterpret_cast<float4*>(smem + (bars + 256u - smem_u32(smem)));
        float2* const part_s = reinterpret_cast<float2*>(token_s + P.n_pad);           // [warp][n_pad]
        auto epilogue_sync = [&]() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        auto counts = [&](long long t) { return t >= 0 && t < P.vocab; };
        if (logits && blockIdx.x == 0 && warp == 0) {
            int counted = 0;
            for (int i = lane; i < P.n; i += 32) counted += counts(P.targets[i]) ? 1 : 0;
            counted = __reduce_add_sync(full_mask, counted);
            if (lane == 0) {
                P.counted[0] = P.kind == HL_STATS ? counted : PARTS * P.n;
                P.counted[1] = 0;
                if (P.kind == HL_DLOGITS) *P.factor = P.grad_step ? 1.0f : P.mean ? P.grad[0] / (float)max(counted, 1) : P.grad[0];
            }
        }
        if (P.kind == HL_DLOGITS) {
            if (threadIdx.x < P.n) {
                const long long t = P.targets[threadIdx.x];
                const float2 s = P.stats[threadIdx.x];
                token_s[threadIdx.x] = make_float4(s.x, s.y, P.grad_step ? P.grad[threadIdx.x] : 1.0f, __int_as_float(counts(t) ? (int)t : -1));
            }
            for (int i = blockIdx.x; i < P.n; i += gridDim.x) {
                const bool in = counts(P.targets[i]);
                for (int c = threadIdx.x; c < P.hidden / 8; c += HF_EPI_WARPS * 32) {
                    const uint4 v = in ? reinterpret_cast<const uint4*>(P.x + i * P.ldx)[c] : make_uint4(0, 0, 0, 0);
                    reinterpret_cast<uint4*>(P.packed + (long long)i * P.hidden)[c] = v;
                    if (PARTS > 1) reinterpret_cast<uint4*>(P.packed + (long long)(P.n + i) * P.hidden)[c] = v;
                }
            }
            epilogue_sync();
        }
        bool healthy = true;
        uint32_t buf = 0, ph = 0;
        for (int u = blockIdx.x; u < P.units; u += gridDim.x) {
            int k0, k1;
            k_range(u, &k0, &k1);
            float acc[TOKENS];
#pragma unroll
            for (int q = 0; q < TOKENS; ++q) acc[q] = 0.0f;
            for (int k = k0; k < k1; k += sum_stages) {
                if (healthy) healthy = __all_sync(full_mask, mbar_wait_bounded(hl_acc(bars, buf), ph, P.status, DEV_TIMEOUT_ACC));
                tc_fence_after();
#pragma unroll
                for (int q = 0; q < TOKENS / 32; ++q) {
                    if (32 * q >= P.n_pad) continue;
                    uint32_t v[32];
                    tmem_ld32(my_tmem + buf * 2u * (uint32_t)P.n_pad + 32u * q, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) acc[32 * q + e] += healthy ? __uint_as_float(v[e]) : __uint_as_float(0x7FC00000u);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && healthy) mbar_arrive(hl_free(bars, buf));
                buf ^= 1u;
                if (buf == 0) ph ^= 1u;
            }
            if (logits) {
                const int half = P.rows / 2, in_piece = u * P.rows + block * half + in_block, row = P.v0 + in_piece;
                const bool mine = in_block < half && in_piece < P.cols;
#pragma unroll
                for (int q = 0; q < TOKENS / 32; ++q) {
                    if (32 * q >= P.n_pad) continue;
                    const int token = 32 * q + lane;
                    if (P.kind == HL_STATS) {
                        float v[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = acc[32 * q + e] = mine ? acc[32 * q + e] : -INFINITY;
                        const float top = reduce_columns(v, lane, [](float a, float b) { return fmaxf(a, b); });
                        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = exp2_fast((acc[32 * q + e] - __shfl_sync(full_mask, base, e)) * LOG2E);
                        const float sum = reduce_columns(v, lane, [](float a, float b) { return a + b; });
                        part_s[warp * P.n_pad + token] = make_float2(top, sum);
                        // the token whose target is this row: its logit
                        const long long t = token < P.n ? P.targets[token] : -1;
                        const int rel = t >= 0 && t < P.vocab ? (int)t - (row - lane) : -1;      // lane of this warp that holds it
                        for (unsigned left = __ballot_sync(full_mask, rel >= 0 && rel < 32); left; left &= left - 1) {
                            const int e = __ffs(left) - 1, holder = __shfl_sync(full_mask, rel, e);
                            float own = 0.0f;
#pragma unroll
                            for (int c = 0; c < 32; ++c) own = c == e ? acc[32 * q + c] : own;
                            if (lane == holder && mine) P.at[32 * q + e] = own;
                        }
                    } else {
                        const bool in_d = in_block < half && in_piece < P.ld_d;
                        const long long lo_rows = (long long)P.n * P.ld_d;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int c = 32 * q + e;
                            if (c >= P.n) continue;
                            float g = 0.0f;
                            const float4 r = token_s[c];
                            if (mine && __float_as_int(r.w) >= 0) {
                                g = exp2_fast(fmaf(acc[c] - r.x, LOG2E, -r.y));
                                if (__float_as_int(r.w) == row) g -= 1.0f;
                                g *= r.z;
                            }
                            if (!in_d) continue;
                            uint16_t* at = P.d + (long long)c * P.ld_d + in_piece;
                            if (PARTS == 1) {
                                *at = float_to_bf16(g);
                            } else {
                                const float hi = bf16_round(g), rest = g - hi;         // (exact)
                                const uint32_t both = pack_bf16x2(hi, fabsf(hi) < INFINITY ? rest : 0.0f);
                                *at = (uint16_t)both;
                                at[lo_rows] = (uint16_t)(both >> 16);
                            }
                        }
                    }
                }
                if (P.kind == HL_STATS) {                              // the warps' statistics joined, a thread a token
                    epilogue_sync();
                    if ((int)threadIdx.x < P.n_pad) {
                        float top = -INFINITY, sum = 0.0f;
                        for (int w = 0; w < HF_EPI_WARPS; ++w) top = fmaxf(top, part_s[w * P.n_pad + threadIdx.x].x);
                        const float base = top == -INFINITY ? 0.0f : top;
                        for (int w = 0; w < HF_EPI_WARPS; ++w) {
                            const float2 v = part_s[w * P.n_pad + threadIdx.x];
                            sum += v.y * exp2_fast((v.x - base) * LOG2E);
                        }
                        P.part[(long long)u * P.n_pad + threadIdx.x] = make_float2(top, sum);
                    }
                    epilogue_sync();
                }
            } else {
                const int split = u / P.h_tiles, h = (u - split * P.h_tiles) * HL_TILE + block * 128 + in_block;
                float* dst = P.slab + (long long)split * P.n * P.hidden + h;
                if (h < P.hidden) {
#pragma unroll
                    for (int c = 0; c < TOKENS; ++c) {
                        if (c >= P.n) continue;
                        float* at = dst + (long long)c * P.hidden;
                        *at = P.add ? *at + acc[c] : acc[c];
                    }
                }
            }
        }
    } else if (warp == HF_EPI_WARPS) {
        // =========================================================== TMA
        bool good = true;
        uint32_t s = 0, ph = 0, fills = 0;
        const uint32_t bytes = (logits ? (uint32_t)P.rows * 128u : HF_A_BYTES) + (uint32_t)(P.n_pad * parts) * 128u;
        for (int u = blockIdx.x; good && u < P.units; u += gridDim.x) {
            int k0, k1;
            k_range(u, &k0, &k1);
            const int h0 = logits ? 0 : u % P.h_tiles * HL_TILE, r0 = P.v0 + (logits ? u * P.rows : 0);
            for (int i = k0; i < k1; ++i) {
                good = __all_sync(full_mask, mbar_wait_bounded(hl_empty(bars, s), ph ^ 1u, P.status, DEV_TIMEOUT_EMPTY));
                if (!good) break;
                const uint32_t dst = s0 + s * stage_bytes, bar = hl_full(bars, s);
                const int k = P.kind == HL_DLOGITS ? k1 - 1 - i : i;   // backwards: the L2 still holds the columns that the loss read last
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar, bytes);
                    if (logits) {
                        tma_load_2d<false>(dst, &amap, k * HL_KS, r0, bar);
                        tma_load_2d<false>(dst + 2 * HL_BOX, &amap, k * HL_KS, r0 + P.rows / 2, bar);
                    } else {
#pragma unroll
                        for (int b = 0; b < 4; ++b) tma_load_2d<false>(dst + b * HL_BOX, &amap, h0 + 64 * b, r0 + k * HL_KS, bar);
                    }
                    tma_load_2d<false>(dst + HF_A_BYTES, &bmap, k * HL_KS, 0, bar);
                    if (PARTS > 1 && !logits) tma_load_2d<false>(dst + HF_A_BYTES + (uint32_t)P.n_pad * 128u, &bmap, k * HL_KS, P.n, bar);
                }
                __syncwarp();
                ++fills;
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
        }
        hl_landed<false>(bars, fills, stages, P.status);
    } else {
        // =========================================================== MMA
        HfIssue I = {s0, bars, tmem, stage_bytes, stages, (uint32_t)P.n_pad, P.status, 0, 0, 0, 0, 0, false};
        bool good = true;
        for (int u = blockIdx.x; good && u < P.units; u += gridDim.x) {
            int first, last;
            k_range(u, &first, &last);
            good = logits ? I.unit<false, 1>(last - first, sum_stages) : I.unit<true, PARTS>(last - first, sum_stages);
        }
        hl_multiplied<false>(bars, I.uses, stages, P.status);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == HF_EPI_WARPS + 1) { tc_fence_after(); tmem_dealloc<false>(tmem, 512); }
}

}  // namespace cb
