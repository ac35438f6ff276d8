// Softmax cross entropy of hidden states against the rows of a head, l[n, v] = x[n] . W[v], loss[n] = log sum_v exp l[n, v] - l[n, t[n]], and
// its gradients, d = (softmax(l) - onehot(t)) * g, dx = d W, dW = d^T x, in pieces of the vocabulary: no more than a piece of l or d exists.
//
// One kernel does all four products.  A pair of CTAs holds a tile of 256 x 256 results (tcgen05.mma.cta_group::2, each CTA 128 rows of A and
// 128 columns of B per stage of 64, so that a stage costs an SM 32 KB for 512 clocks of MMA) and walks a list of tiles:
//   stats     A = x, B = W (both K-major): maximum and sum of exp of every row over the tile's columns, and the target's logit
//   dlogits   the same product again; d, rounded to bf16, goes to the piece's scratch [tokens][columns]
//   dx        A = d (K-major), B = W with the vocabulary as K (N-major as it lies): fp32 sums over the pieces, in slabs [split][token][hidden]
//   dw        A = d with the tokens as K (M-major as it lies), B = x the same: dW, rounded once
// Operands come by TMA in boxes of 64 x 64, whatever their order: a box is 64 rows of 128 swizzled bytes, and which of its sides is K is
// the descriptor's business.
//   warps 0-7  epilogue: warp w owns TMEM lanes 32 * (w % 4).. (a thread = a row) and columns 128 * (w / 4)..
//   warp 8     TMA         warp 9     MMA (of the pair's first CTA)
// Two accumulators of 256 columns: the epilogue of a tile runs under the next one's products.
//
// Tokens without a target are left out beforehand (prepare kernel: targets and rows of x that count, packed in order), so a prompt that is not
// trained on costs nothing, and nothing in its rows, NaN included, reaches a sum.  How many count is known on the device alone; tiles behind
// them are not visited.
//
// Precision.  The tensor core cuts every product at its running sum's last bits, always towards zero: over 5376 columns that is 1e-5 of a
// logit, all in one direction.  So logits are summed in tensor memory over 512 columns at a time, and these sums in fp32 registers.  d is rounded
// to bf16 (2^-8 of an element at most, at random), because the tensor core multiplies two operands of one type.  A factor g that all tokens share
// stays out of d and multiplies the sums: -g + a little, rounded in the target's column of every token, would be off by the same for all of
// them, while -1 + a little is not (2048 columns, 5000 rows, 600 tokens, error in 2-norm with g inside 2.6e-3).
#pragma once
#include "staged_input.cuh"
#include "tcgen05.cuh"

namespace cb {

constexpr int HL_TILE = 256;               // rows and columns of a pair's tile
constexpr int HL_KS = 64;                  // K per stage
constexpr int HL_STAGES = 6;
constexpr uint32_t HL_BOX = 64 * 128;      // bytes of 64 rows x 64 bf16
constexpr uint32_t HL_STAGE_BYTES = 4 * HL_BOX;
constexpr int HL_EPI_WARPS = 8;
constexpr int HL_THREADS = HL_EPI_WARPS * 32 + 64;
constexpr int HL_SUM_STAGES = 8;           // stages of logits that are summed in tensor memory
constexpr uint32_t HL_SMEM = HL_STAGES * HL_STAGE_BYTES + 256 + 1024;
constexpr int HL_JOBS = 3;
constexpr float LOG2E = 1.44269504088896341f;

enum HlKind : int { HL_STATS = 0, HL_DLOGITS = 1, HL_DX = 2, HL_DW = 3 };

// Tiles of one product.  Tokens in tiles of 256 (their number comes from the device), the vocabulary of a piece, or hidden columns.
struct HlJob {
    int kind;
    int v0, cols;                          // piece of the vocabulary: its first row, and its rows inside the vocabulary
    int n_tiles;                           // tiles along B's side: of the piece (stats, dlogits) or of hidden columns (dx, dw)
    int splits;                            // dx: ranges of the piece that are summed in slabs of their own
    int add;                               // dx: the slabs hold the sums of earlier pieces
    int buf;                               // which of the two scratch pieces holds d
};

struct HlParams {
    HlJob job[HL_JOBS];
    int n_jobs;
    const int* count;                      // tokens that count
    int tok0, tok_tiles;                   // stats: first token, and at most this many tiles of tokens
    int n_rows;                            // rows of the packed x (and of a slab)
    int hidden;
    const int* target;                     // [rows of the packed x]
    float2* part;                          // stats: [2 * tiles of the vocabulary][ld_part] maximum, sum of exp(l - maximum)
    float* at;                             // stats: [rows] the target's logit
    int ld_part;
    const float4* row;                     // dlogits: [rows] maximum, log2 of the sum, factor of the row
    const float* factor;                   // dw: of the sums
    uint16_t* d[2];                        // [rounded rows][ld_d]
    int ld_d;
    float* slab;                           // dx
    uint16_t* dw;
    long long ld_dw;
    int wide;                              // dw's rows are 32-byte aligned
    uint32_t* status;
};

struct HlTile { int job, kind, m, n, k0, k1; };

// Tile i of the launch's list.  Jobs follow one another.  Logits: tokens in groups of at most 12 tiles, so that a group's x stays in the L2
// while the vocabulary streams by, once a group; gradients: neighbours share the operand that is longer.
__device__ __forceinline__ bool hl_tile(const HlParams& P, int tokens, int i, HlTile* t) {
    const int nt = min(max((tokens - P.tok0 + HL_TILE - 1) / HL_TILE, 1), P.tok_tiles);
#pragma unroll
    for (int j = 0; j < HL_JOBS; ++j) {
        if (j >= P.n_jobs) return false;
        const HlJob& J = P.job[j];
        const int m_tiles = J.kind == HL_DW ? (J.cols + HL_TILE - 1) / HL_TILE : nt;
        const int all = m_tiles * J.n_tiles * J.splits;
        if (i >= all) { i -= all; continue; }
        t->job = j;
        t->kind = J.kind;
        t->k0 = 0;
        if (J.kind <= HL_DLOGITS) {
            const int groups = (nt + 11) / 12, per = (nt + groups - 1) / groups;
            const int g = i / (per * J.n_tiles), in = i - g * per * J.n_tiles, width = min(per, nt - g * per);
            t->n = in / width;
            t->m = g * per + in - t->n * width;
            t->k1 = (P.hidden + HL_KS - 1) / HL_KS;
        } else if (J.kind == HL_DX) {
            const int ks = (J.cols + HL_KS - 1) / HL_KS, s = i / (m_tiles * J.n_tiles), in = i - s * m_tiles * J.n_tiles;
            t->m = in / J.n_tiles;
            t->n = in - t->m * J.n_tiles;
            t->k0 = (int)((long long)ks * s / J.splits);
            t->k1 = (int)((long long)ks * (s + 1) / J.splits);
            t->m |= s << 20;                               // the split rides along
        } else {
            t->m = i / J.n_tiles;
            t->n = i - t->m * J.n_tiles;
            t->k1 = max((tokens + HL_KS - 1) / HL_KS, 1);
        }
        return true;
    }
    return false;
}

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

__global__ void __launch_bounds__(HL_THREADS, 1) head_product_kernel(const __grid_constant__ HlParams P, const __grid_constant__ CUtensorMap xmap,
                                                                     const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap dmap0,
                                                                     const __grid_constant__ CUtensorMap dmap1) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full_mask = 0xFFFFFFFFu;
    const uint32_t s0 = (smem_u32(smem) + 1023u) & ~1023u;
    const uint32_t bars = s0 + HL_STAGES * HL_STAGE_BYTES;
    auto bar_full = [&](uint32_t s) { return bars + 8u * s; };
    auto bar_empty = [&](uint32_t s) { return bars + 64u + 8u * s; };
    auto bar_acc = [&](uint32_t b) { return bars + 128u + 8u * b; };
    auto bar_free = [&](uint32_t b) { return bars + 144u + 8u * b; };
    const uint32_t tmem_slot = bars + 160u;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < HL_STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(bar_acc(b), 1); mbar_init(bar_free(b), 2 * HL_EPI_WARPS); }
        mbar_fence_init();
        fence_proxy_async();
    }
    if (warp == HL_EPI_WARPS + 1) { tmem_alloc<true>(tmem_slot, 512); tmem_relinquish<true>(); }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();                                    // the other CTA's barriers are in place before anyone arrives on them
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);
    const int tokens = *P.count;
    HlTile t;

    if (warp < HL_EPI_WARPS) {
        // =========================================================== epilogue
        const uint32_t my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(warp >> 2) * 128u;
        const int my_row = (int)rank * 128 + (warp & 3) * 32 + lane, my_col = (warp >> 2) * 128;
        bool healthy = true;
        uint32_t buf = 0, ph = 0;
        for (int i = pair; hl_tile(P, tokens, i, &t); i += pairs) {
            const HlJob& J = P.job[t.job];
            const bool logits = t.kind <= HL_DLOGITS;
            const int split = t.m >> 20, row = (t.m & 0xFFFFF) * HL_TILE + my_row, col = t.n * HL_TILE + my_col;
            const int r = t.kind == HL_STATS ? P.tok0 + row : row;
            // what a row of logits needs; requested under the products
            int target = -1;
            float4 rowv = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (logits && r < tokens) {
                target = P.target[r] - J.v0 - col;
                if (t.kind == HL_DLOGITS) rowv = P.row[r];
            }
            float acc[128];
#pragma unroll
            for (int q = 0; q < 128; ++q) acc[q] = 0.0f;
            for (int k = t.k0; k < t.k1; k += logits ? HL_SUM_STAGES : t.k1 - t.k0) {
                if (healthy) healthy = __all_sync(full_mask, mbar_wait_bounded<true>(bar_acc(buf), ph, P.status, DEV_TIMEOUT_ACC));
                if (healthy) {
                    tc_fence_after();
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t v[32];
                        tmem_ld32(my_tmem + buf * 256u + 32u * q, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[32 * q + e] += __uint_as_float(v[e]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_rank(bar_free(buf), 0));
                }
                buf ^= 1u;
                if (buf == 0) ph ^= 1u;
            }
            if (!healthy) {                                // a wait gave up: everything that this tile feeds becomes NaN
#pragma unroll
                for (int q = 0; q < 128; ++q) acc[q] = __uint_as_float(0x7FC00000u);
            }
            if (t.kind == HL_STATS) {
                const int valid = J.cols - col;            // columns of this half inside the vocabulary
                if (valid < 128) {
#pragma unroll
                    for (int q = 0; q < 128; ++q)
                        if (q >= valid) acc[q] = -INFINITY;
                }
                float m[4] = {acc[0], acc[1], acc[2], acc[3]};
#pragma unroll
                for (int q = 4; q < 128; ++q) m[q & 3] = fmaxf(m[q & 3], acc[q]);
                const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), base = top == -INFINITY ? 0.0f : top;
                if (__any_sync(full_mask, target >= 0 && target < 128)) {
                    float own = 0.0f;
#pragma unroll
                    for (int q = 0; q < 128; ++q) own = q == target ? acc[q] : own;
                    if (target >= 0 && target < 128) P.at[r] = own;
                }
                // (the difference first: the product of a large logit with log2(e) would be rounded where the difference is exact)
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < 128; ++q) s[q & 3] += exp2_fast((acc[q] - base) * LOG2E);
                P.part[(long long)(2 * t.n + (warp >> 2)) * P.ld_part + row] = make_float2(top, (s[0] + s[1]) + (s[2] + s[3]));
            } else if (t.kind == HL_DLOGITS) {
                const bool in = row < tokens;
                const int valid = in ? J.cols - col : 0;
                uint16_t* dst = P.d[J.buf] + (long long)row * P.ld_d + col;
                const bool mine = __any_sync(full_mask, target >= 0 && target < 128);
#pragma unroll
                for (int q = 0; q < 128; q += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float p[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int c = q + 2 * e + h;
                            p[h] = exp2_fast(fmaf(acc[c] - rowv.x, LOG2E, -rowv.y));
                            if (mine && c == target) p[h] -= 1.0f;
                            p[h] = c < valid ? p[h] * rowv.z : 0.0f;
                        }
                        w[e] = pack_bf16x2(p[0], p[1]);
                    }
                    store32(dst + q, w);
                }
            } else if (t.kind == HL_DX) {
                if (row < tokens) {
                    float* dst = P.slab + ((long long)split * P.n_rows + row) * P.hidden + col;
#pragma unroll
                    for (int q = 0; q < 128; q += 4) {
                        if (col + q >= P.hidden) continue;
                        float4 v = make_float4(acc[q], acc[q + 1], acc[q + 2], acc[q + 3]);
                        if (J.add) {
                            const float4 o = *reinterpret_cast<const float4*>(dst + q);
                            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                        }
                        *reinterpret_cast<float4*>(dst + q) = v;
                    }
                }
            } else {
                const float g = *P.factor;
                if (row < J.cols) {
                    uint16_t* dst = P.dw + (long long)(J.v0 + row) * P.ld_dw + col;
#pragma unroll
                    for (int q = 0; q < 128; q += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(acc[q + 2 * e] * g, acc[q + 2 * e + 1] * g);
                        if (P.wide && col + q + 16 <= P.hidden) {
                            store32(dst + q, w);
                        } else {                           // (the width is a multiple of 8)
                            if (col + q < P.hidden) *reinterpret_cast<uint4*>(dst + q) = make_uint4(w[0], w[1], w[2], w[3]);
                            if (col + q + 8 < P.hidden) *reinterpret_cast<uint4*>(dst + q + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
            }
        }
    } else if (warp == HL_EPI_WARPS) {
        // =========================================================== TMA
        bool good = true;
        uint32_t s = 0, ph = 0;
        const int mine = (int)rank * 128;
        for (int i = pair; good && hl_tile(P, tokens, i, &t); i += pairs) {
            const HlJob& J = P.job[t.job];
            const int m0 = (t.m & 0xFFFFF) * HL_TILE + mine, n0 = t.n * HL_TILE + mine;
            const CUtensorMap* const dmap = J.buf ? &dmap1 : &dmap0;
            const CUtensorMap *am, *bm;
            bool a_rows, b_rows;                           // the operand's rows are the tensor's rows (K-major), else its columns
            int ax, ay, bx, by;                            // at K = 0
            if (t.kind <= HL_DLOGITS) {
                am = &xmap; a_rows = true; ax = 0; ay = m0 + (t.kind == HL_STATS ? P.tok0 : 0);
                bm = &wmap; b_rows = true; bx = 0; by = J.v0 + n0;
            } else if (t.kind == HL_DX) {
                am = dmap; a_rows = true; ax = 0; ay = m0;
                bm = &wmap; b_rows = false; bx = n0; by = J.v0;
            } else {
                am = dmap; a_rows = false; ax = m0; ay = 0;
                bm = &xmap; b_rows = false; bx = n0; by = 0;
            }
            for (int k = t.k0; k < t.k1; ++k) {
                good = __all_sync(full_mask, mbar_wait_bounded<true>(bar_empty(s), ph ^ 1u, P.status, DEV_TIMEOUT_EMPTY));
                if (!good) break;
                const uint32_t bar = map_to_rank(bar_full(s), 0), dst = s0 + s * HL_STAGE_BYTES;
                const int kk = k * HL_KS;
                if (elect_one()) {
                    if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * HL_STAGE_BYTES);
                    const int x = a_rows ? ax + kk : ax, y = a_rows ? ay : ay + kk;
                    tma_load_2d<true>(dst, am, x, y, bar);
                    tma_load_2d<true>(dst + HL_BOX, am, a_rows ? x : x + 64, a_rows ? y + 64 : y, bar);
                    const int u = b_rows ? bx + kk : bx, v = b_rows ? by : by + kk;
                    tma_load_2d<true>(dst + 2 * HL_BOX, bm, u, v, bar);
                    tma_load_2d<true>(dst + 3 * HL_BOX, bm, b_rows ? u : u + 64, b_rows ? v + 64 : v, bar);
                }
                __syncwarp();
                if (++s == HL_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (rank == 0) {
        // =========================================================== MMA
        bool good = true;
        uint32_t s = 0, ph = 0, buf = 0, aph = 0;
        for (int i = pair; good && hl_tile(P, tokens, i, &t); i += pairs) {
            const bool a_mn = t.kind == HL_DW, b_mn = t.kind >= HL_DX;
            const uint32_t idesc = umma_idesc(HL_TILE, HL_TILE) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
            const uint64_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;
            const int per = t.kind <= HL_DLOGITS ? HL_SUM_STAGES : t.k1 - t.k0;
            for (int k0 = t.k0; good && k0 < t.k1; k0 += per) {
                good = __all_sync(full_mask, mbar_wait_bounded<true>(bar_free(buf), aph ^ 1u, P.status, DEV_TIMEOUT_EMPTY));
                if (!good) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * 256u;
                const int k1 = min(t.k1, k0 + per);
                for (int k = k0; k < k1; ++k) {
                    good = __all_sync(full_mask, mbar_wait_bounded<true>(bar_full(s), ph, P.status, DEV_TIMEOUT_FULL));
                    if (!good) break;
                    cluster_acquire();                     // the other CTA's half
                    tc_fence_after();
                    const uint32_t at = s0 + s * HL_STAGE_BYTES;
                    const uint64_t ad = a_mn ? umma_smem_desc_mn(at, HL_BOX) : umma_smem_desc(at);
                    const uint64_t bd = b_mn ? umma_smem_desc_mn(at + 2 * HL_BOX, HL_BOX) : umma_smem_desc(at + 2 * HL_BOX);
                    if (elect_one()) {
#pragma unroll
                        for (int q = 0; q < HL_KS / 16; ++q) umma_bf16<true>(d, ad + a_step * q, bd + b_step * q, idesc, (k > k0 || q > 0) ? 1u : 0u);
                        umma_commit<true>(bar_empty(s), 3);
                    }
                    __syncwarp();
                    if (++s == HL_STAGES) { s = 0; ph ^= 1u; }
                }
                if (good && elect_one()) umma_commit<true>(bar_acc(buf), 3);
                __syncwarp();
                buf ^= 1u;
                if (buf == 0) aph ^= 1u;
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();                                    // the pair frees its tensor memory together
    if (warp == HL_EPI_WARPS + 1) { tc_fence_after(); tmem_dealloc<true>(tmem, 512); }
}

// ----------------------------------------------------------------------------- before and after the products
struct HlPrepareParams {
    const uint16_t* x;
    long long ldx;
    const long long* targets;
    int n, hidden, per_block;
    long long vocab;
    int* count;                            // [0] tokens that count, [1] blocks of the last kernel that have finished
    int* slot;                             // [n] a token's place among those that count, or -1
    int* target;                           // [n] by place
    uint16_t* packed;                      // [n][hidden] by place
    const float2* stats;                   // backward: [n] maximum and log2 of the sum
    const float* grad;                     // gradient of the loss, of every token (grad_step 1) or of the sum or mean (0)
    int grad_step, mean;
    float4* row;                           // backward: [n] by place
    float* factor;                         // backward: what multiplies the sums
};

constexpr int HL_PREP_THREADS = 256;
// Tokens that count, packed in their order.  Every block counts those before its own for itself (the targets are a few KB, and in the L2).
__global__ void __launch_bounds__(HL_PREP_THREADS) head_prepare_kernel(const HlPrepareParams P) {
    __shared__ int before_s, total_s, slots_s[HL_PREP_THREADS], sums_s[HL_PREP_THREADS / 32];
    const int first = blockIdx.x * P.per_block, last = min(first + P.per_block, P.n);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) before_s = total_s = 0;
    __syncthreads();
    auto counts = [&](int i) { const long long t = P.targets[i]; return t >= 0 && t < P.vocab; };
    int before = 0, total = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < P.n; i += HL_PREP_THREADS) {
        const int c = counts(i) ? 1 : 0;
        total += c;
        if (i < first) before += c;
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before);
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    if (lane == 0) { atomicAdd(&before_s, before); atomicAdd(&total_s, total); }
    __syncthreads();
    total = total_s;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        P.count[0] = total;
        P.count[1] = 0;
        if (P.factor) *P.factor = P.grad_step ? 1.0f : P.mean ? P.grad[0] / (float)max(total, 1) : P.grad[0];
    }
    const int packs = P.hidden / 8;
    int base = before_s;
    for (int i0 = first; i0 < last; i0 += HL_PREP_THREADS) {
        const int i = i0 + (int)threadIdx.x;
        const bool in = i < last && counts(i);
        const unsigned ballot = __ballot_sync(0xFFFFFFFFu, in);
        if (lane == 0) sums_s[warp] = __popc(ballot);
        __syncthreads();
        int place = base + __popc(ballot & ((1u << lane) - 1u));
        for (int w = 0; w < HL_PREP_THREADS / 32; ++w) {
            if (w < warp) place += sums_s[w];
            base += sums_s[w];
        }
        slots_s[threadIdx.x] = in ? place : -1;
        if (i < last) P.slot[i] = in ? place : -1;
        if (in) {
            P.target[place] = (int)P.targets[i];
            if (P.row) {
                const float2 s = P.stats[i];
                P.row[place] = make_float4(s.x, s.y, P.grad_step ? P.grad[i] : 1.0f, 0.0f);
            }
        }
        __syncthreads();
        const int here = min(last - i0, HL_PREP_THREADS);
        for (int j = 0; j < here; ++j) {
            const int p = slots_s[j];
            if (p < 0) continue;
            const uint4* src = reinterpret_cast<const uint4*>(P.x + (long long)(i0 + j) * P.ldx);
            uint4* dst = reinterpret_cast<uint4*>(P.packed + (long long)p * P.hidden);
            for (int c = threadIdx.x; c < packs; c += HL_PREP_THREADS) dst[c] = src[c];
        }
        __syncthreads();
    }
    // the rest of the last tile of rows: products with it are never used, but they are with zeros of d
    const int end = min(P.n, (max(total, 1) + HL_TILE - 1) / HL_TILE * HL_TILE);
    for (int p = total + (int)blockIdx.x; p < end; p += gridDim.x)
        for (int c = threadIdx.x; c < packs; c += HL_PREP_THREADS) reinterpret_cast<uint4*>(P.packed + (long long)p * P.hidden)[c] = make_uint4(0, 0, 0, 0);
}

struct HlJoinParams {
    const float2* part;
    const float* at;
    const int* slot;
    int* count;
    int n, parts, ld_part, tok0, tokens;   // places tok0 .. tok0 + tokens are in `part`
    float* loss;                           // [n]
    float2* stats;                         // [n] or null
    float* total;                          // sum or mean, or null
    int mean;
};

constexpr int HL_JOIN_THREADS = 512, HL_JOIN_TOKENS = 8, HL_JOIN_SLICES = HL_JOIN_THREADS / HL_JOIN_TOKENS;
// The tiles' statistics of eight tokens, joined in a fixed order; the last block to finish adds up the losses.
__global__ void __launch_bounds__(HL_JOIN_THREADS) head_join_kernel(const HlJoinParams P) {
    __shared__ float m_s[HL_JOIN_SLICES][HL_JOIN_TOKENS], s_s[HL_JOIN_SLICES][HL_JOIN_TOKENS];
    __shared__ bool last_s;
    const int which = threadIdx.x % HL_JOIN_TOKENS, slice = threadIdx.x / HL_JOIN_TOKENS;
    const int i = blockIdx.x * HL_JOIN_TOKENS + which;
    const int p = i < P.n ? P.slot[i] : -1;
    const bool here = p >= P.tok0 && p < P.tok0 + P.tokens;
    float m = -INFINITY, s = 0.0f;
    if (here) {
        const float2* part = P.part + (p - P.tok0);
#pragma unroll 8
        for (int k = slice; k < P.parts; k += HL_JOIN_SLICES) {
            const float2 v = part[(long long)k * P.ld_part];
            const float top = fmaxf(m, v.x), base = top == -INFINITY ? 0.0f : top;
            s = s * exp2_fast((m - base) * LOG2E) + v.y * exp2_fast((v.x - base) * LOG2E);
            m = top;
        }
    }
    m_s[slice][which] = m;
    s_s[slice][which] = s;
    __syncthreads();
    for (int half = HL_JOIN_SLICES / 2; half > 0; half /= 2) {
        if (slice < half) {
            const float om = m_s[slice + half][which], os = s_s[slice + half][which];
            const float top = fmaxf(m, om), base = top == -INFINITY ? 0.0f : top;
            s = s * exp2_fast((m - base) * LOG2E) + os * exp2_fast((om - base) * LOG2E);
            m = top;
            m_s[slice][which] = m;
            s_s[slice][which] = s;
        }
        __syncthreads();
    }
    if (slice == 0 && i < P.n) {
        if (here) {
            P.loss[i] = (m - P.at[p]) + logf(s);
            if (P.stats) P.stats[i] = make_float2(m, log2f(s));
        } else if (p < 0) {
            P.loss[i] = 0.0f;
            if (P.stats) P.stats[i] = make_float2(0.0f, 0.0f);
        }
    }
    if (!P.total) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_s = atomicAdd(&P.count[1], 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    float* sum_s = &s_s[0][0];
    float sum = 0.0f;
    for (int k = threadIdx.x; k < P.n; k += HL_JOIN_THREADS) sum += __ldcg(P.loss + k);
    sum_s[threadIdx.x] = sum;
    __syncthreads();
    for (int half = HL_JOIN_THREADS / 2; half > 0; half /= 2) {
        if (threadIdx.x < half) sum_s[threadIdx.x] += sum_s[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x == 0) *P.total = P.mean ? sum_s[0] / (float)max(P.count[0], 1) : sum_s[0];
}

// dx of every token: the sum of its slabs times the factor that all share, or zeros
__global__ void __launch_bounds__(256) head_dx_kernel(const float* slab, const int* slot, int n_rows, int hidden, int splits, const float* factor, uint16_t* dx,
                                                    long long ld) {
    const int i = blockIdx.x, p = slot[i];
    const float g = *factor;
    for (int c = threadIdx.x * 8; c < hidden; c += 256 * 8) {
        float v[8] = {};
        if (p >= 0) {
            for (int s = 0; s < splits; ++s) {
                const float4* q = reinterpret_cast<const float4*>(slab + ((long long)s * n_rows + p) * hidden + c);
                const float4 a = q[0], b = q[1];
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            }
        }
        *reinterpret_cast<uint4*>(dx + (long long)i * ld + c) =
            p < 0 ? make_uint4(0, 0, 0, 0)
                  : make_uint4(pack_bf16x2(v[0] * g, v[1] * g), pack_bf16x2(v[2] * g, v[3] * g), pack_bf16x2(v[4] * g, v[5] * g), pack_bf16x2(v[6] * g, v[7] * g));
    }
}

}  // namespace cb
