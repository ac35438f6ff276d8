// Softmax cross entropy of hidden states against the rows of a head, l[n, v] = x[n] . W[v], loss[n] = log sum_v exp l[n, v] - l[n, t[n]], and
// its gradients, d = (softmax(l) - onehot(t)) * g, dx = d W, dW = d^T x, in pieces of the vocabulary: no more than a piece of l or d exists.
//
// One kernel does all four products.  A pair of CTAs holds a tile of 256 x 256 results (tcgen05.mma.cta_group::2, each CTA 128 rows of A and
// 128 columns of B per stage of 64, so that a stage costs an SM 32 KB for 512 clocks of MMA) and walks a list of tiles:
//   stats     A = x, B = W (both K-major): maximum and sum of exp of every row over the tile's columns, and the target's logit
//   dlogits   the same product again; d, rounded to bf16, goes to the piece's scratch [tokens][columns]
//   dx        A = d (K-major), B = W with the vocabulary as K (N-major as it lies): fp32 sums over the pieces, in slabs [split][token][hidden]
//   dw        A = d with the tokens as K (M-major as it lies), B = x the same: dW, rounded once
// Operands come by TMA in boxes of 64 columns, whatever their order: a box is rows of 128 swizzled bytes, and which of its sides is K is the
// descriptor's business.
//   warps 0-7  epilogue: warp w owns TMEM lanes 32 * (w % 4).. (a thread = a row) and columns 128 * (w / 4)..
//   warp 8     TMA         warp 9     MMA (of the pair's first CTA)        warps 10, 11     none: they fill a warpgroup
// An epilogue thread holds 128 sums.  The 168 registers that 384 threads have each do not hold them and what belongs to them, and what is
// spilled goes to the L2 (227 KB of shared memory leave little L1): warps 8-11 hand registers over, 216 to 72.  48 bytes a thread are spilled all the same (12 words;
// 148 bytes of stores and 432 of loads in the whole code).
// Two accumulators of 256 columns: the epilogue of a tile runs under the next one's products.
//
// What bounds it: the tensor pipe, and behind it the power limit.  Busy (profiler, one launch): logits 87 % (2047 tokens, 32000 x 4096) to 93 % (2048 tokens,
// 65536 x 5376), their gradient 85 %, both products 89 %, at 1.38 to 1.55 GHz.  2047 tokens of 32000 x 4096 take 370 us (1.45 PFLOP/s) in a short loop
// and 423 us (1.27 PFLOP/s) in a long one, where the library's own product of that size takes 398 us and keeps the logits.  The rest is the way from tile to
// tile: the first chunk waits for the accumulator, the last one for the epilogue of the tile before.
//
// Tokens without a target are left out beforehand (prepare kernel: targets and rows of x that count, packed in order), so a prompt that is not
// trained on costs nothing, and nothing in its rows, NaN included, reaches a sum.  How many count is known on the device alone; tiles behind
// them are not visited.
//
// Precision.  The tensor core cuts every product at its running sum's last bits, always towards zero: over 5376 columns that is 1e-5 of a
// logit, all in one direction.  So logits are summed in tensor memory over 512 columns at a time, and these sums in fp32 registers; gradients, which are
// rounded to bf16 in the end, over 4096 tokens or rows of the vocabulary at a time (all at once, dx over 2^19 rows was off by 1.3e-3 where sums of 0.8
// cancel).
// d is rounded to bf16 (2^-8 of an element at most, at random), because the tensor core multiplies two operands of one type: gradients are off by 1.8e-3 to
// 1.9e-3 in 2-norm (2.1e-3 for a few hundred tokens of small models), 1.7e-3 of it their own last rounding.  As hi + lo it would be 12 n V H operations
// instead of 8 here, where the tensor pipe is the bound; up to 64 tokens, where it is not, have both values (head_few.cuh).  A factor g that all tokens share
// stays out of d and multiplies the sums: -g + a little, rounded in the target's column of every token, would be off by the same for all of
// them, while -1 + a little is not (2048 columns, 5000 rows, 600 tokens, error in 2-norm with g inside 2.6e-3).
#pragma once
#include "staged_input.cuh"
#include "tcgen05.cuh"

namespace cb {

constexpr int HL_TILE = 256;               // rows and columns of a pair's tile
constexpr int HL_KS = 64;                  // K per stage
constexpr int HL_STAGES = 5, HL_LOGIT_STAGES = 7;         // of logits alone: nothing goes out by shared memory
constexpr uint32_t HL_BOX = 64 * 128;      // bytes of 64 rows x 64 bf16
constexpr uint32_t HL_STAGE_BYTES = 4 * HL_BOX;
constexpr int HL_EPI_WARPS = 8;
constexpr int HL_COLS = 128;               // columns of an epilogue warp
constexpr int HL_THREADS = HL_EPI_WARPS * 32 + 128;
constexpr int HL_REGS = 168, HL_EPI_REGS = 216, HL_ROLE_REGS = 72;     // of a thread: at the launch, epilogue, the others
static_assert(HL_EPI_REGS * HL_EPI_WARPS * 32 + HL_ROLE_REGS * 128 <= HL_REGS * HL_THREADS, "no more than the block was launched with");
constexpr int HL_SUM_STAGES = 8;           // stages of logits that are summed in tensor memory
constexpr int HL_GRAD_STAGES = 64;         // ... of gradients, whose results are rounded to bf16
constexpr uint32_t HL_OUT_BYTES = 32 * 128;                // results of a warp on their way out: 32 rows of 128 swizzled bytes, twice
constexpr uint32_t HL_SMEM = HL_STAGES * HL_STAGE_BYTES + HL_EPI_WARPS * 2 * HL_OUT_BYTES + 256 + 1024;
static_assert(HL_LOGIT_STAGES * HL_STAGE_BYTES <= HL_STAGES * HL_STAGE_BYTES + HL_EPI_WARPS * 2 * HL_OUT_BYTES && HL_LOGIT_STAGES <= 8, "room and barriers");
constexpr int HL_JOBS = 3;
constexpr float LOG2E = 1.44269504088896341f;

enum HlKind : int { HL_STATS = 0, HL_DLOGITS = 1, HL_DX = 2, HL_DW = 3 };

// Tiles of one product.  Tokens in tiles of 256 (their number comes from the device), the vocabulary of a piece, or hidden columns.
struct HlJob {
    int kind;
    int v0, cols;                          // piece of the vocabulary: its first row, and its rows inside the vocabulary
    int n_tiles;                           // tiles along B's side: of the piece (stats, dlogits) or of hidden columns (dx, dw)
    int width;                             // their columns: 256, of logits any multiple of 32 up to that (what the instruction of a pair takes)
    int splits;                            // dx: ranges of the piece that are summed in slabs of their own
    int add;                               // dx: the slabs hold the sums of earlier pieces
    int buf;                               // which of the two scratch pieces holds d
};

struct HlParams {
    HlJob job[HL_JOBS];
    int n_jobs;
    int stages;
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
    uint32_t* status;
};
struct HlMaps {
    CUtensorMap x, w, d[2];                // bf16, boxes of 64 x 64: operands whose rows are K
    CUtensorMap x_rows, w_rows, d_rows[2]; // 64 columns of 128 rows, of w half a tile's: operands whose columns are K
    CUtensorMap slab, dw;                  // results: fp32 [split][token][hidden], boxes of 32 x 32; bf16, boxes of 64 columns x 32 rows
};

struct HlTile { int m, n, split, k0, k1; };

// The tiles of a pair of CTAs, one after another.  Jobs follow one another, a job's tiles go round the pairs.  dx comes first, in few long tiles: the pairs
// that get one less than others take that many more tiles of dw, so that all end together (2458 tokens of 4096 x 32000, 160 tiles of
// dx on 74 pairs: 1012 -> 897 us for both products).
struct HlList {
    int pair, pairs, tokens, token_tiles;
    int job, next;                         // current job, and the number of the next tile that the pair takes of it
    HlJob J;                               // the job, in registers
    int m_tiles, tiles;
    int shift;                             // the pair's place in the round of the current job
    int extra, few_from, few;              // rounds that only the pairs from few_from on take part in, `few` of them
    // The last tile as (outer, base + inner): gradients of one range (token or row tile, hidden tile), logits (vocabulary tile, token tile of the group that
    // begins at `base`).  The next one is a step away; outer < 0: work it out from its number.
    int outer, inner, base, outers, inners, step_out, step_in;

    __device__ __forceinline__ HlList(const HlParams& P, int pair_, int pairs_, int tokens_) {
        pair = pair_; pairs = pairs_; tokens = tokens_;
        token_tiles = min(max((tokens - P.tok0 + HL_TILE - 1) / HL_TILE, 1), P.tok_tiles);
        next = 0;
        shift = pair;
        extra = few_from = 0;
        few = pairs;
        open(P, 0);
    }
    __device__ __forceinline__ void open(const HlParams& P, int j) {
        job = j;
        outer = -1;
        if (j < P.n_jobs) J = P.job[j];
        m_tiles = J.kind == HL_DW ? (J.cols + HL_TILE - 1) / HL_TILE : token_tiles;
        tiles = m_tiles * J.n_tiles * J.splits;
    }
    __device__ __forceinline__ int stages(const HlParams& P) const {
        return J.kind <= HL_DLOGITS ? (P.hidden + HL_KS - 1) / HL_KS : J.kind == HL_DX ? (J.cols + HL_KS - 1) / HL_KS / J.splits : max((tokens + HL_KS - 1) / HL_KS, 1);
    }
    __device__ __forceinline__ bool take(const HlParams& P, HlTile* t) {
        if (outer >= 0) {
            outer += step_out;
            inner += step_in;
            if (inner >= inners) { inner -= inners; ++outer; }
            if (outer < outers) {
                t->m = J.kind <= HL_DLOGITS ? base + inner : outer;
                t->n = J.kind <= HL_DLOGITS ? outer : inner;
                ++next;
                return true;
            }
            outer = -1;                                                // none is left, or in another group
        }
        while (job < P.n_jobs) {
            int i = tiles;
            if (next < extra) {
                if (pair >= few_from) i = pair - few_from + next * few;
                else next = extra;                                     // (not in these rounds)
            }
            if (next >= extra && next < tiles) i = extra * few + shift + (next - extra) * pairs;
            if (i < tiles) {
                place(P, i, t);
                if (next >= extra && (J.kind <= HL_DLOGITS || J.splits == 1)) {
                    outer = J.kind <= HL_DLOGITS ? t->n : t->m;
                    inner = J.kind <= HL_DLOGITS ? t->m - base : t->n;
                    if (J.kind > HL_DLOGITS) { outers = m_tiles; inners = J.n_tiles; }
                    step_out = pairs / inners;
                    step_in = pairs - step_out * inners;
                }
                ++next;
                return true;
            }
            // the next job: who is ahead, and by how many of its tiles
            const int rest = max(tiles - extra * few, 0) % pairs;      // places of the last round that were taken
            const int ahead = rest && J.kind == HL_DX ? stages(P) : 0;
            next = extra = 0;
            shift = shift >= rest ? shift - rest : shift - rest + pairs;       // the others go first
            open(P, job + 1);
            if (job < P.n_jobs && ahead) {
                few_from = rest;
                few = pairs - rest;
                const int each = stages(P);
                extra = min((ahead + each / 2) / each, tiles / few);
            }
        }
        return false;
    }
    // Tile i of a job.  Logits: tokens in groups of at most 12 tiles, so that a group's x stays in the L2 while the vocabulary streams by, once a
    // group; gradients: neighbours share the operand that is longer.
    __device__ __forceinline__ void place(const HlParams& P, int i, HlTile* t) {
        t->k0 = 0;
        t->split = 0;
        if (J.kind <= HL_DLOGITS) {
            const int groups = (token_tiles + 11) / 12, per = (token_tiles + groups - 1) / groups;
            const int g = i / (per * J.n_tiles), in = i - g * per * J.n_tiles;
            base = g * per;
            inners = min(per, token_tiles - base);
            outers = J.n_tiles;
            t->n = in / inners;
            t->m = base + in - t->n * inners;
            t->k1 = (P.hidden + HL_KS - 1) / HL_KS;
        } else if (J.kind == HL_DX) {
            const int ks = (J.cols + HL_KS - 1) / HL_KS, one = token_tiles * J.n_tiles, s = i / one, in = i - s * one;
            t->split = s;
            t->m = in / J.n_tiles;
            t->n = in - t->m * J.n_tiles;
            t->k0 = (int)((long long)ks * s / J.splits);
            t->k1 = (int)((long long)ks * (s + 1) / J.splits);
        } else {
            t->m = i / J.n_tiles;
            t->n = i - t->m * J.n_tiles;
            t->k1 = max((tokens + HL_KS - 1) / HL_KS, 1);
        }
    }
};

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }       // all but the last one
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// where the barriers of a block lie, from `bars` on: stage full, stage empty, accumulator complete, accumulator free
__device__ __forceinline__ uint32_t hl_full(uint32_t bars, uint32_t s) { return bars + 8u * s; }
__device__ __forceinline__ uint32_t hl_empty(uint32_t bars, uint32_t s) { return bars + 64u + 8u * s; }
__device__ __forceinline__ uint32_t hl_acc(uint32_t bars, uint32_t b) { return bars + 128u + 8u * b; }
__device__ __forceinline__ uint32_t hl_free(uint32_t bars, uint32_t b) { return bars + 144u + 8u * b; }

// Nothing may be on its way when a CTA ends, also where a wait gave up: a copy would land in the shared memory of the block that comes next, a product in its tensor
// memory.  `fills` stages were filled, one after another; each of the last `depth` has its barrier's latest phase.
template <bool CLUSTER>
__device__ __forceinline__ void hl_landed(uint32_t bars, uint32_t fills, uint32_t depth, uint32_t* status) {
    for (uint32_t i = fills > depth ? fills - depth : 0; i < fills; ++i) mbar_wait_bounded<CLUSTER>(hl_full(bars, i % depth), i / depth & 1u, status, DEV_TIMEOUT_FULL);
}
// A commit follows all products before it, so the one behind the last stage that was used, the `uses`th, is enough
template <bool CLUSTER>
__device__ __forceinline__ void hl_multiplied(uint32_t bars, uint32_t uses, uint32_t depth, uint32_t* status) {
    if (uses) mbar_wait_bounded<CLUSTER>(hl_empty(bars, (uses - 1) % depth), (uses - 1) / depth & 1u, status, DEV_TIMEOUT_ACC);
}

// The warp that loads the operands, both CTAs each its half; the bytes of both are counted on the first one's barrier
struct HlLoad {
    uint32_t s0, bars, first_full, rank, depth;            // depth: how many stages there are
    uint32_t* status;
    uint32_t s, ph;                                        // stage that comes next, and its phase
    uint32_t fills;                                        // how many were filled
    bool ready;                                            // the stage was seen empty

    template <bool A_MN, bool B_MN>
    __device__ __forceinline__ bool tile(const CUtensorMap* a, int ax, int ay, const CUtensorMap* b, int bx, int by, int stages, uint32_t bytes) {
        const uint32_t full_mask = 0xFFFFFFFFu;
        for (int k = 0; k < stages; ++k) {
            if (!ready && !__all_sync(full_mask, mbar_wait_bounded<true>(hl_empty(bars, s), ph ^ 1u, status, DEV_TIMEOUT_EMPTY))) return false;
            const uint32_t next = s + 1 == depth ? 0 : s + 1, next_ph = next ? ph : ph ^ 1u;
            const bool seen = mbar_test_cluster(hl_empty(bars, next), next_ph ^ 1u);
            const uint32_t dst = s0 + s * HL_STAGE_BYTES, bar = first_full + 8u * s;
            if (elect_one()) {
                if (rank == 0) mbar_arrive_expect_tx(hl_full(bars, s), bytes);
                tma_load_2d<true>(dst, a, ax, ay, bar);
                if (A_MN) tma_load_2d<true>(dst + HL_BOX, a, ax + 64, ay, bar);
                tma_load_2d<true>(dst + 2 * HL_BOX, b, bx, by, bar);
                if (B_MN) tma_load_2d<true>(dst + 3 * HL_BOX, b, bx + 64, by, bar);
            }
            __syncwarp();
            ready = __all_sync(full_mask, seen);
            (A_MN ? ay : ax) += HL_KS;
            (B_MN ? by : bx) += HL_KS;
            ++fills;
            s = next;
            ph = next_ph;
        }
        return true;
    }
};

// The warp that issues the MMAs.  A stage is 512 clocks of MMA, and its wait, four MMAs and commit one after another took 630: so the next stage's
// barrier is asked before the MMAs of this one are issued (without waiting), and the order of the operands is known at compile time
// (descriptors differ in their low words alone).
struct HlIssue {
    uint32_t s0, bars, tmem, depth;
    uint32_t* status;
    uint32_t s, ph, buf, aph;                              // stage and accumulator that come next, and their phases
    uint32_t uses;                                         // how many stages were used
    bool ready;                                            // the stage was seen full

    template <bool A_MN, bool B_MN>
    __device__ __forceinline__ bool tile(int stages, int per, uint32_t width) {
        const uint32_t full_mask = 0xFFFFFFFFu;
        const uint32_t idesc = umma_idesc(width, HL_TILE) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
        constexpr uint32_t A_STEP = A_MN ? 2048 >> 4 : 32 >> 4, B_STEP = B_MN ? 2048 >> 4 : 32 >> 4;
        for (int k0 = 0; k0 < stages; k0 += per) {
            if (!__all_sync(full_mask, mbar_wait_bounded<true>(hl_free(bars, buf), aph ^ 1u, status, DEV_TIMEOUT_EMPTY))) return false;
            tc_fence_after();
            const uint32_t d = tmem + buf * 256u;
            for (int k = k0; k < min(stages, k0 + per); ++k) {
                if (!ready && !__all_sync(full_mask, mbar_wait_bounded<true>(hl_full(bars, s), ph, status, DEV_TIMEOUT_FULL))) return false;
                cluster_acquire();                         // the other CTA's half
                tc_fence_after();
                const uint32_t next = s + 1 == depth ? 0 : s + 1, next_ph = next ? ph : ph ^ 1u;
                const bool seen = mbar_test_cluster(hl_full(bars, next), next_ph);
                const uint32_t at = (s0 >> 4) + s * (HL_STAGE_BYTES >> 4);
                const uint32_t a = at | (A_MN ? (HL_BOX >> 4) << 16 : 1u << 16), b = (at + (2 * HL_BOX >> 4)) | (B_MN ? (HL_BOX >> 4) << 16 : 1u << 16);
                if (elect_one()) {
#pragma unroll
                    for (int q = 0; q < HL_KS / 16; ++q) umma_low<true>(d, a + A_STEP * q, b + B_STEP * q, idesc, (k > k0 || q > 0) ? 1u : 0u);
                    umma_commit<true>(hl_empty(bars, s), 3);
                }
                __syncwarp();
                ++uses;
                ready = __all_sync(full_mask, seen);
                s = next;
                ph = next_ph;
            }
            if (elect_one()) umma_commit<true>(hl_acc(bars, buf), 3);
            __syncwarp();
            buf ^= 1u;
            if (buf == 0) aph ^= 1u;
        }
        return true;
    }
};

__global__ void __launch_bounds__(HL_THREADS, 1) head_product_kernel(const __grid_constant__ HlParams P, const __grid_constant__ HlMaps M) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full_mask = 0xFFFFFFFFu;
    const uint32_t s0 = (smem_u32(smem) + 1023u) & ~1023u;
    const uint32_t outs = s0 + HL_STAGES * HL_STAGE_BYTES, bars = outs + HL_EPI_WARPS * 2 * HL_OUT_BYTES;
    const uint32_t tmem_slot = bars + 160u;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < (uint32_t)P.stages; ++s) { mbar_init(hl_full(bars, s), 1); mbar_init(hl_empty(bars, s), 1); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(hl_acc(bars, b), 1); mbar_init(hl_free(bars, b), 2 * HL_EPI_WARPS); }
        mbar_fence_init();
        fence_proxy_async();
    }
    if (warp == HL_EPI_WARPS + 1) { tmem_alloc<true>(tmem_slot, 512); tmem_relinquish<true>(); }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();                                    // the other CTA's barriers are in place before anyone arrives on them
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);
    pdl_next();
    pdl_wait();
    const int tokens = *P.count;
    HlList list(P, pair, pairs, tokens);
    HlTile t;

    if (warp < HL_EPI_WARPS) {
        // =========================================================== epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(HL_EPI_REGS));
        const int part = warp >> 2;                        // which columns of the tile
        const uint32_t my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)part * HL_COLS;
        const int my_row = (int)rank * 128 + (warp & 3) * 32 + lane, my_col = part * HL_COLS;
        const uint32_t out = outs + (uint32_t)warp * 2 * HL_OUT_BYTES, my_out = out + (uint32_t)lane * 128u;
        const uint32_t x7 = (uint32_t)(lane & 7);
        const float factor = P.factor ? *P.factor : 0.0f;
        bool healthy = true;
        uint32_t buf = 0, ph = 0, side = 0;                // which accumulator comes next, and which half of `out`
        auto wait_acc = [&]() {
            if (healthy) healthy = __all_sync(full_mask, mbar_wait_bounded<true>(hl_acc(bars, buf), ph, P.status, DEV_TIMEOUT_ACC));
            tc_fence_after();
        };
        auto free_acc = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && healthy) mbar_arrive_cluster(map_to_rank(hl_free(bars, buf), 0));
            buf ^= 1u;
            if (buf == 0) ph ^= 1u;
        };
        float acc[HL_COLS];
        auto spoil = [&]() {                               // a wait gave up: everything that this tile feeds becomes NaN
            if (healthy) return;
#pragma unroll
            for (int e = 0; e < HL_COLS; ++e) acc[e] = __uint_as_float(0x7FC00000u);
        };
        auto take_columns = [&]() {                        // the accumulator's columns
            wait_acc();
            uint32_t(&v)[4][32] = *reinterpret_cast<uint32_t(*)[4][32]>(&acc);
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(my_tmem + buf * 256u + 32u * q, v[q]);
            tmem_ld_wait();
            free_acc();
        };
        auto add_columns = [&]() {                         // on top of what there is
            wait_acc();
#pragma unroll
            for (int q = 0; q < HL_COLS; q += 32) {
                uint32_t v[32];
                tmem_ld32(my_tmem + buf * 256u + (uint32_t)q, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[q + e] += __uint_as_float(v[e]);
            }
            free_acc();
        };
        while (list.take(P, &t)) {
            const HlJob& J = list.J;
            const int row = t.m * HL_TILE + my_row, col = t.n * J.width + my_col;
            if (J.kind <= HL_DLOGITS) {
                const int r = J.kind == HL_STATS ? P.tok0 + row : row;
                // what a row of logits needs; requested under the products
                int target = -1;
                float4 rowv = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r < tokens) {
                    target = P.target[r] - J.v0 - col;
                    if (J.kind == HL_DLOGITS) rowv = P.row[r];
                }
                take_columns();
                for (int k = t.k0 + HL_SUM_STAGES; k < t.k1; k += HL_SUM_STAGES) add_columns();
                spoil();
                int here = min(J.width - my_col, HL_COLS);             // columns of this warp that are the tile's
                if (J.kind == HL_DLOGITS) here = min(here, P.ld_d - col);
                const int valid = min(here, J.cols - col);             // ... and inside the vocabulary
                if (target >= here) target = -1;
                if (J.kind == HL_STATS) {
                    if (valid < HL_COLS) {
#pragma unroll
                        for (int q = 0; q < HL_COLS; ++q)
                            if (q >= valid) acc[q] = -INFINITY;
                    }
                    float m[4] = {acc[0], acc[1], acc[2], acc[3]};
#pragma unroll
                    for (int q = 4; q < HL_COLS; ++q) m[q & 3] = fmaxf(m[q & 3], acc[q]);
                    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), base = top == -INFINITY ? 0.0f : top;
                    if (__any_sync(full_mask, target >= 0)) {
                        float own = 0.0f;
#pragma unroll
                        for (int q = 0; q < HL_COLS; ++q) own = q == target ? acc[q] : own;
                        if (target >= 0) P.at[r] = own;
                    }
                    // (the difference first: the product of a large logit with log2(e) would be rounded where the difference is exact)
                    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 0; q < HL_COLS; ++q) s[q & 3] += exp2_fast((acc[q] - base) * LOG2E);
                    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
                    P.part[(long long)(2 * t.n + part) * P.ld_part + row] = make_float2(top, sum);
                } else if (row < P.n_rows) {
                    const int kept = row < tokens ? valid : 0;
                    uint16_t* dst = P.d[J.buf] + (long long)row * P.ld_d + col;
#pragma unroll
                    for (int q = 0; q < HL_COLS; q += 16) {
                        if (q >= here) continue;
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float p[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int c = q + 2 * e + h;
                                p[h] = exp2_fast(fmaf(acc[c] - rowv.x, LOG2E, -rowv.y));
                                if (c == target) p[h] -= 1.0f;
                                p[h] = c < kept ? p[h] * rowv.z : 0.0f;
                            }
                            w[e] = pack_bf16x2(p[0], p[1]);
                        }
                        store32(dst + q, w);
                    }
                }
            } else {                                       // (a copy of its own: shared with the logits it spills, dw of 16 tokens 55 -> 68 us)
                take_columns();
                for (int k = t.k0 + HL_GRAD_STAGES; k < t.k1; k += HL_GRAD_STAGES) add_columns();
                spoil();
                if (col >= P.hidden) continue;
                // out by the copy engine, over shared memory: 64 columns of dw at a time; 32 of dx, which it adds up: one addition a piece, in their order
                if (J.kind == HL_DX) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (col + 32 * q >= P.hidden) continue;
                        if (lane == 0) bulk_wait_read();               // the last copy but one is out of here
                        __syncwarp();
                        const float* v = acc + 32 * q;
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            sts128(my_out + side + (((uint32_t)c ^ x7) << 4), __float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]), __float_as_uint(v[4 * c + 2]),
                                   __float_as_uint(v[4 * c + 3]));
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            if (J.add) tma_add_3d(&M.slab, out + side, col + 32 * q, row, t.split);
                            else tma_store_3d(&M.slab, out + side, col + 32 * q, row, t.split);
                            bulk_commit();
                        }
                        side ^= HL_OUT_BYTES;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (col + 64 * q >= P.hidden) continue;
                        if (lane == 0) bulk_wait_read();
                        __syncwarp();
                        const float* v = acc + 64 * q;
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            sts128(my_out + side + (((uint32_t)c ^ x7) << 4), pack_bf16x2(v[8 * c] * factor, v[8 * c + 1] * factor),
                                   pack_bf16x2(v[8 * c + 2] * factor, v[8 * c + 3] * factor), pack_bf16x2(v[8 * c + 4] * factor, v[8 * c + 5] * factor),
                                   pack_bf16x2(v[8 * c + 6] * factor, v[8 * c + 7] * factor));
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&M.dw, out + side, col + 64 * q, J.v0 + row);
                            bulk_commit();
                        }
                        side ^= HL_OUT_BYTES;
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_all();
    } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(HL_ROLE_REGS));
    if (warp == HL_EPI_WARPS) {
        // =========================================================== TMA
        HlLoad L = {s0, bars, map_to_rank(hl_full(bars, 0), 0), rank, (uint32_t)P.stages, P.status, 0, 0, 0, false};
        bool good = true;
        const int mine = (int)rank * 128;
        while (good && list.take(P, &t)) {
            const HlJob& J = list.J;
            const int m0 = t.m * HL_TILE + mine, n0 = t.n * J.width + (int)rank * (J.width / 2), k0 = t.k0 * HL_KS, stages = t.k1 - t.k0;
            const uint32_t bytes = 2 * (2 * HL_BOX + (uint32_t)J.width * 64u);             // of both CTAs
            if (J.kind <= HL_DLOGITS) good = L.tile<false, false>(&M.x_rows, k0, m0 + (J.kind == HL_STATS ? P.tok0 : 0), &M.w_rows, k0, J.v0 + n0, stages, bytes);
            else if (J.kind == HL_DX) good = L.tile<false, true>(&M.d_rows[J.buf], k0, m0, &M.w, n0, J.v0 + k0, stages, bytes);
            else good = L.tile<true, true>(&M.d[J.buf], m0, k0, &M.x, n0, k0, stages, bytes);
        }
        // (the first CTA's barriers count the copies of both, and neither ends before the other)
        if (rank == 0) hl_landed<true>(bars, L.fills, L.depth, P.status);
    } else if (warp == HL_EPI_WARPS + 1 && rank == 0) {
        // =========================================================== MMA
        HlIssue I = {s0, bars, tmem, (uint32_t)P.stages, P.status, 0, 0, 0, 0, 0, false};
        bool good = true;
        while (good && list.take(P, &t)) {
            const int kind = list.J.kind, stages = t.k1 - t.k0;
            const uint32_t width = (uint32_t)list.J.width;
            good = kind <= HL_DLOGITS ? I.tile<false, false>(stages, HL_SUM_STAGES, width) : kind == HL_DX ? I.tile<false, true>(stages, HL_GRAD_STAGES, width)
                                                                                                         : I.tile<true, true>(stages, HL_GRAD_STAGES, width);
        }
        hl_multiplied<true>(bars, I.uses, I.depth, P.status);
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
    pdl_next();
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
    const int* slot;                       // null: every token is at its own place, and counts if its target is inside the vocabulary
    const long long* targets;
    long long vocab;
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
    pdl_next();
    pdl_wait();
    __shared__ float m_s[HL_JOIN_SLICES][HL_JOIN_TOKENS], s_s[HL_JOIN_SLICES][HL_JOIN_TOKENS];
    __shared__ bool last_s;
    const int which = threadIdx.x % HL_JOIN_TOKENS, slice = threadIdx.x / HL_JOIN_TOKENS;
    const int i = blockIdx.x * HL_JOIN_TOKENS + which;
    int p = -1;
    if (i < P.n) {
        if (P.slot) {
            p = P.slot[i];
        } else {
            const long long t = P.targets[i];
            if (t >= 0 && t < P.vocab) p = i;
        }
    }
    const bool here = p >= P.tok0 && p < P.tok0 + P.tokens;
    float m = -INFINITY, s = 0.0f;
    const float own = here && slice == 0 ? P.at[p] : 0.0f; // (asked for early)
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
            P.loss[i] = (m - own) + logf(s);
            if (P.stats) P.stats[i] = make_float2(m, log2f(s));
        } else if (p < 0) {
            P.loss[i] = 0.0f;
            if (P.stats) P.stats[i] = make_float2(0.0f, 0.0f);
        }
    }
    if (!P.total) return;
    if (gridDim.x > 1) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last_s = atomicAdd(&P.count[1], 1) == (int)gridDim.x - 1;
        __syncthreads();
        if (!last_s) return;
        __threadfence();
    }
    __syncthreads();
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

// dx of every token: the sum of its slabs times the factor that all share, or zeros.  A thread has eight columns.  Without slots every token is at its own
// place, and counts if its target is inside the vocabulary.
constexpr int HL_DX_THREADS = 256;
__global__ void __launch_bounds__(HL_DX_THREADS) head_dx_kernel(const float* slab, const int* slot, const long long* targets, long long vocab, int n_rows, int hidden,
                                                               int splits, const float* factor, uint16_t* dx, long long ld) {
    pdl_next();
    pdl_wait();
    const int i = blockIdx.x, c = ((int)blockIdx.y * HL_DX_THREADS + (int)threadIdx.x) * 8;
    const int p = slot ? slot[i] : targets[i] >= 0 && targets[i] < vocab ? i : -1;
    if (c >= hidden) return;
    const float g = *factor;
    float v[8] = {};
    if (p >= 0) {
#pragma unroll 8
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

}  // namespace cb
