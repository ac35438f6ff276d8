// Embedding lookup with a factor, y[n] = s * E[id[n]], and its gradient, dE[v] = s * sum over { n : id[n] = v } of dy[n].
//
// An id outside the table (-1: padding) reads zeros and takes part in no sum; its row of dy is not read.
//
// The gradient is dense and mostly zeros: what bounds it is writing them.  It goes by sorted tokens, so that every sum has one owner and one
// order (ascending n) and no atomics are needed:
//   1. blocks of 2048 ids sort (id, n) in shared memory, while all others write the zeros of the whole table;
//   2. more than one block: every element finds its place among all by binary searches in the other blocks' sorted ids;
//   3. tiles of 32 sorted tokens add up the rows of each run of equal ids (fp32) and write the table rows of runs that lie inside the tile;
//      what a run has in tiles that it leaves or enters goes to scratch, one row at either end of a tile;
//   4. one block per run that crosses tiles adds those rows in order.
// The zeros of rows that are overwritten in 3 and 4 are written twice: a few per cent of the table, for which the sort costs nothing.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

namespace cb {

constexpr int EMB_THREADS = 256;
constexpr int EG_BLOCK = 2048;             // ids that a block sorts
constexpr int EG_SORT_THREADS = 1024;
constexpr int EG_TILE = 32;                // sorted tokens of a tile
constexpr int EG_SUM_THREADS = 128;
constexpr uint32_t EG_NONE = 0xFFFFFFFFu;  // sorts behind every row

struct Bf16 { uint16_t v; };
struct Fp16 { uint16_t v; };

// N values of a type as they lie in memory, to fp32 and back (one rounding to nearest)
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(Bf16 x) { return bf16_to_float(x.v); }
__device__ __forceinline__ float value_of(Fp16 x) { return __half2float(__ushort_as_half(x.v)); }
__device__ __forceinline__ void set_value(float& d, float x) { d = x; }
__device__ __forceinline__ void set_value(Bf16& d, float x) { d.v = float_to_bf16(x); }
__device__ __forceinline__ void set_value(Fp16& d, float x) { d.v = __half_as_ushort(__float2half_rn(x)); }
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack { T v[N]; };

struct EmbedParams {
    const long long* ids;
    const void* table;
    void* out;
    long long n, ld, ld_out, n_rows;
    int chunks, threads_per_row;           // packs of a row; a power of two
    float scale;
    bool plain;                            // scale 1: bits are copied
};

// `threads_per_row` threads a token, four packs of each in flight
template <typename T, int N>
__global__ void __launch_bounds__(EMB_THREADS) embed_kernel(const EmbedParams P) {
    const int per = P.threads_per_row, lane = threadIdx.x & (per - 1);
    const long long t = (long long)blockIdx.x * (EMB_THREADS / per) + threadIdx.x / per;
    if (t >= P.n) return;
    const long long id = P.ids[t];
    const bool in = id >= 0 && id < P.n_rows;
    const Pack<T, N>* src = reinterpret_cast<const Pack<T, N>*>(reinterpret_cast<const T*>(P.table) + (in ? id : 0) * P.ld);
    Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(reinterpret_cast<T*>(P.out) + t * P.ld_out);
    for (int c = lane; c < P.chunks; c += 4 * per) {
        Pack<T, N> v[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && c + i * per < P.chunks) v[i] = src[c + i * per];
        if (!P.plain && in) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) set_value(v[i].v[e], value_of(v[i].v[e]) * P.scale);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i * per < P.chunks) dst[c + i * per] = v[i];
    }
}

struct EmbedGradParams {
    const long long* ids;
    const void* grad;
    void* out;                             // [n_rows][width], contiguous, 16-byte aligned
    long long n, ld, n_rows;
    int width, blocks, tiles;              // blocks of ids, tiles of sorted tokens
    float scale;
    uint32_t* block_ids;                   // [blocks][EG_BLOCK] sorted within each block
    uint32_t* block_pos;
    uint32_t* ids_sorted;                  // [n] (one block: the same memory as block_ids)
    uint32_t* pos_sorted;
    float* part;                           // [tiles][2][width]: what a tile has of the run that entered it, of the one that leaves it
};

// Step 1.  Bitonic sort of (id, n) in shared memory: unique keys, so the order of equal ids is that of the tokens.
__global__ void __launch_bounds__(EG_SORT_THREADS) embed_grad_sort_kernel(const EmbedGradParams P, long long out_bytes) {
    if ((int)blockIdx.x >= P.blocks) {                     // zeros
        uint4* out = reinterpret_cast<uint4*>(P.out);
        const long long packs = out_bytes / 16, step = (long long)(gridDim.x - P.blocks) * EG_SORT_THREADS;
        const long long first = (long long)(blockIdx.x - P.blocks) * EG_SORT_THREADS + threadIdx.x;
        for (long long i = first; i < packs; i += step) out[i] = make_uint4(0, 0, 0, 0);
        if (first < out_bytes % 16) reinterpret_cast<uint8_t*>(P.out)[packs * 16 + first] = 0;
        return;
    }
    __shared__ unsigned long long key[EG_BLOCK];
    const long long base = (long long)blockIdx.x * EG_BLOCK;
    const int here = (int)min((long long)EG_BLOCK, P.n - base);
    int size = 2;
    while (size < here) size *= 2;
    for (int i = threadIdx.x; i < size; i += EG_SORT_THREADS) {
        uint32_t id = EG_NONE;
        if (i < here) {
            const long long v = P.ids[base + i];
            if (v >= 0 && v < P.n_rows) id = (uint32_t)v;
        }
        key[i] = (unsigned long long)id << 32 | (uint32_t)i;
    }
    __syncthreads();
    for (int k = 2; k <= size; k *= 2) {
        for (int j = k / 2; j > 0; j /= 2) {
            for (int t = threadIdx.x; t < size / 2; t += EG_SORT_THREADS) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;
                const unsigned long long x = key[a], y = key[b];
                if ((x > y) == ((a & k) == 0)) { key[a] = y; key[b] = x; }
            }
            __syncthreads();
        }
    }
    for (int i = threadIdx.x; i < EG_BLOCK; i += EG_SORT_THREADS) {
        const bool in = i < here;
        if (!in && P.blocks == 1) break;
        P.block_ids[base + i] = in ? (uint32_t)(key[i] >> 32) : EG_NONE;
        if (in) P.block_pos[base + i] = (uint32_t)(base + (uint32_t)key[i]);
    }
}

// Step 2.  An element's place: its own in its block, plus how many of every other block come before it (equal ids: of earlier blocks).
__global__ void __launch_bounds__(256) embed_grad_place_kernel(const EmbedGradParams P) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= P.n) return;
    const int mine = (int)(i / EG_BLOCK);
    const uint32_t id = P.block_ids[i];
    long long place = i % EG_BLOCK;
#pragma unroll 4
    for (int b = 0; b < P.blocks; ++b) {
        const uint32_t* s = P.block_ids + (long long)b * EG_BLOCK;
        int below = 0;                                     // how many of s come before (id, mine)
#pragma unroll
        for (int step = EG_BLOCK / 2; step > 0; step /= 2) {
            const uint32_t v = s[below + step - 1];
            if (v < id || (v == id && b < mine)) below += step;
        }
        const uint32_t v = s[below];
        if (v < id || (v == id && b < mine)) ++below;
        if (b != mine) place += below;
    }
    if (place < P.n) {
        P.ids_sorted[place] = id;
        P.pos_sorted[place] = P.block_pos[i];
    }
}

// Step 3.
template <typename T, int N>
__global__ void __launch_bounds__(EG_SUM_THREADS) embed_grad_sum_kernel(const EmbedGradParams P) {
    __shared__ uint32_t id_s[EG_TILE + 2], pos_s[EG_TILE];
    const long long t0 = (long long)blockIdx.x * EG_TILE;
    const int here = (int)min((long long)EG_TILE, P.n - t0);
    for (int i = threadIdx.x; i < EG_TILE + 2; i += EG_SUM_THREADS) {       // the tile's ids and one on either side
        const long long at = t0 + i - 1;
        id_s[i] = at >= 0 && at < P.n ? P.ids_sorted[at] : EG_NONE;
        if (i < here) pos_s[i] = P.pos_sorted[t0 + i];
    }
    __syncthreads();
    const int col = ((int)blockIdx.y * EG_SUM_THREADS + (int)threadIdx.x) * N;
    if (col >= P.width) return;
    const T* grad = reinterpret_cast<const T*>(P.grad) + col;
    T* out = reinterpret_cast<T*>(P.out) + col;
    float* part = P.part + (long long)blockIdx.x * 2 * P.width + col;
    float sum[N] = {};
    bool entered = id_s[0] == id_s[1];                     // the run began in an earlier tile
    for (int i0 = 0; i0 < here; i0 += 8) {
        Pack<T, N> v[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < here && id_s[i0 + i + 1] != EG_NONE) v[i] = *reinterpret_cast<const Pack<T, N>*>(grad + (long long)pos_s[i0 + i] * P.ld);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= here) continue;
            const uint32_t id = id_s[i0 + i + 1];
            if (id == EG_NONE) return;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += value_of(v[i].v[e]);
            const bool last = i0 + i + 1 == here, ends = id_s[i0 + i + 2] != id;
            if (!last && !ends) continue;
            if (entered || !ends) {
                float* p = part + (entered ? 0 : P.width);
#pragma unroll
                for (int e = 0; e < N; ++e) p[e] = sum[e];
            } else {
                Pack<T, N> o;
#pragma unroll
                for (int e = 0; e < N; ++e) set_value(o.v[e], sum[e] * P.scale);
                *reinterpret_cast<Pack<T, N>*>(out + (long long)id * P.width) = o;
            }
            entered = false;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0.0f;
        }
    }
}

// Step 4.  A run that leaves tile a for the first time: its rows in the tiles a .. b.  Eight warps take a part of them each.
template <typename T>
__global__ void __launch_bounds__(256) embed_grad_join_kernel(const EmbedGradParams P) {
    const long long a = blockIdx.x, end = (a + 1) * EG_TILE;
    if (end >= P.n) return;
    const uint32_t id = P.ids_sorted[end - 1];
    if (id == EG_NONE || P.ids_sorted[end] != id) return;
    if (a > 0 && P.ids_sorted[end - EG_TILE] == id && P.ids_sorted[end - EG_TILE - 1] == id) return;      // it came from an earlier tile
    long long lo = end, hi = P.n;                          // first element behind the run
    while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (P.ids_sorted[mid] <= id) lo = mid + 1;
        else hi = mid;
    }
    const int rows = (int)((lo - 1) / EG_TILE - a);        // tiles that it enters
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = ((int)blockIdx.y * 32 + lane) * 4;
    __shared__ float sum_s[8][128];
    float sum[4] = {};
    const int first = (int)((long long)rows * warp / 8), last = (int)((long long)rows * (warp + 1) / 8);
    const float* part = P.part + (a + 1) * 2 * P.width + col;
#pragma unroll 4
    for (int r = first; r < last; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < P.width) sum[e] += part[(long long)r * 2 * P.width + e];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum_s[warp][lane * 4 + e] = sum[e];
    __syncthreads();
    const int c = (int)blockIdx.y * 128 + threadIdx.x;
    if (threadIdx.x >= 128 || c >= P.width) return;
    float total = P.part[a * 2 * P.width + P.width + c];
    for (int w = 0; w < 8; ++w) total += sum_s[w][threadIdx.x];
    T o;
    set_value(o, total * P.scale);
    reinterpret_cast<T*>(P.out)[(long long)id * P.width + c] = o;
}

}  // namespace cb
