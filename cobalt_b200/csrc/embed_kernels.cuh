// Embedding lookup with a factor, y[n] = s * E[id[n]], and its gradient, dE[v] = s * sum over { n : id[n] = v } of dy[n].
//
// An id outside the table (-1: padding) reads zeros and takes part in no sum; its row of dy is not read.
//
// Lookup: bound by memory.  32 bytes a thread, converted in pairs: 8192 rows of 5376 bf16 values in 25.8 us, 176 MB at 6.8 TB/s; a value
// at a time with 16-byte loads took 50 us.  Rows off 16-byte boundaries go a value at a time: 8192 of 5375 bf16 values 98 us, 8192 of 1001 fp32 values 20.5
// (of 1000: 9.7).
//
// The gradient is dense and mostly zeros: what bounds it is writing them.  It goes by sorted tokens, so that every sum has one owner and one fixed
// order, which the ids alone decide, and no atomics on values are needed:
//   1. up to 6144 tokens (unless one block sorts them while a large table is cleared): every element finds its place among the sorted ones by
//      counting those before it, while all other blocks write zeros to the whole table;
//      more: blocks of 2048 ids sort (id, n) in registers and shared memory beside the zeros, and
//   2. every element finds its place among those of 16 blocks by binary searches in the others' sorted ids (the rest of the zeros is written beside
//      it), then among those of 256 blocks, and so on;
//   3. tiles of 16 sorted tokens add up the rows of each run of equal ids (fp32) and write the table rows of runs that lie inside the tile;
//      what a run has in tiles that it leaves or enters goes to scratch, one row at either end of a tile, and the tile where it begins to a list;
//   4. the runs of the list add those rows in order, runs of more than 64 of them in eight ranges first.
// So a row's sum is one of fp32 partial sums over up to 16 tokens each (fewer at either end), in the tokens' order, not one chain through all of them.
// The zeros of rows that are overwritten in 3 and 4 are written twice: a few per cent of the table, for which sorting costs nothing.
// Zeros go out as one 32-byte store a thread of blocks that hold 32 KB each: 7.5 TB/s over 2.8 GB, where a grid that strides over the table
// reaches 6.2 TB/s whatever the width of its stores (bulk copies from shared memory: 6.3).  16384 tokens of a table of 262144 x 5376: 438 us, of which
// 385 write zeros, 60 add up; 2047 of 32000 x 4096: 48 us, 36 of them zeros.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"
#include "staged_input.cuh"

namespace cb {

constexpr int EMB_THREADS = 256;
constexpr int EG_BLOCK = 2048;             // ids that a block sorts
constexpr int EG_SORT_THREADS = 1024;
constexpr int EG_TILE = 16;                // sorted tokens of a tile
constexpr int EG_JOIN_GRID = 256;          // blocks along the list of runs that cross tiles
constexpr int EG_JOIN_THREADS = 256, EG_JOIN_COLS = 4 * EG_JOIN_THREADS;
constexpr int EG_PLACE_THREADS = 256;
constexpr int EG_GROUP = 16;               // sorted runs that become one in a step
constexpr int EG_SUM_THREADS = 128;
constexpr int EG_RANK = 6144, EG_RANK_THREADS = 1024, EG_RANK_IDS = 32;     // tokens that are placed by counting, and how many a block
constexpr uint32_t EG_NONE = 0xFFFFFFFFu;  // sorts behind every row

struct Bf16 { uint16_t v; };
struct Fp16 { uint16_t v; };

// A 32-bit word of a type's values as they lie in memory: to fp32 and back (one rounding to nearest), and single values
template <typename T> constexpr int PER_WORD = 4 / sizeof(T);
__device__ __forceinline__ void word_values(Bf16, uint32_t w, float* v) { v[0] = __uint_as_float(w << 16); v[1] = __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ void word_values(Fp16, uint32_t w, float* v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    v[0] = f.x; v[1] = f.y;
}
__device__ __forceinline__ void word_values(float, uint32_t w, float* v) { v[0] = __uint_as_float(w); }
__device__ __forceinline__ uint32_t word_of(Bf16, const float* v) { return pack_bf16x2(v[0], v[1]); }
__device__ __forceinline__ uint32_t word_of(Fp16, const float* v) {
    const __half2 h = __floats2half2_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t word_of(float, const float* v) { return __float_as_uint(v[0]); }
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(Bf16 x) { return bf16_to_float(x.v); }
__device__ __forceinline__ float value_of(Fp16 x) { return __half2float(__ushort_as_half(x.v)); }
__device__ __forceinline__ void set_value(float& d, float x) { d = x; }
__device__ __forceinline__ void set_value(Bf16& d, float x) { d.v = float_to_bf16(x); }
__device__ __forceinline__ void set_value(Fp16& d, float x) { d.v = __half_as_ushort(__float2half_rn(x)); }

// W words of a row at a time (rows on such boundaries), or a value (W = 0)
template <typename T, int W> constexpr int PACK = W ? W * PER_WORD<T> : 1;
template <typename T, int W>
struct Pack {
    uint32_t w[W];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (W == 8) {
            asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
        } else {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (W == 8)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
        else
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void values(float (&v)[PACK<T, W>]) const {
#pragma unroll
        for (int i = 0; i < W; ++i) word_values(T{}, w[i], v + i * PER_WORD<T>);
    }
    __device__ __forceinline__ void set(const float (&v)[PACK<T, W>], float scale) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float x[PER_WORD<T>];
#pragma unroll
            for (int e = 0; e < PER_WORD<T>; ++e) x[e] = v[i * PER_WORD<T> + e] * scale;
            w[i] = word_of(T{}, x);
        }
    }
};
template <typename T>
struct Pack<T, 0> {
    T x;
    __device__ __forceinline__ void clear() { x = T{}; }
    __device__ __forceinline__ void load(const T* p) { x = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = x; }
    __device__ __forceinline__ void values(float (&v)[1]) const { v[0] = value_of(x); }
    __device__ __forceinline__ void set(const float (&v)[1], float scale) { set_value(x, v[0] * scale); }
};

struct EmbedParams {
    const long long* ids;
    const void* table;
    void* out;
    long long n, ld, ld_out, n_rows;
    int chunks, threads_per_row;           // packs of a row; a power of two
    float scale;
    bool plain;                            // scale 1: bits are copied
    uint32_t* status;                      // or null
};

// `threads_per_row` threads a token
template <typename T, int W>
__global__ void __launch_bounds__(EMB_THREADS) embed_kernel(const EmbedParams P) {
    const int per = P.threads_per_row, lane = threadIdx.x & (per - 1);
    const long long t = (long long)blockIdx.x * (EMB_THREADS / per) + threadIdx.x / per;
    if (t >= P.n) return;
    const long long id = P.ids[t];
    const bool in = id >= 0 && id < P.n_rows;
    if (id >= P.n_rows && lane == 0 && P.status) atomicCAS(P.status, 0u, (uint32_t)DEV_OUTSIDE);
    const T* src = reinterpret_cast<const T*>(P.table) + (in ? id : 0) * P.ld;
    T* dst = reinterpret_cast<T*>(P.out) + t * P.ld_out;
    for (int c = lane; c < P.chunks; c += per) {
        Pack<T, W> v;
        v.clear();
        if (in) {
            v.load(src + c * PACK<T, W>);
            if (!P.plain) {
                float x[PACK<T, W>];
                v.values(x);
                v.set(x, P.scale);
            }
        }
        v.store(dst + c * PACK<T, W>);
    }
}

struct EmbedGradParams {
    const long long* ids;
    const void* grad;
    void* out;                             // [n_rows][width], contiguous, 16-byte aligned
    long long n, ld, n_rows;
    int width, blocks, tiles;              // blocks of ids, tiles of sorted tokens
    int join_blocks;                       // step 4: blocks along the list
    float scale;
    uint32_t* block_ids;                   // [n] sorted within blocks of EG_BLOCK, or all of them
    uint32_t* block_pos;
    const uint32_t* ids_sorted;            // [n] (one block, or placed by counting: the same memory as block_ids)
    const uint32_t* pos_sorted;
    float* part;                           // [tiles][2][width]: what a tile has of the run that entered it, of the one that leaves it
    uint32_t* runs;                        // [0]: number of runs that cross tiles, [1..]: the tiles where they begin
    long long out_bytes, zero_first;       // of them, those that are cleared beside the sort; the rest beside step 2
};

constexpr int EG_ZERO_BYTES = 32 * EG_SORT_THREADS;        // of a block
// block `b` of those that clear the bytes [from, to), EG_ZERO_BYTES each; `from` is a multiple of 32
template <int THREADS>
__device__ __forceinline__ void embed_grad_zero(const EmbedGradParams& P, long long b, long long from, long long to) {
#pragma unroll
    for (int step = 0; step < EG_ZERO_BYTES / 32 / THREADS; ++step) {
        const long long at = from + b * EG_ZERO_BYTES + (step * THREADS + (int)threadIdx.x) * 32;
        uint8_t* p = reinterpret_cast<uint8_t*>(P.out) + at;
        if (at + 32 <= to && !((uintptr_t)p & 31)) {
            asm volatile("st.global.v8.b32 [%0], {%1,%1,%1,%1,%1,%1,%1,%1};" ::"l"(p), "r"(0) : "memory");
        } else {
            for (int i = 0; i < 32 && at + i < to; i += 16) {
                if (at + i + 16 <= to) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
                else
                    for (int k = i; at + k < to; ++k) p[k] = 0;        // the last bytes of the table
            }
        }
    }
}

// Steps 1 and 2 at once, of up to EG_RANK tokens: an element's place is how many come before it, counted by comparing it with all: n^2 comparisons on all SMs
// are less than the chain of a sort's steps on one, and a launch less (1500 tokens of 10007 x 333 fp32: 17.9 -> 11.8 us, 3000 of 20000 x 256: 23.5 -> 13.8, 6000 of
// 32000 x 1024: 30.7 -> 24.5; 8192 of 32000 x 4096 69.5 -> 73.6).  A block places 32 elements, one a lane; its warps each look through a
// share of the ids.
__global__ void __launch_bounds__(EG_RANK_THREADS) embed_grad_rank_kernel(const EmbedGradParams P, int rank_blocks) {
    if ((int)blockIdx.x >= rank_blocks) {
        embed_grad_zero<EG_RANK_THREADS>(P, blockIdx.x - rank_blocks, 0, P.out_bytes);
        return;
    }
    constexpr int SLICES = EG_RANK_THREADS / 32;
    __shared__ alignas(16) uint32_t id_s[EG_RANK];
    __shared__ int count_s[SLICES][EG_RANK_IDS];
    const int n = (int)P.n, padded = (n + 3) & ~3, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && threadIdx.x == 0) P.runs[0] = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < padded; i += EG_RANK_THREADS) {
        const long long v = i < n ? P.ids[i] : -1;
        id_s[i] = v >= 0 && v < P.n_rows ? (uint32_t)v : EG_NONE;
    }
    __syncthreads();
    const int e0 = (int)blockIdx.x * EG_RANK_IDS, e1 = e0 + EG_RANK_IDS;
    const int slice = (padded / 4 + SLICES - 1) / SLICES * 4, j0 = min(warp * slice, padded), j1 = min(j0 + slice, padded);
    const int at = e0 + lane;
    const uint32_t mine = id_s[min(at, padded - 1)];
    int before = 0;
    auto four = [&](int j, auto f) {
        const uint4 v = *reinterpret_cast<const uint4*>(id_s + j);
        before += (f(v.x, j) ? 1 : 0) + (f(v.y, j + 1) ? 1 : 0) + (f(v.z, j + 2) ? 1 : 0) + (f(v.w, j + 3) ? 1 : 0);
    };
    // earlier tokens come before equal ids, later ones do not (e0 and e1 are multiples of four)
#pragma unroll 8
    for (int j = j0; j < min(j1, e0); j += 4) four(j, [&](uint32_t v, int) { return v <= mine; });
    for (int j = max(j0, e0); j < min(j1, e1); j += 4) four(j, [&](uint32_t v, int k) { return v < mine || (v == mine && k < at); });
#pragma unroll 8
    for (int j = max(j0, e1); j < j1; j += 4) four(j, [&](uint32_t v, int) { return v < mine; });
    count_s[warp][lane] = before;
    __syncthreads();
    const int i = e0 + (int)threadIdx.x;
    if (threadIdx.x < EG_RANK_IDS && i < n) {
        int place = 0;
#pragma unroll
        for (int w = 0; w < SLICES; ++w) place += count_s[w][threadIdx.x];
        P.block_ids[place] = id_s[i];
        P.block_pos[place] = i;
    }
}

// Step 1.  Bitonic sort of the keys (id, n): unique, so the order of equal ids is that of the tokens.  A thread holds two neighbouring elements;
// partners up to 32 apart are in its warp, others meet in shared memory.
__global__ void __launch_bounds__(EG_SORT_THREADS) embed_grad_sort_kernel(const EmbedGradParams P) {
    if ((int)blockIdx.x >= P.blocks) {
        embed_grad_zero<EG_SORT_THREADS>(P, blockIdx.x - P.blocks, 0, P.zero_first);
        return;
    }
    __shared__ ulonglong2 key_s[EG_SORT_THREADS];
    const long long base = (long long)blockIdx.x * EG_BLOCK;
    const int here = (int)min((long long)EG_BLOCK, P.n - base);
    const uint32_t i0 = 2 * threadIdx.x;
    if (blockIdx.x == 0 && threadIdx.x == 0) P.runs[0] = 0;
    unsigned long long key[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint32_t id = EG_NONE;
        if ((int)i0 + e < here) {
            const long long v = P.ids[base + i0 + e];
            if (v >= 0 && v < P.n_rows) id = (uint32_t)v;
        }
        key[e] = (unsigned long long)id << 32 | (i0 + e);
    }
    uint32_t size = 2;
    while ((int)size < here) size *= 2;
    for (uint32_t k = 2; k <= size; k *= 2) {
        const bool up = (i0 & k) == 0;                     // (k = 2: the two elements of a thread are one group)
        for (uint32_t j = k / 2; j > 1; j /= 2) {
            unsigned long long other[2];
            if (j <= 32) {
                other[0] = __shfl_xor_sync(0xFFFFFFFFu, key[0], j / 2);
                other[1] = __shfl_xor_sync(0xFFFFFFFFu, key[1], j / 2);
            } else {
                key_s[threadIdx.x] = make_ulonglong2(key[0], key[1]);
                __syncthreads();
                const ulonglong2 o = key_s[threadIdx.x ^ (j / 2)];
                other[0] = o.x; other[1] = o.y;
                __syncthreads();
            }
            const bool low = ((i0 & j) == 0) == up;        // keeps the smaller one
#pragma unroll
            for (int e = 0; e < 2; ++e) key[e] = (key[e] < other[e]) == low ? key[e] : other[e];
        }
        if ((key[0] > key[1]) == up) { const unsigned long long t = key[0]; key[0] = key[1]; key[1] = t; }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = (int)i0 + e;
        if (i >= here) continue;
        P.block_ids[base + i] = (uint32_t)(key[e] >> 32);
        P.block_pos[base + i] = (uint32_t)(base + (uint32_t)key[e]);
    }
}

// Step 2.  Sorted runs of 2^LOG ids (the last one shorter) become runs of EG_GROUP times that: an element's place is its own in its run, plus how many of
// every other run of the group come before it (equal ids: of earlier runs).  All runs at once would be fewer steps, but the work is quadratic:
// 4.5 ms for the gradient of 2^20 tokens (32000 x 1024), which in three steps of 0.32 ms together takes 1.05.
template <int LOG>
__global__ void __launch_bounds__(EG_PLACE_THREADS) embed_grad_place_kernel(const EmbedGradParams P, int place_blocks, const uint32_t* ids, const uint32_t* pos,
                                                                            uint32_t* ids_out, uint32_t* pos_out) {
    constexpr int run = 1 << LOG;
    if ((int)blockIdx.x >= place_blocks) {
        embed_grad_zero<EG_PLACE_THREADS>(P, blockIdx.x - place_blocks, P.zero_first, P.out_bytes);
        return;
    }
    const int n = (int)P.n, i = (int)blockIdx.x * EG_PLACE_THREADS + (int)threadIdx.x;
    if (i >= n) return;
    const int mine = i / run, first = mine / EG_GROUP * EG_GROUP, last = min(first + EG_GROUP, (n + run - 1) / run);
    const uint32_t id = ids[i];
    int place = first * run + (i - mine * run);
#pragma unroll 4
    for (int b = first; b < last; ++b) {
        const uint32_t* s = ids + b * run;
        const int here = min(run, n - b * run);
        int below = 0;                                     // how many of s come before (id, mine)
#pragma unroll
        for (int step = run / 2; step > 0; step /= 2) {
            const int at = below + step - 1;
            if (at < here) {
                const uint32_t v = s[at];
                if (v < id || (v == id && b < mine)) below += step;
            }
        }
        if (below < here) {
            const uint32_t v = s[below];
            if (v < id || (v == id && b < mine)) ++below;
        }
        if (b != mine) place += below;
    }
    ids_out[place] = id;
    pos_out[place] = pos[i];
}

// Step 3.  A block takes some columns of a tile; all tiles of one range of columns come first (the grid's second dimension would end at 65535 of them).
template <typename T, int W>
__global__ void __launch_bounds__(EG_SUM_THREADS) embed_grad_sum_kernel(const EmbedGradParams P) {
    constexpr int N = PACK<T, W>, AHEAD = 8;               // rows in flight
    __shared__ uint32_t id_s[EG_TILE + 2], pos_s[EG_TILE];
    const int cols = (int)(blockIdx.x / (unsigned)P.tiles), tile = (int)(blockIdx.x - (unsigned)cols * (unsigned)P.tiles);
    const long long t0 = (long long)tile * EG_TILE;
    const int here = (int)min((long long)EG_TILE, P.n - t0);
    if (threadIdx.x < EG_TILE + 2) {                       // the tile's ids and one on either side
        const int i = threadIdx.x;
        const long long at = t0 + i - 1;
        id_s[i] = at >= 0 && at < P.n ? P.ids_sorted[at] : EG_NONE;
        if (i < here) pos_s[i] = P.pos_sorted[t0 + i];
    }
    __syncthreads();
    const uint32_t tail = id_s[here];
    if (cols == 0 && threadIdx.x == 0 && tail != EG_NONE && id_s[here + 1] == tail && id_s[0] != tail) P.runs[1 + atomicAdd(P.runs, 1u)] = (uint32_t)tile;
    const int col = (cols * EG_SUM_THREADS + (int)threadIdx.x) * N;
    if (col >= P.width) return;
    const T* grad = reinterpret_cast<const T*>(P.grad) + col;
    T* out = reinterpret_cast<T*>(P.out) + col;
    float* part = P.part + (long long)tile * 2 * P.width + col;
    float sum[N] = {};
    bool entered = id_s[0] == id_s[1];                     // the run began in an earlier tile
    for (int i0 = 0; i0 < here; i0 += AHEAD) {
        Pack<T, W> v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            v[i].clear();
            if (i0 + i < here && id_s[i0 + i + 1] != EG_NONE) v[i].load(grad + (long long)pos_s[i0 + i] * P.ld);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t id = i0 + i < here ? id_s[i0 + i + 1] : EG_NONE;
            float x[N];
            v[i].values(x);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += x[e];
            const bool last = i0 + i + 1 == here, ends = id_s[min(i0 + i + 2, EG_TILE + 1)] != id;
            if (id == EG_NONE || (!last && !ends)) continue;
            if (entered || !ends) {
                float* p = part + (entered ? 0 : P.width);
                if constexpr (N % 4 == 0) {
#pragma unroll
                    for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
                } else {
                    p[0] = sum[0];
                }
            } else {
                Pack<T, W> o;
                o.set(sum, P.scale);
                o.store(out + (long long)id * P.width);
            }
            entered = false;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0.0f;
        }
    }
}

// Step 4.  A run that leaves tile a for the first time: its rows in the tiles a .. b.  A block takes 1024 columns: of short runs a thread four of them,
// of long ones eight warps a part of the rows each.
template <typename T>
__device__ __forceinline__ void embed_grad_write(const EmbedGradParams& P, uint32_t id, int col, const float (&v)[4]) {
    alignas(16) T o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) set_value(o[e], v[e] * P.scale);
    T* out = reinterpret_cast<T*>(P.out) + (long long)id * P.width + col;
    if (P.width % 4 == 0) {                                // rows of whole packs, and the table begins on a 16-byte boundary
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(o);
        else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < P.width) out[e] = o[e];
    }
}
// four columns of `rows` rows of `part`, two rows apart each, on top of v
__device__ __forceinline__ void embed_grad_rows(const EmbedGradParams& P, const float* part, int col, int rows, float (&v)[4]) {
    if (P.width % 4 == 0) {
#pragma unroll 8
        for (int r = 0; r < rows; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(part + (long long)r * 2 * P.width + col);
            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < P.width) v[e] += part[(long long)r * 2 * P.width + col + e];
    }
}
template <typename T>
__global__ void __launch_bounds__(EG_JOIN_THREADS) embed_grad_join_kernel(const EmbedGradParams P) {
    __shared__ alignas(16) float sum_s[8][EG_JOIN_COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cols = (int)(blockIdx.x / (unsigned)P.join_blocks), col0 = cols * EG_JOIN_COLS, n_runs = (int)P.runs[0];
    for (int k = (int)blockIdx.x - cols * P.join_blocks; k < n_runs; k += P.join_blocks) {
        const long long a = P.runs[1 + k], end = (a + 1) * EG_TILE;
        const uint32_t id = P.ids_sorted[end];
        int rows = 0;                                      // tiles that it enters: those that begin with its id
        for (int more = EG_JOIN_THREADS; more == EG_JOIN_THREADS; rows += more) {
            const long long at = (a + 1 + rows + threadIdx.x) * EG_TILE;
            more = __syncthreads_count(at < P.n && P.ids_sorted[at] == id);
        }
        const float* first = P.part + (a * 2 + 1) * P.width;           // of the tile where it begins
        const float* others = P.part + (a + 1) * 2 * P.width;
        const int col = col0 + (int)threadIdx.x * 4;
        if (rows <= 64) {
            if (col < P.width) {
                float v[4] = {};
                embed_grad_rows(P, first, col, 1, v);
                embed_grad_rows(P, others, col, rows, v);
                embed_grad_write<T>(P, id, col, v);
            }
            continue;
        }
        const int from = (int)((long long)rows * warp / 8), to = (int)((long long)rows * (warp + 1) / 8);
        float v[8][4] = {};
#pragma unroll 2
        for (int r = from; r < to; ++r)
#pragma unroll
            for (int g = 0; g < 8; ++g)
                if (col0 + g * 128 + lane * 4 < P.width) embed_grad_rows(P, others + (long long)r * 2 * P.width, col0 + g * 128 + lane * 4, 1, v[g]);
#pragma unroll
        for (int g = 0; g < 8; ++g) *reinterpret_cast<float4*>(&sum_s[warp][g * 128 + lane * 4]) = make_float4(v[g][0], v[g][1], v[g][2], v[g][3]);
        __syncthreads();
        if (col < P.width) {
            float total[4] = {};
            embed_grad_rows(P, first, col, 1, total);
            for (int w = 0; w < 8; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) total[e] += sum_s[w][threadIdx.x * 4 + e];
            embed_grad_write<T>(P, id, col, total);
        }
        __syncthreads();
    }
}

}  // namespace cb
