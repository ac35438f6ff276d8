// C ABI of the operators at the ends of a vocabulary: embedding lookup and head loss, with their gradients.  See include/cobalt_b200.h.
#include <algorithm>

#include "embed_kernels.cuh"
#include "head_few.cuh"
#include "head_loss.cuh"

using namespace cb;

namespace {

constexpr int MAX_DEVICES = 64;

__device__ uint32_t g_vocab_status;

int sm_count(int* n) {
    static int sms[MAX_DEVICES], major[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return COBALT_ELAUNCH;
    if (dev < 0 || dev >= MAX_DEVICES) return COBALT_EINVAL;
    if (!sms[dev]) {
        if (cudaDeviceGetAttribute(&major[dev], cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return COBALT_ELAUNCH;
        int count = 0;
        if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return COBALT_ELAUNCH;
        sms[dev] = count;
    }
    if (major[dev] != 10) return COBALT_EARCH;
    *n = sms[dev];
    return COBALT_OK;
}
// the status word of the current device (part of the library's image: nothing is allocated)
uint32_t* status_word() {
    static void* words[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return nullptr;
    if (!words[dev] && cudaGetSymbolAddress(&words[dev], g_vocab_status) != cudaSuccess) return nullptr;
    return (uint32_t*)words[dev];
}
int launched() { return cudaGetLastError() == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH; }
template <typename A, typename B>
auto ceil_div(A a, B b) { return (a + b - 1) / b; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// bytes of a value of a type of the embedding calls, 0: no such type
int type_bytes(int type) { return type == COBALT_FP32 ? 4 : type == COBALT_FP16 || type == COBALT_BF16 ? 2 : 0; }
// The statements with T, the type as it lies in memory, and W, the 32-bit words that its rows can be read in at a time (0: a value at a time)
#define EMBED_TYPES(TYPE, ...)                                              \
    if ((TYPE) == COBALT_FP32) { using T = float; __VA_ARGS__; }                   \
    else if ((TYPE) == COBALT_FP16) { using T = Fp16; __VA_ARGS__; }               \
    else { using T = Bf16; __VA_ARGS__; }
// the largest of 8, 4 and 0 words that divides all addresses and strides
int words_at_once(uintptr_t all) { return !(all & 31) ? 8 : !(all & 15) ? 4 : 0; }

struct EmbedGradScratch {
    int blocks, tiles;
    size_t block_ids, block_pos, ids, pos, runs, part, bytes;
};
EmbedGradScratch embed_grad_scratch(int64_t n, int width) {
    EmbedGradScratch s = {};
    s.blocks = (int)ceil_div(n, EG_BLOCK);
    s.tiles = (int)ceil_div(n, EG_TILE);
    const size_t list = align256((size_t)n * 4);
    s.block_ids = 0;
    s.block_pos = list;
    s.ids = 2 * list;
    s.pos = 3 * list;
    s.runs = (s.blocks > 1 ? 4 : 2) * list;
    s.part = s.runs + align256(((size_t)s.tiles + 1) * 4);
    s.bytes = s.part + (s.tiles > 1 ? align256((size_t)s.tiles * 2 * width * 4) : 0);
    return s;
}
constexpr int64_t EMBED_MAX_TOKENS = 1 << 24;
constexpr int EMBED_MAX_WIDTH = 1 << 28;
static_assert(EG_BLOCK == 1 << 11 && EG_GROUP == 1 << 4 && EMBED_MAX_TOKENS <= 1 << 27, "steps of placing");

// ----------------------------------------------------------------------------- head loss
constexpr int HEAD_MAX_TOKENS = 1 << 20, HEAD_MAX_HIDDEN = 1 << 16;
constexpr int HEAD_STATS_TOKENS = 16384;               // tokens whose tile statistics are held at once (8 bytes for 128 columns)
constexpr size_t HEAD_PIECE_BYTES = (size_t)256 << 20;

typedef CUresult (*TensorMapEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                      const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// A matrix (or `depth` of them in a row, ld * rows apart) with boxes of 128 swizzled bytes x box_rows; zeros outside, nothing written there.  A box has
// half of 256 bytes in a row of memory, and the L2 fetches the other half, the next box, with it (W once for one token: 54.3 -> 50.8 us).
int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* p, int64_t ld, int64_t rows, int64_t cols, int box_rows, int depth = 0) {
    static TensorMapEncodeFn encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) return COBALT_ELAUNCH;
        encode = (TensorMapEncodeFn)fn;
    }
    const cuuint64_t size = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
    const cuuint64_t dim[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth}, stride[2] = {(cuuint64_t)ld * size, (cuuint64_t)ld * size * (cuuint64_t)rows};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    return encode(map, type, depth ? 3 : 2, const_cast<void*>(p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? COBALT_OK : COBALT_EINVAL;
}
int bf16_map(CUtensorMap* map, const void* p, int64_t ld, int64_t rows, int64_t cols, int box_rows = 64) {
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, ld, rows, cols, box_rows);
}

// Encoding a map is a driver call and needs the device's context on this thread, which a thread that has launched nothing yet (autograd's) does not have
int bind_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH;
}

// Columns of a tile of logits.  Tiles go round the pairs; with few of them the last round is far from full, and narrower tiles fill it: the
// rounds times a tile's cost (its columns, and 16 for what it costs besides) are smallest.  Less than 160 columns gain nothing: issuing a stage takes 330 clocks,
// the MMAs of 160 columns 320 (333 tokens of 10007 x 1000, three rounds of 96 columns instead of two of 160: 28.6 instead of 24.1 us).
int tile_width(int64_t token_tiles, int64_t cols, int pairs) {
    int best = HL_TILE;
    int64_t least = INT64_MAX;
    for (int w = HL_TILE; w >= 160; w -= 32) {
        const int64_t cost = ceil_div(token_tiles * ceil_div(cols, w), pairs) * (w + 16);
        if (cost < least) { least = cost; best = w; }
    }
    return best;
}

bool head_rows_ok(const void* p, int64_t ld, int64_t width) { return p && !((uintptr_t)p & 15) && !(ld & 7) && ld >= width; }
int head_sizes(int n, int hidden, int64_t vocab) {
    if (n <= 0 || hidden <= 0 || hidden % 8 || vocab <= 0) return COBALT_EINVAL;
    if (n > HEAD_MAX_TOKENS || hidden > HEAD_MAX_HIDDEN || vocab > 0x7FFFF000ll) return COBALT_ETOOBIG;
    return COBALT_OK;
}

// Rows of W of a unit of the few-token kernel: as few rounds of the CTAs as units of at most 256 rows allow, and these evenly filled
int few_rows(int64_t cols, int sms) {
    const int64_t rounds = ceil_div(cols, (int64_t)256 * sms);
    return (int)(ceil_div(ceil_div(cols, rounds * sms), 16) * 16);
}

struct HeadScratch {
    bool few;                              // the few-token kernel forms the logits and dx
    int piece, pieces, splits, stats_tokens, width;      // width: of a tile of logits; few: rows of a unit
    size_t count, slot, target, at, row, packed, part, slab, d[2], bytes;
};
// Ranges of a piece that dx is summed over separately: with dw's tiles to fill up the rounds, so many that every pair has one; without, as gives the
// shortest last round (a range more costs about 3 % of a round: its slab is written and read)
int dx_splits(int64_t tiles, bool want_w, int pairs) {
    int best = 1;
    if (want_w) return (int)std::max<int64_t>(pairs / tiles, 1);
    double least = 1e30;
    for (int s = 1; s <= std::max<int64_t>(2 * pairs / tiles, 4); ++s) {
        const double cost = (double)ceil_div(tiles * s, pairs) / s + 0.03 * s;
        if (cost < least) { least = cost; best = s; }
    }
    return best;
}
HeadScratch head_scratch(int n, int hidden, int64_t vocab, bool backward, bool want_x, bool want_w, int sms) {
    HeadScratch s = {};
    const size_t rows = (size_t)ceil_div(n, HL_TILE) * HL_TILE;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t p = at; at += align256(bytes); return p; };
    s.few = n <= HF_TOKENS;
    if (!backward && s.few) {                              // x is read where it lies
        s.stats_tokens = ceil_div(n, 32) * 32;
        s.width = few_rows(vocab, sms);
        s.count = take(256);
        s.at = take((size_t)n * 4);
        s.part = take((size_t)ceil_div(vocab, s.width) * s.stats_tokens * 8);
        s.bytes = at;
        return s;
    }
    s.count = take(256);
    s.slot = take((size_t)n * 4);
    s.target = take((size_t)n * 4);
    const size_t d_rows = (size_t)n * (backward && s.few ? hf_parts(n) : 1);  // of d, and of x beside it
    s.packed = take(d_rows * hidden * 2);
    if (!backward) {
        s.stats_tokens = (int)std::min<size_t>(rows, HEAD_STATS_TOKENS);
        s.at = take((size_t)n * 4);
        s.width = tile_width(ceil_div(s.stats_tokens, HL_TILE), vocab, sms / 2);
        s.part = take((size_t)ceil_div(vocab, s.width) * 2 * s.stats_tokens * 8);
    } else {
        s.row = take((size_t)n * 16);
        // pieces of equal size, each within HEAD_PIECE_BYTES of scratch
        const int64_t most = std::max<int64_t>(HEAD_PIECE_BYTES / 2 / d_rows / HL_TILE * HL_TILE, HL_TILE);
        s.pieces = (int)ceil_div(vocab, most);
        s.piece = (int)(ceil_div(ceil_div(vocab, s.pieces), HL_TILE) * HL_TILE);
        s.pieces = (int)ceil_div(vocab, s.piece);
        for (int b = 0; b < 2; ++b) s.d[b] = b < s.pieces ? take(d_rows * s.piece * 2) : s.d[0];
        s.width = s.few ? few_rows(s.piece, sms) : tile_width(rows / HL_TILE, s.piece, sms / 2);
        if (want_x) {
            const int64_t tiles = (int64_t)(rows / HL_TILE) * ceil_div(hidden, HL_TILE);
            // (a range of at least one stage, of the last piece too)
            const int64_t last = vocab - (int64_t)(s.pieces - 1) * s.piece;
            const int most = s.few ? std::max((int)(sms / ceil_div(hidden, HL_TILE)), 1) : dx_splits(tiles, want_w, sms / 2);
            s.splits = (int)std::min<int64_t>({most, std::max(s.piece / 512, 1), ceil_div(last, HL_KS)});
            s.slab = take((size_t)s.splits * n * hidden * 4);
        }
    }
    s.bytes = at;
    return s;
}

int prepare(const HlPrepareParams& in, cudaStream_t st) {
    HlPrepareParams P = in;
    P.per_block = (int)ceil_div(P.n, 1024);
    head_prepare_kernel<<<ceil_div(P.n, P.per_block), HL_PREP_THREADS, 0, st>>>(P);
    return launched();
}
// a kernel whose start may overlap the end of the one before (it waits for that one's results itself)
template <typename... Params, typename... Args>
int launch_next(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, const Args&... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH;
}
template <int TOKENS>
int few_sized(const HfParams& P, const CUtensorMap& a, const CUtensorMap& b, int sms, bool first, cudaStream_t st) {
    static bool configured[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return COBALT_ELAUNCH;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(head_few_kernel<TOKENS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return COBALT_ELAUNCH;
        configured[dev] = true;
    }
    const dim3 grid((unsigned)std::min(P.units, sms));
    const uint32_t smem = hf_smem(P.n_pad, P.kind == HL_DX ? hf_parts(TOKENS) : 1);
    if (!first) return launch_next(head_few_kernel<TOKENS>, grid, HF_THREADS, smem, 1, st, P, a, b);
    head_few_kernel<TOKENS><<<grid, HF_THREADS, smem, st>>>(P, a, b);
    return launched();
}
int few(const HfParams& P, const CUtensorMap& a, const CUtensorMap& b, int sms, bool first, cudaStream_t st) {
    return P.n <= HF_TOKENS / 2 ? few_sized<HF_TOKENS / 2>(P, a, b, sms, first, st) : few_sized<HF_TOKENS>(P, a, b, sms, first, st);
}
int product(const HlParams& P, const HlMaps& M, int64_t tiles, int sms, cudaStream_t st) {
    static bool configured[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return COBALT_ELAUNCH;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(head_product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)HL_SMEM) != cudaSuccess) return COBALT_ELAUNCH;
        // warps that ask for registers wait for them: never launch a build that does not bring as many as are handed around
        cudaFuncAttributes built;
        if (cudaFuncGetAttributes(&built, head_product_kernel) != cudaSuccess || built.numRegs != HL_REGS) return COBALT_ELAUNCH;
        configured[dev] = true;
    }
    if (tiles > 0x3FFFFFFF) return COBALT_ETOOBIG;
    return launch_next(head_product_kernel, dim3((unsigned)(2 * std::min<int64_t>(tiles, sms / 2))), HL_THREADS, HL_SMEM, 2, st, P, M);
}

}  // namespace

extern "C" {

int cobalt_embed(const int64_t* ids, int64_t n, const void* table, int64_t ld, int type, int64_t n_rows, int width, float scale, void* out, int64_t ld_out,
                 void* stream) {
    return cobalt_embed_watched(ids, n, table, ld, type, n_rows, width, scale, out, ld_out, nullptr, stream);
}

int cobalt_embed_watched(const int64_t* ids, int64_t n, const void* table, int64_t ld, int type, int64_t n_rows, int width, float scale, void* out, int64_t ld_out,
                         void* status, void* stream) {
    const int size = type_bytes(type);
    if (!ids || !table || !out || !size || n <= 0 || n_rows <= 0 || width <= 0 || ld < width || ld_out < width) return COBALT_EINVAL;
    if (((uintptr_t)ids & 7) || (((uintptr_t)table | (uintptr_t)out) & (size - 1)) || ((uintptr_t)status & 3)) return COBALT_EINVAL;
    if (width > EMBED_MAX_WIDTH) return COBALT_ETOOBIG;
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc) return rc;
    const int words = words_at_once((uintptr_t)table | (uintptr_t)out | (uintptr_t)(ld * size) | (uintptr_t)(ld_out * size) | (uintptr_t)((int64_t)width * size));
    EmbedParams P;
    P.ids = (const long long*)ids;
    P.table = table; P.out = out;
    P.n = n; P.ld = ld; P.ld_out = ld_out; P.n_rows = n_rows;
    P.chunks = words ? width * size / (4 * words) : width;
    P.threads_per_row = 8;
    while (P.threads_per_row < EMB_THREADS && P.threads_per_row < P.chunks) P.threads_per_row *= 2;
    P.scale = scale;
    P.plain = scale == 1.0f;
    P.status = (uint32_t*)status;
    const int64_t blocks = ceil_div(n, EMB_THREADS / P.threads_per_row);
    if (blocks > 0x7FFFFFFFll) return COBALT_ETOOBIG;
    cudaStream_t st = (cudaStream_t)stream;
    EMBED_TYPES(type, {
        if (words == 8) embed_kernel<T, 8><<<(unsigned)blocks, EMB_THREADS, 0, st>>>(P);
        else if (words == 4) embed_kernel<T, 4><<<(unsigned)blocks, EMB_THREADS, 0, st>>>(P);
        else embed_kernel<T, 0><<<(unsigned)blocks, EMB_THREADS, 0, st>>>(P);
    });
    return launched();
}

size_t cobalt_embed_grad_scratch_bytes(int64_t n, int width) {
    return n <= 0 || n > EMBED_MAX_TOKENS || width <= 0 || width > EMBED_MAX_WIDTH ? 0 : embed_grad_scratch(n, width).bytes;
}

int cobalt_embed_grad(const int64_t* ids, int64_t n, const void* grad, int64_t ld, int type, int64_t n_rows, int width, float scale, void* out, void* scratch,
                      size_t scratch_bytes, void* stream) {
    const int size = type_bytes(type);
    if (!ids || !grad || !out || !size || n <= 0 || n_rows <= 0 || width <= 0 || ld < width) return COBALT_EINVAL;
    if (((uintptr_t)ids & 7) || ((uintptr_t)grad & (size - 1)) || ((uintptr_t)out & 15)) return COBALT_EINVAL;
    if (n > EMBED_MAX_TOKENS || n_rows > 0x7FFFFFFFll || width > EMBED_MAX_WIDTH) return COBALT_ETOOBIG;
    const EmbedGradScratch s = embed_grad_scratch(n, width);
    if (!scratch || ((uintptr_t)scratch & 255) || scratch_bytes < s.bytes) return COBALT_ESCRATCH;
    int sms = 0;
    int rc = sm_count(&sms);
    if (rc) return rc;
    uint8_t* base = (uint8_t*)scratch;
    EmbedGradParams P;
    P.ids = (const long long*)ids;
    P.grad = grad; P.out = out;
    P.n = n; P.ld = ld; P.n_rows = n_rows;
    P.width = width; P.blocks = s.blocks; P.tiles = s.tiles;
    P.scale = scale;
    P.block_ids = (uint32_t*)(base + s.block_ids);
    P.block_pos = (uint32_t*)(base + s.block_pos);
    P.ids_sorted = P.block_ids;
    P.pos_sorted = P.block_pos;
    P.part = (float*)(base + s.part);
    P.runs = (uint32_t*)(base + s.runs);
    P.out_bytes = P.zero_first = n_rows * width * size;
    // Counting takes about 4 us on as many SMs as there are blocks, the sort of one block 8 to 9 on one: under zeros that take longer the latter costs
    // less (2047 tokens of 32000 x 4096: 48.1 us, 49.0 by counting; 300 of 5000 x 512: 12.8 and 8.2)
    const bool count = n <= EG_RANK && !(s.blocks == 1 && P.out_bytes >= 64 << 20);
    // The first step of placing takes about 1.5 us a block of ids that it looks through; zeros are written at 7 MB in a microsecond meanwhile
    if (!count && s.blocks > 1) P.zero_first = (P.out_bytes - std::min<int64_t>(P.out_bytes / 2, (int64_t)std::min(s.blocks, EG_GROUP) * (10 << 20))) / 32 * 32;
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t zeros = ceil_div(P.zero_first, EG_ZERO_BYTES);
    const int words = std::min(words_at_once((uintptr_t)grad | (uintptr_t)(ld * size) | (uintptr_t)((int64_t)width * size)), 4);
    const int64_t sums = (int64_t)s.tiles * ceil_div(width, EG_SUM_THREADS * (words ? 16 / size : 1));
    P.join_blocks = std::min(s.tiles, EG_JOIN_GRID);
    const int64_t joins = (int64_t)P.join_blocks * ceil_div(width, EG_JOIN_COLS);
    if (zeros > 0x3FFFFFFFll || sums > 0x7FFFFFFFll || joins > 0x7FFFFFFFll) return COBALT_ETOOBIG;
    if (count) {
        const int ranks = (int)ceil_div(n, EG_RANK_IDS);
        embed_grad_rank_kernel<<<(unsigned)(ranks + zeros), EG_RANK_THREADS, 0, st>>>(P, ranks);
    } else {
        embed_grad_sort_kernel<<<(unsigned)(s.blocks + zeros), EG_SORT_THREADS, 0, st>>>(P);
    }
    if ((rc = launched())) return rc;
    uint32_t *ids_to = (uint32_t*)(base + s.ids), *pos_to = (uint32_t*)(base + s.pos);
    for (int64_t run = EG_BLOCK; !count && run < n; run *= EG_GROUP) {
        const int64_t places = ceil_div(n, EG_PLACE_THREADS), rest = run == EG_BLOCK ? ceil_div(P.out_bytes - P.zero_first, EG_ZERO_BYTES) : 0;
        // (the runs that tokens up to EMBED_MAX_TOKENS need)
        const auto place = run == EG_BLOCK ? embed_grad_place_kernel<11> : run == EG_BLOCK * EG_GROUP ? embed_grad_place_kernel<15>
                           : run == EG_BLOCK * EG_GROUP * EG_GROUP ? embed_grad_place_kernel<19> : embed_grad_place_kernel<23>;
        place<<<(unsigned)(places + rest), EG_PLACE_THREADS, 0, st>>>(P, (int)places, P.ids_sorted, P.pos_sorted, ids_to, pos_to);
        if ((rc = launched())) return rc;
        uint32_t* const ids_was = const_cast<uint32_t*>(P.ids_sorted), *const pos_was = const_cast<uint32_t*>(P.pos_sorted);
        P.ids_sorted = ids_to;
        P.pos_sorted = pos_to;
        ids_to = ids_was;
        pos_to = pos_was;
    }
    EMBED_TYPES(type, {
        if (words) embed_grad_sum_kernel<T, 4><<<(unsigned)sums, EG_SUM_THREADS, 0, st>>>(P);
        else embed_grad_sum_kernel<T, 0><<<(unsigned)sums, EG_SUM_THREADS, 0, st>>>(P);
    });
    if ((rc = launched())) return rc;
    if (s.tiles > 1) {
        EMBED_TYPES(type, { embed_grad_join_kernel<T><<<(unsigned)joins, EG_JOIN_THREADS, 0, st>>>(P); });
    }
    return launched();
}

size_t cobalt_head_loss_scratch_bytes(int n, int hidden, int64_t vocab) {
    int sms = 0;
    return head_sizes(n, hidden, vocab) || sm_count(&sms) ? 0 : head_scratch(n, hidden, vocab, false, false, false, sms).bytes;
}

int cobalt_head_loss(const void* x, int64_t ldx, const void* weight, int64_t ldw, const int64_t* targets, int n, int hidden, int64_t vocab, float* loss,
                     float* stats, float* total, int mean, void* scratch, size_t scratch_bytes, void* status, void* stream) {
    int rc = head_sizes(n, hidden, vocab);
    if (rc) return rc;
    if (!head_rows_ok(x, ldx, hidden) || !head_rows_ok(weight, ldw, hidden) || !targets || !loss) return COBALT_EINVAL;
    if (((uintptr_t)targets & 7) || (((uintptr_t)loss | (uintptr_t)total) & 3) || ((uintptr_t)stats & 7) || ((uintptr_t)status & 3)) return COBALT_EINVAL;
    if (!scratch || ((uintptr_t)scratch & 255)) return COBALT_ESCRATCH;
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
    const HeadScratch s = head_scratch(n, hidden, vocab, false, false, false, sms);
    if (scratch_bytes < s.bytes) return COBALT_ESCRATCH;
    if ((rc = bind_device())) return rc;
    uint8_t* base = (uint8_t*)scratch;
    cudaStream_t st = (cudaStream_t)stream;
    uint32_t* const word = status ? (uint32_t*)status : status_word();
    if (!word) return COBALT_ELAUNCH;
    HlJoinParams J = {};
    J.targets = (const long long*)targets;
    J.vocab = vocab;
    J.part = (float2*)(base + s.part);
    J.at = (float*)(base + s.at);
    J.count = (int*)(base + s.count);
    J.n = n; J.ld_part = s.stats_tokens;
    J.loss = loss; J.stats = (float2*)stats; J.mean = mean;
    if (s.few) {
        HfParams F = {};
        F.kind = HL_STATS;
        F.n = n; F.n_pad = s.stats_tokens;
        F.cols = (int)vocab; F.rows = s.width;
        F.units = (int)ceil_div(vocab, s.width);
        F.hidden = hidden;
        F.targets = J.targets; F.vocab = vocab;
        F.counted = J.count;
        F.part = (float2*)(base + s.part);
        F.at = (float*)(base + s.at);
        F.status = word;
        CUtensorMap wm, xm;
        if ((rc = bf16_map(&wm, weight, ldw, vocab, hidden, s.width / 2)) || (rc = bf16_map(&xm, x, ldx, n, hidden, F.n_pad))) return rc;
        if ((rc = few(F, wm, xm, sms, true, st))) return rc;
        J.parts = F.units;
        J.tokens = n;
        J.total = total;
        return launch_next(head_join_kernel, dim3((unsigned)ceil_div(n, HL_JOIN_TOKENS)), HL_JOIN_THREADS, 0, 1, st, J);
    }
    HlPrepareParams A = {};
    A.x = (const uint16_t*)x; A.ldx = ldx;
    A.targets = (const long long*)targets;
    A.n = n; A.hidden = hidden; A.vocab = vocab;
    A.count = J.count;
    A.slot = (int*)(base + s.slot);
    A.target = (int*)(base + s.target);
    A.packed = (uint16_t*)(base + s.packed);
    HlParams P = {};
    P.status = word;
    HlMaps M = {};
    if ((rc = bf16_map(&M.x_rows, A.packed, hidden, n, hidden, 128)) || (rc = bf16_map(&M.w_rows, weight, ldw, vocab, hidden, s.width / 2))) return rc;
    if ((rc = prepare(A, st))) return rc;
    const int v_tiles = (int)ceil_div(vocab, s.width);
    P.n_jobs = 1;
    P.stages = HL_LOGIT_STAGES;
    P.job[0].kind = HL_STATS;
    P.job[0].cols = (int)vocab;
    P.job[0].n_tiles = v_tiles;
    P.job[0].width = s.width;
    P.job[0].splits = 1;
    P.count = A.count;
    P.n_rows = n; P.hidden = hidden;
    P.target = A.target;
    P.part = (float2*)(base + s.part);
    P.at = (float*)(base + s.at);
    P.ld_part = s.stats_tokens;
    J.slot = A.slot;
    J.parts = 2 * v_tiles;
    for (int tok0 = 0; tok0 < n; tok0 += s.stats_tokens) {
        J.tok0 = P.tok0 = tok0;
        J.tokens = std::min(n - tok0, s.stats_tokens);
        P.tok_tiles = ceil_div(J.tokens, HL_TILE);
        J.total = tok0 + s.stats_tokens >= n ? total : nullptr;
        if ((rc = product(P, M, (int64_t)P.tok_tiles * v_tiles, sms, st))) return rc;
        if ((rc = launch_next(head_join_kernel, dim3((unsigned)ceil_div(n, HL_JOIN_TOKENS)), HL_JOIN_THREADS, 0, 1, st, J))) return rc;
    }
    return COBALT_OK;
}

size_t cobalt_head_loss_grad_scratch_bytes(int n, int hidden, int64_t vocab, int want_x, int want_w) {
    int sms = 0;
    return head_sizes(n, hidden, vocab) || sm_count(&sms) ? 0 : head_scratch(n, hidden, vocab, true, want_x != 0, want_w != 0, sms).bytes;
}

int cobalt_head_loss_grad(const void* x, int64_t ldx, const void* weight, int64_t ldw, const int64_t* targets, const float* stats, const float* grad,
                          int64_t grad_step, int mean, int n, int hidden, int64_t vocab, void* dx, int64_t ld_dx, void* dw, int64_t ld_dw, void* scratch,
                          size_t scratch_bytes, void* status, void* stream) {
    int rc = head_sizes(n, hidden, vocab);
    if (rc) return rc;
    if (!head_rows_ok(x, ldx, hidden) || !head_rows_ok(weight, ldw, hidden) || !targets || !stats || !grad || (!dx && !dw)) return COBALT_EINVAL;
    if ((dx && !head_rows_ok(dx, ld_dx, hidden)) || (dw && !head_rows_ok(dw, ld_dw, hidden))) return COBALT_EINVAL;
    if (((uintptr_t)targets & 7) || ((uintptr_t)stats & 7) || (((uintptr_t)grad | (uintptr_t)status) & 3) || grad_step < 0 || grad_step > 1) return COBALT_EINVAL;
    if (!scratch || ((uintptr_t)scratch & 255)) return COBALT_ESCRATCH;
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
    const HeadScratch s = head_scratch(n, hidden, vocab, true, dx != nullptr, dw != nullptr, sms);
    if (scratch_bytes < s.bytes) return COBALT_ESCRATCH;
    if ((rc = bind_device())) return rc;
    uint8_t* base = (uint8_t*)scratch;
    cudaStream_t st = (cudaStream_t)stream;
    HlPrepareParams A = {};
    A.x = (const uint16_t*)x; A.ldx = ldx;
    A.targets = (const long long*)targets;
    A.n = n; A.hidden = hidden; A.vocab = vocab;
    A.count = (int*)(base + s.count);
    A.slot = (int*)(base + s.slot);
    A.target = (int*)(base + s.target);
    A.packed = (uint16_t*)(base + s.packed);
    A.stats = (const float2*)stats;
    A.grad = grad; A.grad_step = (int)grad_step; A.mean = mean;
    A.row = (float4*)(base + s.row);
    A.factor = (float*)(base + s.count) + 2;
    HlParams P = {};
    P.status = status ? (uint32_t*)status : status_word();
    if (!P.status) return COBALT_ELAUNCH;
    const int n_pad = ceil_div(n, 32) * 32;
    const bool two = s.pieces > 1;
    HlMaps M = {};
    // what a kernel reads by rows it takes in boxes of 128 (few tokens: all of them), x where it lies if they are few
    const int box = s.few ? n_pad : 128;
    const int64_t d_rows = (int64_t)n * (s.few ? hf_parts(n) : 1);
    if ((rc = bf16_map(&M.w_rows, weight, ldw, vocab, hidden, s.width / 2)) ||
        (rc = s.few ? bf16_map(&M.x_rows, x, ldx, n, hidden, box) : bf16_map(&M.x_rows, A.packed, hidden, n, hidden, box)) ||
        (dw && (rc = bf16_map(&M.x, A.packed, hidden, d_rows, hidden))) || (dx && (rc = bf16_map(&M.w, weight, ldw, vocab, hidden)))) return rc;
    for (int b = 0; b <= two; ++b) {
        if (dw && (rc = bf16_map(&M.d[b], base + s.d[b], s.piece, d_rows, s.piece))) return rc;
        if (dx && (rc = bf16_map(&M.d_rows[b], base + s.d[b], s.piece, d_rows, s.piece, box))) return rc;
    }
    if (dx && !s.few && (rc = make_map(&M.slab, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, base + s.slab, hidden, n, hidden, 32, s.splits))) return rc;
    if (dw && (rc = bf16_map(&M.dw, dw, ld_dw, vocab, hidden, 32))) return rc;
    if (!s.few && (rc = prepare(A, st))) return rc;
    P.count = A.count;
    P.tok_tiles = ceil_div(n, HL_TILE);
    P.n_rows = n; P.hidden = hidden;
    P.target = A.target;
    P.row = A.row;
    P.factor = A.factor;
    P.d[0] = (uint16_t*)(base + s.d[0]); P.d[1] = (uint16_t*)(base + s.d[1]);
    P.ld_d = s.piece;
    auto join_dx = [&](const int* slot) {
        const dim3 grid((unsigned)n, (unsigned)ceil_div(hidden, 8 * HL_DX_THREADS));
        return launch_next(head_dx_kernel, grid, HL_DX_THREADS, 0, 1, st, (const float*)(base + s.slab), slot, A.targets, (long long)vocab, n, hidden, s.splits,
                           (const float*)A.factor, (uint16_t*)dx, (long long)ld_dx);
    };
    // One launch per piece and one more: the products with piece i's d beside the logits of piece i + 1
    const int h_tiles = ceil_div(hidden, HL_TILE);
    for (int i = 0; i <= s.pieces; ++i) {
        int64_t tiles = 0;
        P.n_jobs = 0;
        auto piece = [&](int kind, int k) -> HlJob& {
            HlJob& j = P.job[P.n_jobs++];
            j = HlJob{};
            j.kind = kind;
            j.v0 = k * s.piece;
            j.cols = (int)std::min<int64_t>(s.piece, vocab - j.v0);
            j.splits = 1;
            j.buf = k & 1;
            j.width = HL_TILE;
            return j;
        };
        // few tokens: logits and dx by their own kernel
        HfParams F = {};
        F.n = n; F.n_pad = n_pad;
        F.hidden = hidden;
        F.targets = A.targets; F.vocab = vocab;
        F.counted = A.count;
        F.stats = A.stats;
        F.grad = A.grad; F.grad_step = A.grad_step; F.mean = mean;
        F.factor = A.factor;
        F.x = A.x; F.ldx = ldx;
        F.packed = A.packed;
        F.ld_d = s.piece;
        F.slab = (float*)(base + s.slab);
        F.status = P.status;
        auto few_piece = [&](int kind, int k) {
            F.kind = kind;
            F.v0 = k * s.piece;
            F.cols = (int)std::min<int64_t>(s.piece, vocab - F.v0);
            F.d = P.d[k & 1];
        };
        if (s.few && i > 0 && dx) {
            few_piece(HL_DX, i - 1);
            F.h_tiles = h_tiles; F.splits = s.splits; F.add = i > 1;
            F.units = h_tiles * s.splits;
            if ((rc = few(F, M.w, M.d_rows[(i - 1) & 1], sms, false, st))) return rc;
            // (before dw: its writes fill the L2, and reading the slabs behind them took 17 us where it takes 8)
            if (i == s.pieces && (rc = join_dx(nullptr))) return rc;
        }
        if (!s.few && i > 0 && dx) {
            HlJob& j = piece(HL_DX, i - 1);
            j.n_tiles = h_tiles;
            j.splits = s.splits;
            j.add = i > 1;
            tiles += (int64_t)P.tok_tiles * h_tiles * s.splits;
        }
        if (i > 0 && dw) {
            HlJob& j = piece(HL_DW, i - 1);
            j.n_tiles = h_tiles;
            tiles += (int64_t)ceil_div(j.cols, HL_TILE) * h_tiles;
        }
        if (s.few && i < s.pieces) {
            few_piece(HL_DLOGITS, i);
            F.rows = s.width;
            F.units = ceil_div(ceil_div(F.cols, HL_KS) * HL_KS, s.width);
            if ((rc = few(F, M.w_rows, M.x_rows, sms, i == 0, st))) return rc;
        }
        if (!s.few && i < s.pieces) {
            HlJob& j = piece(HL_DLOGITS, i);
            j.width = s.width;
            j.n_tiles = ceil_div(ceil_div(j.cols, HL_KS) * HL_KS, s.width);    // (dx reads whole stages of d)
            tiles += (int64_t)P.tok_tiles * j.n_tiles;
        }
        P.stages = i == 0 ? HL_LOGIT_STAGES : HL_STAGES;
        if (P.n_jobs && (rc = product(P, M, tiles, sms, st))) return rc;
    }
    return dx && !s.few ? join_dx(A.slot) : COBALT_OK;
}

int cobalt_vocab_status(void* stream, uint32_t* status_out) {
    if (!status_out) return COBALT_EINVAL;
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc) return rc;
    uint32_t* word = status_word();
    if (!word) return COBALT_ELAUNCH;
    if (cudaMemcpyAsync(status_out, word, 4, cudaMemcpyDeviceToHost, (cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    if (cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    if (*status_out == 0) return COBALT_OK;
    // cleared only once it was read as set: kernels write it while it is 0 alone
    if (cudaMemsetAsync(word, 0, 4, (cudaStream_t)stream) != cudaSuccess || cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    return COBALT_ETIMEOUT;
}

}  // extern "C"
