// C ABI of the 4-bit KV cache: argument validation and launches.  See include/cobalt_b200.h.
#include <algorithm>
#include <cmath>

#include "kv4_attend.cuh"
#include "kv4_prompt.cuh"

using namespace cb;

namespace {

constexpr int MAX_DEVICES = 64;

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
// the status word of the current device, for calls without one (part of the library's image: nothing is allocated)
uint32_t* status_word() {
    static void* words[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return nullptr;
    if (!words[dev] && cudaGetSymbolAddress(&words[dev], g_kv4_status) != cudaSuccess) return nullptr;
    return (uint32_t*)words[dev];
}
int launched() { return cudaGetLastError() == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH; }
bool dim_ok(int D) { return D > 0 && D % KV4_GROUP == 0 && D <= KV4_GROUP * KV4_MAX_GROUPS; }

// The cache of a call, or why it cannot be one.  Rows (tokens of all sequences) are a grid dimension and an int in the kernels.
int make_cache(Kv4Cache* c, const void* tiles, int64_t seq_stride, const int64_t* positions, int64_t pos_stride, int n_seq, int T, int n_kv, int D,
               int n_slots) {
    if (!tiles || !positions || ((uintptr_t)tiles & 15) || ((uintptr_t)positions & 7) || pos_stride < 0) return COBALT_EINVAL;
    if (n_seq <= 0 || T <= 0 || n_kv <= 0 || n_slots <= 0 || !dim_ok(D)) return COBALT_EINVAL;
    if ((int64_t)n_seq * T > 0x3FFFFFFFll || n_kv > 0xFFFF || n_slots > 0x3FFFFFFF) return COBALT_ETOOBIG;
    c->n_kv = n_kv;
    c->n_slots = n_slots;
    c->n_tiles = (n_slots + KV4_TILE - 1) / KV4_TILE;
    const int64_t one = (int64_t)n_kv * c->n_tiles * kv4_tile_bytes(D / KV4_GROUP);
    if (seq_stride < 0 || (seq_stride & 15) || (n_seq > 1 && seq_stride < one)) return COBALT_EINVAL;
    c->tiles = (uint8_t*)const_cast<void*>(tiles);
    c->seq_stride = seq_stride;
    return COBALT_OK;
}
// rows of bf16 that are read 16 bytes at a time
bool rows_ok(const void* p, int64_t ld, int64_t width) { return p && !((uintptr_t)p & 15) && !(ld & 7) && ld >= width; }

// Whether the device places a cluster of sixteen CTAs of a kernel at all (on one whose SMs are shared out it may not); asked once
template <int G, int NB, bool MANY>
bool places_sixteen() {
    static signed char known[MAX_DEVICES];                             // 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return false;
    if (!known[dev]) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2 * KA_MAX_CLUSTER;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * KA_MAX_CLUSTER);
        cfg.blockDim = dim3(KA_THREADS);
        cfg.dynamicSmemBytes = ka_heads_smem(G, NB);
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        const bool fits = cudaFuncSetAttribute(kv4_attend_heads_kernel<G, NB, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ka_heads_smem(G, NB)) == cudaSuccess &&
                          cudaFuncSetAttribute(kv4_attend_heads_kernel<G, NB, MANY>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                          cudaOccupancyMaxActiveClusters(&n, kv4_attend_heads_kernel<G, NB, MANY>, &cfg) == cudaSuccess && n > 0;
        if (!fits) cudaGetLastError();                                 // not the next launch's
        known[dev] = fits ? 1 : -1;
    }
    return known[dev] > 0;
}
#define KV4_COLUMNS(G_, NB_, CALL)                                     \
    switch ((G_) * 10 + (NB_)) {                                       \
        case 11: { constexpr int G = 1, NB = 1; CALL; } break;         \
        case 12: { constexpr int G = 1, NB = 2; CALL; } break;         \
        case 13: { constexpr int G = 1, NB = 3; CALL; } break;         \
        case 14: { constexpr int G = 1, NB = 4; CALL; } break;         \
        case 21: { constexpr int G = 2, NB = 1; CALL; } break;         \
        case 22: { constexpr int G = 2, NB = 2; CALL; } break;         \
        case 31: { constexpr int G = 3, NB = 1; CALL; } break;         \
        default: { constexpr int G = 4, NB = 1; CALL; } break;         \
    }
bool sixteen_fit(int groups, int nb, bool many) {
    bool fit = false;
    KV4_COLUMNS(groups, nb, fit = (many ? places_sixteen<G, NB, true>() : places_sixteen<G, NB, false>()));
    return fit;
}

struct AttendCfg {
    int cols, nb, col_tiles;
    bool list;
    int grid, share;                   // CTAs; heads: CTAs of a head's cluster
    size_t joins_off, scratch;
};
// Columns are spread evenly over the fewest tiles of 8 * nb that a warp's registers hold.  The work goes by heads, a cluster as large as fills
// the GPU once for each, or by the list, which costs its look-ups and a second kernel but leaves no SM idle and no warp with more
// than its share.  Measured with one token, 32 / 8 heads of 128 (heads / list, us): one sequence of 8192 slots 14.4 / 16.4, 16384 22.1 / 21.7,
// 32768 38.1 / 24.6; 4 sequences of 16384 26.1 / 29.1, 32768 45.8 / 45.7; 16 sequences of 16384 68.7 / 75.9, of 9830 to 32768
// 94.3 / 92.3; 8 / 1 heads of 256, one sequence of 2048 9.9 / 10.7, 4096 12.5 / 11.3.  They meet at 6 tiles per warp plus 64 times the
// share of the GPU that the clusters fill.  Up to eight heads take clusters of sixteen where eight would leave a warp more than four tiles
// (eight / sixteen / list, us: 32 / 8 heads of 128, one sequence of 9000 slots 15.2 / 13.5 / 20.3, 16384 22.2 / 17.6 / 21.5, 32768
// 38.0 / 27.1 / 24.4; 8 / 1 heads of 256, one sequence of 16384 26.8 / 18.4 / 15.2, four of 9000 18.5 / 14.8 / 20.0, of 32768
// 46.1 / 28.3 / 24.0).  Those give way to the list at 6 tiles per warp plus 22 times the share: within 10 % of the better side at most
// lengths, at worst 22 % behind it (8 / 1 heads of 128, four of 3600 to 24000: sixteen 18.7, list, which is taken, 22.9).
// A CTA per head where there are heads for several CTAs per SM.
int attend_config(int n_seq, int T, int n_heads, int n_kv, int D, int n_slots, int window, int sinks, int sms, AttendCfg* c) {
    const int G = D / KV4_GROUP;
    const int64_t cols = (int64_t)(n_heads / n_kv) * T;
    if (cols > 0x3FFFFFFFll) return COBALT_ETOOBIG;
    c->cols = (int)cols;
    const int eights = (c->cols + 7) / 8;
    c->col_tiles = (eights + ka_max_nb(G) - 1) / ka_max_nb(G);
    c->nb = (eights + c->col_tiles - 1) / c->col_tiles;
    c->col_tiles = (eights + c->nb - 1) / c->nb;
    const int64_t entries = (int64_t)n_seq * c->col_tiles, heads = entries * n_kv;
    if (heads > 0x3FFFFFFFll) return COBALT_ETOOBIG;
    const int ctas = std::min(sms * ka_ctas_per_sm(G, c->nb), KC_MAX_STATES);
    // tiles of a head at most, if its tokens follow one another (and if not: the counts of the list are 32-bit)
    const int64_t whole = (n_slots + KV4_TILE - 1) / KV4_TILE;
    int64_t tiles = whole;
    if (window > 0) tiles = std::min(tiles, ((int64_t)window + T) / KV4_TILE + 2 + ((int64_t)sinks + KV4_TILE - 1) / KV4_TILE);
    const bool wide = heads <= KA_WIDE_HEADS && tiles > KA_MAX_CLUSTER * KA_WARPS * 4 && sixteen_fit(G, c->nb, T > 1);
    const int most = wide ? 2 * KA_MAX_CLUSTER : KA_MAX_CLUSTER;
    c->share = 1;
    while (c->share < most && c->share * 2 * heads <= ctas && c->share * KA_MIN_TILES < tiles) c->share *= 2;
    c->list = entries <= KA_ENTRIES && heads * whole < 1000000000ll && heads < 4ll * ctas && 
              tiles * ctas > c->share * KA_WARPS * (6ll * ctas + (c->share > KA_MAX_CLUSTER ? 22 : 64) * heads * c->share);
    c->grid = c->list ? (int)std::min<int64_t>(ctas, (heads * tiles + KA_MIN_TILES - 1) / KA_MIN_TILES) : (int)heads * c->share;
    if (!c->list && heads * c->share > 0x7FFFFFFFll) return COBALT_ETOOBIG;
    c->joins_off = (size_t)c->grid * 2 * ka_state_floats(G, c->nb) * 128;
    c->scratch = c->list ? c->joins_off + (size_t)c->grid * sizeof(int4) : 0;
    return COBALT_OK;
}
template <int G, int NB, bool MANY>
int launch_attend_as(const Kv4AttendParams& P, const Kv4Work& W, const AttendCfg& c, cudaStream_t st) {
    static bool configured[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return COBALT_ELAUNCH;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(kv4_attend_list_kernel<G, NB, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ka_list_smem(G, NB)) != cudaSuccess ||
            cudaFuncSetAttribute(kv4_attend_heads_kernel<G, NB, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ka_heads_smem(G, NB)) != cudaSuccess ||
            cudaFuncSetAttribute(kv4_attend_heads_kernel<G, NB, MANY>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return COBALT_ELAUNCH;
        configured[dev] = true;
    }
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c.grid);
    cfg.blockDim = dim3(KA_THREADS);
    cfg.stream = st;
    cfg.attrs = attr;
    if (!c.list) {
        cfg.dynamicSmemBytes = ka_heads_smem(G, NB);
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)c.share;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = c.share > 1 ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, kv4_attend_heads_kernel<G, NB, MANY>, P, c.share) == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH;
    }
    cfg.dynamicSmemBytes = ka_list_smem(G, NB);
    // (an early start of this kernel under its predecessor left SMs with a carve-out too small for all CTAs: 99 -> 126 us for 440 MB)
    if (cudaLaunchKernelEx(&cfg, kv4_attend_list_kernel<G, NB, MANY>, P, W) != cudaSuccess) return COBALT_ELAUNCH;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)c.grid, NB, G);
    cfg.blockDim = dim3(KC_THREADS);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_combine_kernel<G, NB>, P, W) == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH;
}
template <int G, int NB>
int launch_attend(const Kv4AttendParams& P, const Kv4Work& W, const AttendCfg& c, cudaStream_t st) {
    return P.T > 1 ? launch_attend_as<G, NB, true>(P, W, c, st) : launch_attend_as<G, NB, false>(P, W, c, st);
}

// Whether the prompts' kernel takes a call: at 64 rows per KV head and more, where it is expected to be faster.  Its CTAs walk all keys of their
// rows, a tile of 128 every 2.3 us (128 channels; 1.5 us: 64), so few of them over a long cache are slow; the kernel of few rows splits
// the keys, too, and takes 1.33 ns per tile of 32 slots and tile of columns (16 at 128 channels, 32 at 64), over the whole GPU.  Measured
// (prompt / few, us), 16 / 2 heads of 128, one sequence: 64 tokens over 600 slots 20 / 12, 512 over 600 20 / 21, 512 over 4096 83 / 101,
// 512 over 32768 602 / 697, 128 over 32768 594 / 188; 32 / 8 heads, 4 sequences, 64 tokens over 4096 83 / 107, 32768 658 / 704.
constexpr int KP_MIN_ROWS = 64;
bool prompt_takes(int n_seq, int n_kv, int rep, int T, int D, int n_slots, int window, int sinks, int sms) {
    if ((D != 64 && D != 128) || n_seq > 65535 || rep > KP_ROWS || (int64_t)rep * T < KP_MIN_ROWS) return false;
    double slots = n_slots;
    if (window > 0) slots = std::min(slots, (double)window + sinks + std::min(T, KP_ROWS) + 2 * KP_KEYS);
    const int tok = KP_ROWS / rep;
    const double ctas = (double)((T + tok - 1) / tok) * n_kv * n_seq, eights = ((double)rep * T + 7) / 8;
    const double prompt = std::ceil(ctas / sms) * std::ceil(slots / KP_KEYS) * (D == 128 ? 2.3 : 1.5) + 6.0;
    const double few = std::ceil(eights / ka_max_nb(D / KV4_GROUP)) * n_kv * n_seq * std::ceil(slots / KV4_TILE) * 1.33e-3 + 7.0;
    return prompt < few;
}
template <int G>
int launch_prompt(const Kv4AttendParams& P, cudaStream_t st) {
    static bool configured[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return COBALT_ELAUNCH;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(kv4_prompt_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kp_smem_bytes(G)) != cudaSuccess) return COBALT_ELAUNCH;
        configured[dev] = true;
    }
    const int tok_per_cta = KP_ROWS / P.rep;
    const int64_t blocks = ((int64_t)P.T + tok_per_cta - 1) / tok_per_cta * P.cache.n_kv;
    if (blocks > 0x3FFFFFFFll) return COBALT_ETOOBIG;
    kv4_prompt_kernel<G><<<dim3((unsigned)blocks, (unsigned)P.n_seq), KP_THREADS, kp_smem_bytes(G), st>>>(P, tok_per_cta);
    return cudaGetLastError() == cudaSuccess ? COBALT_OK : COBALT_ELAUNCH;
}

}  // namespace

#define KV4_DISPATCH(D, CALL)                    \
    switch ((D) / KV4_GROUP) {                   \
        case 1: { constexpr int G = 1; CALL; } break; \
        case 2: { constexpr int G = 2; CALL; } break; \
        case 3: { constexpr int G = 3; CALL; } break; \
        default: { constexpr int G = 4; CALL; } break; \
    }

extern "C" {

size_t cobalt_kv4_tile_bytes(int head_dim) { return dim_ok(head_dim) ? (size_t)kv4_tile_bytes(head_dim / KV4_GROUP) : 0; }

int cobalt_kv4_append(const void* k, int64_t ld_k, const void* v, int64_t ld_v, const void* q, int64_t ld_q, void* q_out, int64_t ld_q_out,
                      const int64_t* positions, int64_t pos_seq_stride, void* tiles, int64_t tiles_seq_stride, int n_seq, int T, int n_heads,
                      int n_kv_heads, int head_dim, int n_slots, const float* inv_freq, const void* q_norm_w, const void* k_norm_w, float eps,
                      void* stream) {
    Kv4AppendParams P = {};
    int rc = make_cache(&P.cache, tiles, tiles_seq_stride, positions, pos_seq_stride, n_seq, T, n_kv_heads, head_dim, n_slots);
    if (rc) return rc;
    if (!rows_ok(k, ld_k, (int64_t)n_kv_heads * head_dim) || !rows_ok(v, ld_v, (int64_t)n_kv_heads * head_dim)) return COBALT_EINVAL;
    if (q && (n_heads <= 0 || !rows_ok(q, ld_q, (int64_t)n_heads * head_dim) || !rows_ok(q_out, ld_q_out, (int64_t)n_heads * head_dim))) return COBALT_EINVAL;
    if (q_norm_w && !q) return COBALT_EINVAL;
    if (((uintptr_t)inv_freq | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w) & 3) return COBALT_EINVAL;
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
    P.k = (const uint16_t*)k; P.v = (const uint16_t*)v; P.q = (const uint16_t*)q; P.q_out = (uint16_t*)q_out;
    P.ld_k = ld_k; P.ld_v = ld_v; P.ld_q = ld_q; P.ld_qo = ld_q_out;
    P.positions = (const long long*)positions;
    P.pos_stride = pos_seq_stride;
    P.T = T; P.n_heads = q ? n_heads : 0;
    P.by_T = kv4_div(T);
    P.inv_freq = inv_freq;
    P.q_norm = (const uint16_t*)q_norm_w; P.k_norm = (const uint16_t*)k_norm_w;
    P.eps = eps;
    const int rows = n_seq * T, at_once = 32 / (head_dim / 8), warps = KV4_THREADS / 32;
    const int items = 2 * ((n_kv_heads + at_once - 1) / at_once) + (P.n_heads + at_once - 1) / at_once;
    // few rows: the heads of a row are spread over blocks until the GPU has about two blocks per SM
    const int most = (items + warps - 1) / warps, want = (2 * sms + rows - 1) / rows;
    KV4_DISPATCH(head_dim, (kv4_append_kernel<G><<<dim3((unsigned)rows, (unsigned)std::min(want, most)), KV4_THREADS, 0, (cudaStream_t)stream>>>(P)));
    return launched();
}

int cobalt_kv4_read(const void* tiles, int64_t tiles_seq_stride, const int64_t* positions, int64_t pos_seq_stride, void* k, void* v, int n_seq,
                    int T, int n_kv_heads, int head_dim, int n_slots, void* stream) {
    Kv4Cache C;
    int rc = make_cache(&C, tiles, tiles_seq_stride, positions, pos_seq_stride, n_seq, T, n_kv_heads, head_dim, n_slots);
    if (rc) return rc;
    if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15)) return COBALT_EINVAL;
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
    const int at_once = 32 / (head_dim / 8), per_row = (n_kv_heads + at_once - 1) / at_once;
    const long long items = (long long)n_seq * T * per_row, blocks = (items + KV4_THREADS / 32 - 1) / (KV4_THREADS / 32);
    if (blocks > 0x7FFFFFFFll) return COBALT_ETOOBIG;
    KV4_DISPATCH(head_dim, (kv4_read_kernel<G><<<(unsigned)blocks, KV4_THREADS, 0, (cudaStream_t)stream>>>(
                               C, (const long long*)positions, pos_seq_stride, T, items, per_row, (uint16_t*)k, (uint16_t*)v)));
    return launched();
}

size_t cobalt_kv4_attend_scratch_bytes(int n_seq, int T, int n_heads, int n_kv_heads, int head_dim, int n_slots, int window, int sinks) {
    int sms = 0;
    if (n_seq <= 0 || T <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || n_slots <= 0 || window < 0 || sinks < 0 ||
        !dim_ok(head_dim) || sm_count(&sms)) return 0;
    if (prompt_takes(n_seq, n_kv_heads, n_heads / n_kv_heads, T, head_dim, n_slots, window, sinks, sms)) return 0;
    AttendCfg c;
    return attend_config(n_seq, T, n_heads, n_kv_heads, head_dim, n_slots, window, sinks, sms, &c) ? 0 : c.scratch;
}

int cobalt_kv4_attend_form(int n_seq, int T, int n_heads, int n_kv_heads, int head_dim, int n_slots, int window, int sinks) {
    if (n_seq <= 0 || T <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || n_slots <= 0 || window < 0 || sinks < 0 || !dim_ok(head_dim))
        return COBALT_EINVAL;
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    if (prompt_takes(n_seq, n_kv_heads, n_heads / n_kv_heads, T, head_dim, n_slots, window, sinks, sms)) return COBALT_KV4_PROMPT;
    AttendCfg c;
    if ((rc = attend_config(n_seq, T, n_heads, n_kv_heads, head_dim, n_slots, window, sinks, sms, &c))) return rc;
    return c.list ? COBALT_KV4_LIST : COBALT_KV4_HEADS;
}

int cobalt_kv4_attend(const void* q, int64_t ld_q, const void* tiles, int64_t tiles_seq_stride, const int64_t* positions, int64_t pos_seq_stride,
                      void* out, int n_seq, int T, int n_heads, int n_kv_heads, int head_dim, int n_slots, int window, int sinks, float scale,
                      void* scratch, size_t scratch_bytes, void* stream) {
    return cobalt_kv4_attend_watched(q, ld_q, tiles, tiles_seq_stride, positions, pos_seq_stride, out, n_seq, T, n_heads, n_kv_heads, head_dim, n_slots,
                                     window, sinks, scale, scratch, scratch_bytes, nullptr, stream);
}

int cobalt_kv4_attend_watched(const void* q, int64_t ld_q, const void* tiles, int64_t tiles_seq_stride, const int64_t* positions,
                              int64_t pos_seq_stride, void* out, int n_seq, int T, int n_heads, int n_kv_heads, int head_dim, int n_slots, int window,
                              int sinks, float scale, void* scratch, size_t scratch_bytes, void* status, void* stream) {
    Kv4AttendParams P = {};
    int rc = make_cache(&P.cache, tiles, tiles_seq_stride, positions, pos_seq_stride, n_seq, T, n_kv_heads, head_dim, n_slots);
    if (rc) return rc;
    if (n_heads <= 0 || n_heads % n_kv_heads != 0 || window < 0 || sinks < 0) return COBALT_EINVAL;
    if (!rows_ok(q, ld_q, (int64_t)n_heads * head_dim) || !out || ((uintptr_t)out & 15) || ((uintptr_t)status & 3)) return COBALT_EINVAL;
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
    const bool prompt = prompt_takes(n_seq, n_kv_heads, n_heads / n_kv_heads, T, head_dim, n_slots, window, sinks, sms);
    AttendCfg c = {};
    if (!prompt && (rc = attend_config(n_seq, T, n_heads, n_kv_heads, head_dim, n_slots, window, sinks, sms, &c))) return rc;
    if (c.list && (!scratch || ((uintptr_t)scratch & 255) || scratch_bytes < c.scratch)) return COBALT_ESCRATCH;
    P.q = (const uint16_t*)q; P.ld_q = ld_q;
    P.positions = (const long long*)positions;
    P.pos_stride = pos_seq_stride;
    P.out = (uint16_t*)out;
    P.n_seq = n_seq; P.T = T; P.n_heads = n_heads; P.rep = n_heads / n_kv_heads;
    P.window = window; P.sinks = sinks;
    P.scale_log2 = scale * 1.44269504f;
    P.cols = c.cols; P.col_tiles = c.col_tiles;
    P.status = status ? (uint32_t*)status : status_word();
    if (!P.status) return COBALT_ELAUNCH;
    P.by_rep = kv4_div(P.rep); P.by_kv = kv4_div(n_kv_heads);
    if (prompt) return head_dim == 64 ? launch_prompt<1>(P, (cudaStream_t)stream) : launch_prompt<2>(P, (cudaStream_t)stream);
    P.by_tiles = kv4_div(c.col_tiles);
    Kv4Work W;
    W.partial = (float*)scratch;
    W.joins = (int4*)((uint8_t*)scratch + c.joins_off);
    KV4_COLUMNS(head_dim / KV4_GROUP, c.nb, return (launch_attend<G, NB>(P, W, c, (cudaStream_t)stream)));
}

int cobalt_kv4_status(void* stream, uint32_t* status_out) {
    if (!status_out) return COBALT_EINVAL;
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc) return rc;
    uint32_t* word = status_word();
    if (!word) return COBALT_ELAUNCH;
    if (cudaMemcpyAsync(status_out, word, 4, cudaMemcpyDeviceToHost, (cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    if (cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    if (*status_out == 0) return COBALT_OK;
    // cleared only once it was read as set: kernels write it while it is 0 alone, so a failure on another stream meanwhile is not erased unread
    if (cudaMemsetAsync(word, 0, 4, (cudaStream_t)stream) != cudaSuccess || cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return COBALT_ELAUNCH;
    return COBALT_ETIMEOUT;
}

}  // extern "C"
