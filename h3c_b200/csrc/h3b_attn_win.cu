// Attention with a sliding window and first keys that stay visible, over 16-bit keys and values of one sequence or over
// the paged 8-bit cache of many.
#include "h3b_attn_win.cuh"

namespace h3b {

static int clip(int64_t v) { return v < 0 || v > H3B_WIN_MAX ? H3B_WIN_MAX : (int)v; }

// checks and fields common to both entry points
static int fill(WinArgs &a, h3_cuda *cuda, const char *who, int dtype, const void *q, size_t q_rs, size_t q_hs, size_t rows,
                size_t heads, size_t kv_heads, size_t head_dim, float scale, int64_t left, int64_t right, int64_t sinks,
                int64_t block, void *out, size_t o_rs, size_t o_hs, char *error, size_t error_size) {
    if (!cuda) return fail(error, error_size, "%s: NULL handle", who);
    if (dtype != H3B_BF16 && dtype != H3B_F16) return fail(error, error_size, "%s: dtype must be bf16 or f16", who);
    if (head_dim != 128) return fail(error, error_size, "%s: head_dim %zu unsupported (128 only)", who, head_dim);
    if (!heads || !kv_heads || heads % kv_heads || heads > 65535)
        return fail(error, error_size, "%s: %zu heads over %zu K/V heads", who, heads, kv_heads);
    if (heads / kv_heads > 128) return fail(error, error_size, "%s: more than 128 heads share a K/V head", who);
    if (sinks < 0) return fail(error, error_size, "%s: sinks must not be negative", who);
    if (block < 1) return fail(error, error_size, "%s: block must be at least 1", who);
    if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(error, error_size, "%s: scale must be positive and finite", who);
    if (rows >= (size_t)H3B_WIN_MAX) return fail(error, error_size, "%s: shape too large", who);
    if (rows && (!q || !out)) return fail(error, error_size, "%s: NULL tensor", who);
    if ((q_rs | q_hs | o_rs | o_hs) % 8 || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
        return fail(error, error_size, "%s: pointers must be 16-byte aligned and strides multiples of 8 elements", who);
    if (!q_rs || !q_hs || !o_rs || !o_hs) return fail(error, error_size, "%s: row and head strides must be given", who);
    if ((q_rs | q_hs | o_rs | o_hs) >> 39) return fail(error, error_size, "%s: stride too large", who);
    if (rows * (heads / kv_heads) > 0x7fffff00u) return fail(error, error_size, "%s: shape too large", who);
    // rows of heads or heads of rows, packed or not; divided, because the products may pass 64 bits
    const bool rows_fit = rows < 2 || o_rs >= 128, heads_fit = heads < 2 || o_hs >= 128;
    const bool nested = rows < 2 || heads < 2 || (rows_fit && heads_fit && ((o_rs - 128) / o_hs >= heads - 1 || (o_hs - 128) / o_rs >= rows - 1));
    if (!rows_fit || !heads_fit || !nested) return fail(error, error_size, "%s: rows or heads of the output overlap", who);
    memset(&a, 0, sizeof(a));
    a.q = q; a.out = out;
    a.q_rs = (long long)q_rs; a.q_hs = (long long)q_hs; a.o_rs = (long long)o_rs; a.o_hs = (long long)o_hs;
    a.rows = (int)rows; a.heads = (int)heads; a.kv_heads = (int)kv_heads; a.group = (int)(heads / kv_heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.win.left = clip(left); a.win.right = clip(right); a.win.sinks = clip(sinks); a.win.block = clip(block);
    a.status = cuda->d_status;
    return 1;
}

size_t attn_clusters_of(const h3_cuda *cuda, AttnClusters &c, const void *kernel, int threads, size_t smem, size_t n) {
    const bool keep = cuda->device < 64;
    if (keep) {
        const int known = c.kept[cuda->device][n - 1].load(std::memory_order_relaxed);
        if (known > 0) return (size_t)known;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)n; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        count = 0;                                          // clusters of this size are not used then
    }
    if (keep && count > 0) c.kept[cuda->device][n - 1].store(count, std::memory_order_relaxed);
    return (size_t)count;
}

template <bool KV8> static int launch(h3_cuda *cuda, const WinArgs &a, int f16, size_t len, char *error, size_t error_size) {
    DeviceGuard guard(cuda);
    ProfScope prof(cuda, PROF_ATTN);
    // 16 rows are one pass of the few-row kernel over the keys.  Measured (us, few-row | tile kernel), cache: 16 rows of 32 streams
    // of 4,000 tokens and 8 heads 78 | 137, 24 rows 158 | 137; 16 rows over 30,000 tokens and 24 heads 66 | 102, 24 rows 84 | 101,
    // 48 rows 124 | 101; 16-bit 64 | 84, 83 | 84, 97 | 84.
    // Over some hundreds of keys the meeting of the rows and the tile kernel's start decide.  16-bit, 24 heads, 16 rows over 64,
    // 128, 256, 384, 512 keys: 13.3 | 7.9, 13.7 | 7.9, 11.1 | 9.4, 10.5 | 10.9, 9.7 | 11.2; 9 rows 9.9 | 8.0, 10.0 | 7.9, 8.9 | 9.4,
    // 8.1 | 11.0, 8.3 | 11.2; 8 rows 8.2 | 8.0, 8.5 | 8.0, 7.2 | 9.5, 6.9 | 11.0, 6.6 | 11.3.  Cache, 16 rows over 128 and 512
    // tokens: 24 heads 16.2 | 13.3, 14.0 | 16.8; 32 streams of 8 heads 18.1 | 24.5, 23.8 | 34.7.
    const size_t rows = (size_t)a.max_rows * a.group;
    const bool brief = !KV8 && rows > 8 && attn_window_keys(a.win, len, (size_t)a.max_rows) <= 256;
    if (rows <= 16 && !brief) return launch_attn_few(cuda, a, f16, KV8, len, error, error_size);
    return launch_attn_tile(cuda, a, f16, KV8, len, error, error_size);
}

}  // namespace h3b

using namespace h3b;

extern "C" {

int h3b_window_tiles(size_t keys, int64_t pos0, size_t rows, int64_t left, int64_t right, int64_t sinks, int64_t block,
                     int unit, int *sink_tiles, int *from, int *count) {
    if (!rows || unit < 1 || block < 1 || sinks < 0 || pos0 < 0 || keys >= (size_t)H3B_WIN_MAX || rows >= (size_t)H3B_WIN_MAX ||
        pos0 + (int64_t)rows > H3B_WIN_MAX || !sink_tiles || !from || !count)
        return 0;
    const h3b_win w = {clip(left), clip(right), clip(sinks), clip(block)};
    const h3b_win_tiles t = h3b_win_tiles_of(w, (int)pos0, (int)(pos0 + (int64_t)rows - 1), (int)keys, unit);
    *sink_tiles = t.sink;
    *from = t.from;
    *count = t.count;
    return 1;
}

int h3b_sdpa_window_dev(h3_cuda *cuda, const h3b_sdpa_window_args *x, char *error, size_t error_size) {
    WinArgs a;
    if (!x) return fail(error, error_size, "sdpa_window: NULL arguments");
    if (!fill(a, cuda, "sdpa_window", x->dtype, x->d_q, x->q_row_stride, x->q_head_stride, x->lq, x->heads, x->kv_heads, x->head_dim,
              x->scale, x->left, x->right, x->sinks, x->block, x->d_out, x->o_row_stride, x->o_head_stride, error, error_size))
        return 0;
    const size_t strides = x->k_row_stride | x->k_head_stride | x->v_row_stride | x->v_head_stride;
    if (x->lk >= (size_t)H3B_WIN_MAX) return fail(error, error_size, "sdpa_window: shape too large");
    if (x->q_pos < 0 || x->q_pos > H3B_WIN_MAX - (int64_t)x->lq) return fail(error, error_size, "sdpa_window: q_pos out of range");
    if (x->lk && (!x->d_k || !x->d_v)) return fail(error, error_size, "sdpa_window: NULL tensor");
    if (strides % 8 || ((uintptr_t)x->d_k & 15) || ((uintptr_t)x->d_v & 15))
        return fail(error, error_size, "sdpa_window: pointers must be 16-byte aligned and strides multiples of 8 elements");
    if (!x->k_row_stride || !x->k_head_stride || !x->v_row_stride || !x->v_head_stride)
        return fail(error, error_size, "sdpa_window: row and head strides must be given");
    if (strides >> 39) return fail(error, error_size, "sdpa_window: stride too large");
    if (!x->lq) return 1;
    a.k = x->d_k; a.v = x->d_v;
    a.k_rs = (long long)x->k_row_stride; a.k_hs = (long long)x->k_head_stride;
    a.v_rs = (long long)x->v_row_stride; a.v_hs = (long long)x->v_head_stride;
    a.lk = (int)x->lk; a.q_pos = (int)x->q_pos; a.max_rows = (int)x->lq; a.n_seq = 1;
    return launch<false>(cuda, a, x->dtype == H3B_F16, x->lk, error, error_size);
}

int h3b_kv8_sdpa_dev(h3_cuda *cuda, const h3b_kv8_cache *cache, const h3b_kv8_sdpa_args *x, char *error, size_t error_size) {
    WinArgs a;
    if (!x) return fail(error, error_size, "kv8_sdpa: NULL arguments");
    if (!kv8_cache_ok(cache, "kv8_sdpa", error, error_size)) return 0;
    if (!fill(a, cuda, "kv8_sdpa", x->dtype, x->d_q, x->q_row_stride, x->q_head_stride, x->rows, x->heads, cache->kv_heads,
              cache->head_dim, x->scale, x->left, x->right, x->sinks, x->block, x->d_out, x->o_row_stride, x->o_head_stride, error,
              error_size))
        return 0;
    if (!kv8_batch_ok(cache, "kv8_sdpa", x->rows, x->d_cu_rows, x->d_len, x->d_table, x->table_stride, x->n_seq, x->max_rows, error,
                      error_size))
        return 0;
    if (x->max_len >= (size_t)H3B_WIN_MAX) return fail(error, error_size, "kv8_sdpa: max_len out of range");
    if (!x->rows || !x->n_seq || !x->max_rows) return 1;
    a.kc = cache->d_k; a.vc = cache->d_v; a.ks = cache->d_k_scale; a.vs = cache->d_v_scale;
    a.cu = x->d_cu_rows; a.len = x->d_len; a.table = x->d_table; a.table_stride = (long long)x->table_stride;
    a.pages = (int)cache->pages; a.page_blocks = (int)(cache->page_tokens / KV8_BLOCK);
    a.max_rows = (int)x->max_rows; a.n_seq = (int)x->n_seq;
    return launch<true>(cuda, a, x->dtype == H3B_F16, x->max_len, error, error_size);
}

}  // extern "C"
