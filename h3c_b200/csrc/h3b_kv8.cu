// Paged key/value cache held in E4M3: codes [pages][kv_heads][page_tokens][128], one f32 scale per 64 tokens of a head
// [pages][kv_heads][page_tokens / 64]; value = code * scale.
//
// The scale of a block of 64 tokens x 128 is a power of two: 2^e with the smallest e >= -64 for which the largest
// magnitude is at most 448 * 2^e (448 = the largest E4M3 number).  E4M3 has the same relative precision over 15
// binades, so a power of two costs nothing against absmax / 448, and it makes two things exact: dividing by the scale,
// and raising it later.  Tokens join a half-filled block one by one while a text is decoded; each time the block's
// largest magnitude crosses a power of two, the codes that are there are moved to the new scale, which is exact but for
// codes that become subnormal.  With absmax / 448 every such step would round all of them again.
// A block into which a non-finite value is written gets a NaN scale and zero codes: attention over it gives NaN for
// the rows that see it and nothing else, like the value itself would.
//
// h3b_kv8_append_dev: one CTA per (64-token block of the sequence that receives rows, K/V head, K or V); 16 lanes hold a
// row of 128, every thread keeps its eight 16-byte pieces in registers between the maximum and the conversion: one read,
// one write, no second pass.  Measured (B200): 6,144 tokens of 24 heads 20.9 us = 5.4 TB/s of bytes in and out (a copy:
// 6.5), the integer pipe was the busiest unit (67 %, DRAM 46 %) before the maxima took two values at a time, which made 20.9 us of
// 22.0; one token for each of 64 streams and 8 heads 4.2 us, a launch.
#include "h3b_attn_win.cuh"

namespace h3b {

int kv8_cache_ok(const h3b_kv8_cache *c, const char *who, char *error, size_t error_size) {
    if (!c) return fail(error, error_size, "%s: NULL cache", who);
    if (c->head_dim != 128) return fail(error, error_size, "%s: head_dim %zu unsupported (128 only)", who, c->head_dim);
    if (!c->page_tokens || c->page_tokens % KV8_BLOCK || c->page_tokens > 65536)
        return fail(error, error_size, "%s: page_tokens %zu is not a multiple of %d up to 65536", who, c->page_tokens, KV8_BLOCK);
    if (!c->kv_heads || c->kv_heads > 32767) return fail(error, error_size, "%s: %zu K/V heads", who, c->kv_heads);
    if (!c->pages || c->pages >= 0x7fffffffu / c->kv_heads / c->page_tokens)
        return fail(error, error_size, "%s: a pool of %zu pages is not supported (pages * kv_heads * page_tokens < 2^31)", who, c->pages);
    if (!c->d_k || !c->d_v || !c->d_k_scale || !c->d_v_scale) return fail(error, error_size, "%s: NULL cache tensor", who);
    if (((uintptr_t)c->d_k & 15) || ((uintptr_t)c->d_v & 15) || ((uintptr_t)c->d_k_scale & 3) || ((uintptr_t)c->d_v_scale & 3))
        return fail(error, error_size, "%s: cache codes must be 16-byte aligned, scales 4-byte aligned", who);
    return 1;
}

int kv8_batch_ok(const h3b_kv8_cache *c, const char *who, size_t rows, const int32_t *cu, const int32_t *ext, const int32_t *table,
                 size_t table_stride, size_t n_seq, size_t max_rows, char *error, size_t error_size) {
    if (n_seq > 65535) return fail(error, error_size, "%s: more than 65535 sequences", who);
    if (n_seq && (!cu || !ext || !table)) return fail(error, error_size, "%s: NULL sequence table", who);
    if (((uintptr_t)cu & 3) || ((uintptr_t)ext & 3) || ((uintptr_t)table & 3))
        return fail(error, error_size, "%s: sequence tables must be 4-byte aligned", who);
    if (n_seq && !table_stride) return fail(error, error_size, "%s: table_stride must be given", who);
    if (table_stride >= (size_t)H3B_WIN_MAX / c->page_tokens) return fail(error, error_size, "%s: table_stride out of range", who);
    if (max_rows > rows) return fail(error, error_size, "%s: max_rows %zu of %zu rows", who, max_rows, rows);
    return 1;
}

struct AppendArgs {
    const void *x[2];                        // K, V rows
    long long rs[2], hs[2];
    uint8_t *codes[2];
    float *scales[2];
    const int *cu, *start, *table;
    long long table_stride;
    int rows, max_rows, kv_heads, pages, page_blocks;
    int *status;
};

// 2^e >= a / 448 with the smallest e >= -64; a > 0 finite.  448 = 1.75 * 2^8.
__device__ __forceinline__ float kv8_scale(uint32_t abs_bits) {
    const int x = (int)(abs_bits >> 23) - 127;   // subnormal magnitudes give -127: clamped below
    const int e = max((abs_bits & 0x7fffffu) <= 0x600000u ? x - 8 : x - 7, -64);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

template <typename T> __global__ void __launch_bounds__(128) k_kv8_append(const __grid_constant__ AppendArgs a) {
    __shared__ uint32_t red[4];
    const int s = blockIdx.z, kvh = blockIdx.y >> 1, w = blockIdx.y & 1, tid = threadIdx.x;
    const int r0 = a.cu[s], r1 = a.cu[s + 1], start = a.start[s], nr = r1 - r0;
    if (r0 < 0 || r1 < r0 || r1 > a.rows || nr > a.max_rows || start < 0 ||
        (long long)start + nr > a.table_stride * a.page_blocks * KV8_BLOCK) {
        if (tid == 0 && a.status) atomicCAS(a.status, 0, H3B_ST_EXTENT);
        return;
    }
    const int blk = start / KV8_BLOCK + blockIdx.x;              // 64-token block of the sequence
    const int t0 = blk * KV8_BLOCK;                              // its first token
    const int from = max(start - t0, 0), to = min(start + nr - t0, KV8_BLOCK);   // tokens [from, to) of it are new
    if (from >= to) return;
    const int sub = tid >> 4, c = tid & 15;                      // row of a pass, 16-byte piece of the row
    const T *src = reinterpret_cast<const T *>(a.x[w]) + (long long)(r0 + t0 - start) * a.rs[w] + kvh * a.hs[w] + c * 8;
    uint4 raw[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int t = i * 8 + sub;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t >= from && t < to) raw[i] = __ldg(reinterpret_cast<const uint4 *>(src + t * a.rs[w]));
    }
    // the page is looked up while the rows are on their way
    const int pg = blk / a.page_blocks, page = a.table[s * a.table_stride + pg];
    if (page < 0 || page >= a.pages) {
        if (tid == 0 && a.status) atomicCAS(a.status, 0, H3B_ST_EXTENT);
        return;
    }
    const long long bi = ((long long)page * a.kv_heads + kvh) * a.page_blocks + (blk - pg * a.page_blocks);
    const float before = from > 0 ? kv8_read_scale(a.scales[w][bi]) : 0.0f;      // tokens in front of the new ones keep it at least
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; i++) top = __vmaxu2(top, abs_max8_pair(raw[i]));
    top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();                                             // (and every thread has read the old scale)
    const uint32_t bits = widen_abs<T>(max(max(red[0], red[1]), max(red[2], red[3])));
    float scale = bits >= 0x7f800000u ? __int_as_float(0x7fffffff) : kv8_scale(bits);
    if (from > 0 && !(before <= scale)) scale = before != before ? before : (scale != scale ? scale : before);
    if (tid == 0) a.scales[w][bi] = scale;
    const bool dead = scale != scale;
    const float inv = dead ? 0.0f : 1.0f / scale;
    uint8_t *dst = a.codes[w] + bi * (KV8_BLOCK * 128) + c * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int t = i * 8 + sub;
        if (t >= from && t < to) {
            const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float2 f;
                if (Elem<T>::FMT == 1) f = make_float2(__uint_as_float(v[j] << 16), __uint_as_float(v[j] & 0xffff0000u));
                else f = __half22float2(*reinterpret_cast<const __half2 *>(&v[j]));
                f.x *= inv;
                f.y *= inv;
                h[j] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
            }
            *reinterpret_cast<uint2 *>(dst + t * 128) = dead ? make_uint2(0u, 0u) : make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
        } else if (t < from && scale != before) {                // codes that are there, under the raised scale
            uint2 old = *reinterpret_cast<const uint2 *>(dst + t * 128);
            const float f = before * inv;
            uint32_t words[2] = {old.x, old.y};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float4 x = codes4(words[j]);
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x.x * f, x.y * f), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x.z * f, x.w * f), __NV_SATFINITE, __NV_E4M3);
                words[j] = dead ? 0u : lo | hi << 16;
            }
            *reinterpret_cast<uint2 *>(dst + t * 128) = make_uint2(words[0], words[1]);
        }
    }
}

}  // namespace h3b

using namespace h3b;

extern "C" {

int h3b_kv8_append_dev(h3_cuda *cuda, const h3b_kv8_cache *cache, const h3b_kv8_append_args *x, char *error, size_t error_size) {
    if (!x) return fail(error, error_size, "kv8_append: NULL arguments");
    if (!kv8_cache_ok(cache, "kv8_append", error, error_size)) return 0;
    const size_t strides = x->k_row_stride | x->k_head_stride | x->v_row_stride | x->v_head_stride, max_rows = x->max_rows;
    if (!cuda) return fail(error, error_size, "kv8_append: NULL handle");
    if (x->dtype != H3B_BF16 && x->dtype != H3B_F16) return fail(error, error_size, "kv8_append: dtype must be bf16 or f16");
    if (x->rows >= (size_t)H3B_WIN_MAX) return fail(error, error_size, "kv8_append: shape too large");
    if (x->rows && (!x->d_k || !x->d_v)) return fail(error, error_size, "kv8_append: NULL tensor");
    if (strides % 8 || ((uintptr_t)x->d_k & 15) || ((uintptr_t)x->d_v & 15))
        return fail(error, error_size, "kv8_append: pointers must be 16-byte aligned and strides multiples of 8 elements");
    if (!x->k_row_stride || !x->k_head_stride || !x->v_row_stride || !x->v_head_stride)
        return fail(error, error_size, "kv8_append: row and head strides must be given");
    if (strides >> 39) return fail(error, error_size, "kv8_append: stride too large");
    if (!kv8_batch_ok(cache, "kv8_append", x->rows, x->d_cu_rows, x->d_start, x->d_table, x->table_stride, x->n_seq, max_rows, error,
                      error_size))
        return 0;
    if (!x->rows || !x->n_seq || !max_rows) return 1;
    AppendArgs a;
    memset(&a, 0, sizeof(a));
    a.x[0] = x->d_k; a.x[1] = x->d_v;
    a.rs[0] = (long long)x->k_row_stride; a.rs[1] = (long long)x->v_row_stride;
    a.hs[0] = (long long)x->k_head_stride; a.hs[1] = (long long)x->v_head_stride;
    a.codes[0] = cache->d_k; a.codes[1] = cache->d_v;
    a.scales[0] = cache->d_k_scale; a.scales[1] = cache->d_v_scale;
    a.cu = x->d_cu_rows; a.start = x->d_start; a.table = x->d_table; a.table_stride = (long long)x->table_stride;
    a.rows = (int)x->rows; a.max_rows = (int)max_rows; a.kv_heads = (int)cache->kv_heads; a.pages = (int)cache->pages;
    a.page_blocks = (int)(cache->page_tokens / KV8_BLOCK);
    a.status = cuda->d_status;
    // max_rows rows that start anywhere in a block reach this many blocks
    const dim3 grid((unsigned)ceil_div(max_rows + KV8_BLOCK - 1, KV8_BLOCK), (unsigned)(2 * cache->kv_heads), (unsigned)x->n_seq);
    DeviceGuard guard(cuda);
    ProfScope prof(cuda, PROF_OTHER);
    if (x->dtype == H3B_F16) k_kv8_append<__half><<<grid, 128, 0, cuda->op_stream>>>(a);
    else k_kv8_append<__nv_bfloat16><<<grid, 128, 0, cuda->op_stream>>>(a);
    cuda->launches++;
    H3B_CUDA_OK(cudaGetLastError(), "k_kv8_append launch");
    return 1;
}

}  // extern "C"
