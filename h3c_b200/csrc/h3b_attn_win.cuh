// What the windowed attention kernels share: the call's arguments on the device, the extents of one sequence, and the
// attention of one row by one warp straight from the definition.
#pragma once

#include <cuda_fp8.h>

#include "h3b_attn.cuh"
#include "h3b_internal.h"
#include "h3b_ptx.cuh"
#include "h3b_window.h"

namespace h3b {

constexpr int KV8_BLOCK = 64;   // tokens that share a scale

// One call.  16-bit keys and values: one sequence, cu / len / table are NULL.  8-bit: a paged cache.
struct WinArgs {
    const void *q;
    void *out;
    long long q_rs, q_hs, o_rs, o_hs;        // elements between rows / heads
    int rows, heads, kv_heads, group;        // rows of q and out; group = heads / kv_heads
    float scale_log2;                        // scale of the scores * log2(e)
    h3b_win win;
    int *status;
    // 16-bit K/V
    const void *k, *v;
    long long k_rs, k_hs, v_rs, v_hs;
    int lk, q_pos;
    // 8-bit cache
    const uint8_t *kc, *vc;                  // [pages][kv_heads][page_tokens][128]
    const float *ks, *vs;                    // [pages][kv_heads][page_tokens / 64]
    const int *cu, *len, *table;
    long long table_stride;
    int pages, page_blocks;                  // pages of the pool, 64-token blocks of a page
    int max_rows, n_seq;
};

struct SeqExt {
    int row0, nq, n, pos0;                   // first row of q, rows, keys, position of the first row
};

// Extents of sequence s; one that does not fit the call's arrays is skipped (nq = 0) and reported.
template <bool KV8> __device__ __forceinline__ SeqExt seq_ext(const WinArgs &a, int s) {
    SeqExt e;
    if (!KV8) {
        e.row0 = 0;
        e.nq = a.rows;
        e.n = a.lk;
        e.pos0 = a.q_pos;
        return e;
    }
    const int r0 = a.cu[s], r1 = a.cu[s + 1];
    e.row0 = r0;
    e.nq = r1 - r0;
    e.n = a.len[s];
    e.pos0 = e.n - e.nq;
    if (r0 < 0 || r1 < r0 || r1 > a.rows || e.nq > a.max_rows || e.n < 0 ||
        (long long)e.n > a.table_stride * a.page_blocks * KV8_BLOCK) {
        if (a.status) atomicCAS(a.status, 0, H3B_ST_EXTENT);
        e.nq = e.n = e.pos0 = 0;
    }
    return e;
}

// 64-token block `blk` of sequence s, as an index of (page, head, block of the page); -1 for a page outside the pool
// (reported; the caller treats its tokens as masked).
__device__ __forceinline__ long long kv8_block_index(const WinArgs &a, int s, int blk, int kvh) {
    const int pg = blk / a.page_blocks, page = a.table[s * a.table_stride + pg];
    if (page < 0 || page >= a.pages) {
        if (a.status) atomicCAS(a.status, 0, H3B_ST_EXTENT);
        return -1;
    }
    return ((long long)page * a.kv_heads + kvh) * a.page_blocks + (blk - pg * a.page_blocks);
}

// Scales below 2^-64 count as 2^-64, the smallest that the append writes: a zero (a new cache, a block of zeros quantised
// elsewhere) has no inverse and no logarithm.  NaN stays, and so does a negative one, which is not allowed.
__device__ __forceinline__ float kv8_read_scale(float s) { return s >= 0.0f && s < 0x1p-64f ? 0x1p-64f : s; }

// Probabilities are rounded to the operand type E as 2^(x - m + UP), with m the running maximum as it was last followed: it is
// followed when it has grown by more than 2^LAG.  What is lost of a sum lies at the bottom of the type's range: bf16 has f32's,
// f16 ends at 2^-25 (half its smallest number), so there its range is used up to the top (2^(LAG + UP) < 65504): one key loses at
// most 2^-34 of the largest probability.  (With LAG = 8 and UP = 0 it was 2^-25, and a flat tail of 262,144 keys that held 0.7 % of
// a row was lost altogether.)  Over the cache P carries the value scale, so there it is 2^-34 of the largest probability times
// scale.  UP is whole, so that a probability of 1 stays exact.  The lower LAG is, the more often sums are rescaled.  Measured (us,
// UP 8 | 9 | 10 | 11, LAG 15.9 - UP): 56 heads over 8 in f16 80.1 | 79.5 | 81.5 | 84.1, a frame over 50,220 cached tokens
// 1,112 | 1,114 | 1,118 | 1,143.
template <typename E> struct ProbRange;
template <> struct ProbRange<__half> {
    static constexpr float LAG = 6.9f, UP = 9.0f;
};
template <> struct ProbRange<__nv_bfloat16> {
    static constexpr float LAG = 8.0f, UP = 0.0f;
};

// Largest magnitude of eight 16-bit floats, as two 16-bit patterns side by side: magnitudes order like integers, NaN above
// infinity.
__device__ __forceinline__ uint32_t abs_max8_pair(const uint4 &w) {
    return __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t abs_max8(const uint4 &w) {
    const uint32_t m = abs_max8_pair(w);
    return max(m & 0xffffu, m >> 16);
}
// such a pattern as that of an f32
template <typename T> __device__ __forceinline__ uint32_t widen_abs(uint32_t h) {
    if (Elem<T>::FMT == 1) return h << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

template <typename T> __device__ __forceinline__ float4 load4(const T *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    float4 r;
    if (sizeof(T) == 2 && Elem<T>::FMT == 1) {
        r.x = __uint_as_float(w.x << 16); r.y = __uint_as_float(w.x & 0xffff0000u);
        r.z = __uint_as_float(w.y << 16); r.w = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        r = make_float4(a.x, a.y, b.x, b.y);
    }
    return r;
}
__device__ __forceinline__ float4 codes4(uint32_t w) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}

// four E4M3 codes -> two pairs of f16 (exact)
__device__ __forceinline__ void widen4_e4m3(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}

// largest finite number of a type that a mean of such values may be (bf16: whatever f32 holds)
template <typename T> __device__ __forceinline__ constexpr float largest() { return Elem<T>::FMT == 1 ? 3.402823466e38f : 65504.0f; }
// A weighted mean of f16 values lies between them; half a step of P may put it above 65504, which must not become infinity.
// (Over the cache a code times its scale may lie above it by itself.)
template <typename T, bool KV8> __device__ __forceinline__ float within_type(float x) {
    if (KV8 || Elem<T>::FMT == 1 || !(fabsf(x) < INFINITY)) return x;
    return fminf(fmaxf(x, -largest<T>()), largest<T>());
}

// ---- Values that are not finite, at keys that not every row of a group sees.  A probability of 0 times such a value is not 0, so
// the matrix product hands it to rows that do not see it.  Looking for them in every tile costs time, so the kernels look at
// the results: where a row with a finite sum of probabilities comes out non-finite and the rows of its group differ in what
// they see, the group is gone through a second time.  Then such values count as zero in the tiles that not every row sees
// wholly (a value of any other tile is every row's own), and OddValues gives them back to the rows that see them.  So a group
// costs a second pass over its keys, a search of its edge tiles and at most one more write of its rows, whatever the values are.
// Measured (6,144 tokens of 24 heads, windows of 2,047 keys, 64 sinks, ms): 0.15 without such values, 0.29 with one, 0.63 with
// three in the sinks, which every row sees, 0.87 with nothing else; by frames of 1,024, whose rows see the same, no difference.
template <typename T> __device__ __forceinline__ constexpr uint32_t exponent_ones() { return Elem<T>::FMT == 1 ? 0x7f80u : 0x7c00u; }
// two 16-bit values, each zero if it is not finite
template <typename T> __device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
    constexpr uint32_t e = exponent_ones<T>();
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w >> 16 & e) == e) w &= 0x0000ffffu;
    return w;
}
// a row's sum of probabilities is an ordinary number: what is not finite in its result comes from values
__device__ __forceinline__ bool ordinary(float l) { return l >= 0.0f && l < INFINITY; }

struct OddValues {
    uint32_t nan[4], pos[4], neg[4];         // lane l, bit r: row r of the warp sees one in dimension 4 l + i

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 4; i++) nan[i] = pos[i] = neg[i] = 0u;
    }
    // keys [key, min(key + unit, a.lk)) of K/V head kvh; row r of the warp sees what wr of lane r says, if `live` there
    template <typename T> __device__ __forceinline__ void collect(const WinArgs &a, int kvh, int key, int unit, const h3b_win_row &wr, bool live, int lane) {
        constexpr uint32_t e = exponent_ones<T>();
        const T *v = reinterpret_cast<const T *>(a.v) + kvh * a.v_hs + lane * 4;
        constexpr int N = 16;                // keys whose loads are under way at once
#pragma unroll 1
        for (int k0 = key; k0 < min(key + unit, a.lk); k0 += N) {
            uint2 x[N];
            uint32_t odd = 0u;               // bit u: key k0 + u
#pragma unroll
            for (int u = 0; u < N; u++) x[u] = k0 + u < a.lk ? __ldg(reinterpret_cast<const uint2 *>(v + (long long)(k0 + u) * a.v_rs)) : make_uint2(0u, 0u);
#pragma unroll
            for (int u = 0; u < N; u++) odd |= finite_or_zero<T>(x[u].x) != x[u].x || finite_or_zero<T>(x[u].y) != x[u].y ? 1u << u : 0u;
            odd = __reduce_or_sync(0xffffffffu, odd);
            if (!odd) continue;
#pragma unroll
            for (int u = 0; u < N; u++) {
                if (!(odd >> u & 1u)) continue;
                const uint32_t see = __ballot_sync(0xffffffffu, live && h3b_win_sees(wr, k0 + u));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t b = (i & 2 ? x[u].y : x[u].x) >> (16 * (i & 1)) & 0xffffu, mag = b & 0x7fffu;
                    if (mag > e) nan[i] |= see;
                    else if (mag == e && b >> 15) neg[i] |= see;
                    else if (mag == e) pos[i] |= see;
                }
            }
        }
    }
    // row r has one in some dimension of some lane
    __device__ __forceinline__ bool any(int r) const {
        uint32_t all = 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) all |= nan[i] | pos[i] | neg[i];
        return __any_sync(0xffffffffu, all >> r & 1u);
    }
    // what they add to dimension 4 * lane + i of row r
    __device__ __forceinline__ float of(int r, int i) const {
        const bool p = pos[i] >> r & 1u, n = neg[i] >> r & 1u;
        return (nan[i] >> r & 1u) || (p && n) ? __int_as_float(0x7fffffff) : p ? INFINITY : n ? -INFINITY : 0.0f;
    }
};

// Clusters of `n` (1 to 8) CTAs of a kernel that the chip holds at once.  A cluster lies within one group of SMs and the groups
// of a chip are of different sizes, so this is less than CTAs / n: on one card with 148 SMs, for 1 .. 8, 148, 74, 45, 33, 26, 22, 15,
// 15 with one CTA to an SM, 444, 222, 142, 104, 82, 71, 56, 48 with three.  Asked once for a device (`kept`: of the kernel).
struct AttnClusters {
    std::atomic<int> kept[64][8];
};
size_t attn_clusters_of(const h3_cuda *cuda, AttnClusters &c, const void *kernel, int threads, size_t smem, size_t n);

// Keys that the rows of one CTA can see at most (an estimate that guides how the keys are split).
static inline size_t attn_window_keys(const h3b_win &w, size_t len, size_t rows) {
    const size_t reach = (size_t)w.left + (size_t)w.right + (size_t)w.block + rows + (size_t)w.sinks;
    return reach < len ? reach : len;
}

// many query rows per K/V head: h3b_attn_tile.cu; few: h3b_attn_few.cu.  len: keys of the longest sequence (an estimate guides the split)
int launch_attn_tile(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size);
int launch_attn_few(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size);

}  // namespace h3b
