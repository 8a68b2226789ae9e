// Windowed attention for few query rows per K/V head (one token of a stream, a handful of drafted ones, shared heads):
// the time is that of reading the keys and values once, so the whole chip has to read, and nothing else may wait.
//
// One warp holds up to 16 rows (query rows x heads of one K/V head; rows beyond them are zero) as the A operand of
// m16n8k16 tensor-core products and walks over key tiles of its own: S = Q K^T from registers, online softmax in
// registers, O += P V with P straight from the score fragments.  A warp-private ring of TMA copies feeds it (a warp
// waits for nobody but its own copies).  Tiles are dealt out over the warps of a CTA and the CTAs of a cluster; the
// partial results (m, l, O) meet in shared memory, first of the CTA, then across the cluster, so a split over the keys
// needs neither a workspace nor a second launch.
//
// tcgen05 does not pay here: its smallest product has 64 rows, and S and P would go through tensor memory for 1 to 16.
//
// 8-bit cache: codes are widened to f16 in registers (E4M3 fits f16 exactly), Q goes to f16 under a power of two of its
// row's maximum (bf16 has more range than f16; what is 2^-38 below the row's largest element is lost), and neither K
// nor V is multiplied by its scale: the key scale multiplies 64 score columns, and log2 of the value scale is added to
// their exponent, so P carries it (2^(x + log2 vs - m)) and the row sum takes it out again per 64 keys.  The order of
// the 128 products of a score and of the keys of a sum is free, so every lane takes the 16 bytes it reads as they lie:
// fragments need no shuffles, and the 128-byte swizzle of the copies keeps the reads free of bank conflicts.
#include <algorithm>

#include "h3b_attn_win.cuh"

namespace h3b {

namespace few {
constexpr int WARPS = 4, STAGES = 3, THREADS = WARPS * 32;
constexpr int STAGE = 16384;                       // K half | V half
constexpr int HALF = STAGE / 2;
// shared memory: rings | partial results of the CTA (16 rows x 128 f32, m, l) | barriers
constexpr size_t SMEM_BYTES = 1024 + (size_t)WARPS * STAGES * STAGE + 16 * 128 * 4 + 2 * 16 * 4 + WARPS * 16 * 8 + 256;
constexpr int UNIT8 = 64, UNIT16 = 32;             // keys of a tile
}  // namespace few

struct FewParams {
    WinArgs a;
    CUtensorMap map_k, map_v;                      // 16-bit: {d, head, row} box {64, 1, 32}; 8-bit: {128, rows} box {128, 64}
    int split;                                     // CTAs of a cluster
};

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                               uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                                    uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
    return r;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
// two E4M3 codes (low 16 bits) -> two f16
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
template <typename T> __device__ __forceinline__ float to_f(uint32_t pair, int hi) {
    if (Elem<T>::FMT == 1) return __uint_as_float(hi ? pair & 0xffff0000u : pair << 16);
    return __half2float(__ushort_as_half((unsigned short)(hi ? pair >> 16 : pair & 0xffffu)));
}

// HALF_M: at most 8 rows, the other half of the fragments stays zero and is left out of the softmax
template <typename T, bool KV8, bool HALF_M> __global__ void __launch_bounds__(few::THREADS) k_attn_few(const __grid_constant__ FewParams p) {
    using namespace few;
    constexpr int U = KV8 ? UNIT8 : UNIT16;
    constexpr int NT = U / 8;                      // score tiles of 8 keys
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *acc = reinterpret_cast<float *>(smem + WARPS * STAGES * STAGE);        // [16][128] of this CTA
    float *acc_m = acc + 16 * 128, *acc_l = acc_m + 16;
    float *warp_ml = acc_l + 16;                                                   // [WARPS][16][2]
    uint64_t *bars = reinterpret_cast<uint64_t *>(warp_ml + WARPS * 16 * 2);
    volatile int *abort_word = reinterpret_cast<volatile int *>(bars + WARPS * STAGES);

    const WinArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)blockIdx.x % p.split, mt = (int)blockIdx.x / p.split, kvh = blockIdx.y, s = blockIdx.z;
    const SeqExt e = seq_ext<KV8>(a, s);
    const int r_first = mt * 16, r_end = min(r_first + 16, e.nq * a.group);        // rows = query * group + head of the group
    if (r_first >= r_end) return;                                                  // the whole cluster alike
    const int R = r_end - r_first;
    const int qi_first = r_first / a.group, qi_last = (r_end - 1) / a.group;
    const int p0 = e.pos0 + qi_first, p1 = e.pos0 + qi_last;
    const h3b_win_tiles tiles = h3b_win_tiles_of(a.win, p0, p1, e.n, U);
    const h3b_win_row row_a = h3b_win_of(a.win, p0, e.n), row_z = h3b_win_of(a.win, p1, e.n);
    const int share = (tiles.count + p.split - 1) / p.split;
    const int first = rank * share + warp, last = min((rank + 1) * share, tiles.count);
    const int n_it = first < last ? (last - first + WARPS - 1) / WARPS : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < WARPS * STAGES; i++) mbar_init(&bars[i], 1);
        *abort_word = 0;
        mbar_fence_init();
    }
    __syncthreads();

    // ---- copies: lane 0 issues, all lanes together look up 32 tiles at a time
    uint8_t *ring = smem + warp * STAGES * STAGE;
    uint64_t *bar = bars + warp * STAGES;
    int look_base = 0;
    int my_row = 0;                                // 8-bit: first row of the tile's codes, -1: page outside the pool
    float my_ks = 1.0f, my_vs = 1.0f;
    auto look_up = [&](int it0) {
        look_base = it0;
        if (KV8) {
            const int it = it0 + lane;
            if (it < n_it) {
                const long long bi = kv8_block_index(a, s, h3b_win_tile(tiles, first + it * WARPS), kvh);
                my_row = bi < 0 ? -1 : (int)(bi * KV8_BLOCK);
                my_ks = bi < 0 ? 1.0f : __ldg(a.ks + bi);
                my_vs = bi < 0 ? 1.0f : __ldg(a.vs + bi);
            }
        }
    };
    auto issue = [&](int it, int row) {
        const int st = it % STAGES;
        if (lane == 0) {
            uint8_t *dst = ring + st * STAGE;
            mbar_expect_tx(&bar[st], STAGE);
            if (KV8) {
                tma_load_2d(dst, &p.map_k, &bar[st], 0, max(row, 0));
                tma_load_2d(dst + HALF, &p.map_v, &bar[st], 0, max(row, 0));
            } else {
                const int key = h3b_win_tile(tiles, first + it * WARPS) * U;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    tma_load_3d(dst + h * (HALF / 2), &p.map_k, &bar[st], h * 64, kvh, key);
                    tma_load_3d(dst + HALF + h * (HALF / 2), &p.map_v, &bar[st], h * 64, kvh, key);
                }
            }
        }
    };
    // rows of tiles whose copies are in flight, in issue order (STAGES of them at most)
    int rows_q[STAGES];
    float ks_q[STAGES], vs_q[STAGES];
    auto fetch = [&](int it, int slot) {           // page and scales of tile `it` (warp-uniform), then its copies
        if (it - look_base >= 32) look_up(it);
        const int src = it - look_base;
        rows_q[slot] = KV8 ? __shfl_sync(0xffffffffu, my_row, src) : 0;
        ks_q[slot] = KV8 ? __shfl_sync(0xffffffffu, my_ks, src) : 1.0f;
        vs_q[slot] = KV8 ? __shfl_sync(0xffffffffu, my_vs, src) : 1.0f;
        issue(it, rows_q[slot]);
    };
    if (n_it) {
        look_up(0);
#pragma unroll
        for (int i = 0; i < STAGES; i++)
            if (i < n_it) fetch(i, i);
    }

    // ---- Q fragments: rows g and g + 8.  16-bit keys: the product's own order of d.  8-bit: lane t takes d = 16 t .. 16 t + 15
    // and 64 + 16 t .., the 16-byte pieces of a key that it reads.
    uint32_t qf[8][4];
    float row_scale[2];                            // scale * log2(e), and what brings Q to f16
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = r_first + g + 8 * h;
        const bool live = r < r_end;
        const int qi = live ? r / a.group : qi_first, hd = live ? r - qi * a.group : 0;
        const T *src = reinterpret_cast<const T *>(a.q) + (long long)(e.row0 + qi) * a.q_rs + (long long)(kvh * a.group + hd) * a.q_hs;
        row_scale[h] = a.scale_log2;
        if (KV8) {
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (live) x = __ldg(reinterpret_cast<const uint4 *>(src + (c >> 1) * 64 + t * 16 + (c & 1) * 8));
                w[4 * c] = x.x; w[4 * c + 1] = x.y; w[4 * c + 2] = x.z; w[4 * c + 3] = x.w;
            }
            float top = 0.0f;
            bool odd = false;                      // not finite: as it is, so that it reaches the result
#pragma unroll
            for (int i = 0; i < 16; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float f = fabsf(to_f<T>(w[i], j));
                    odd |= !(f < INFINITY);
                    top = fmaxf(top, f);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            odd = __shfl_xor_sync(0xffffffffu, (int)odd, 1) | odd;
            odd = __shfl_xor_sync(0xffffffffu, (int)odd, 2) | odd;
            int sh = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
            sh = odd || top == 0.0f ? 0 : max(min(sh, 120), -120);
            const float up = __uint_as_float((uint32_t)(127 + sh) << 23), down = __uint_as_float((uint32_t)(127 - sh) << 23);
            row_scale[h] *= down;
#pragma unroll
            for (int i = 0; i < 8; i++) {          // step i: words 2i (k 2t, 2t+1) and 2i + 1 (k 2t+8, 2t+9)
                qf[i][h] = Elem<__half>::pack(to_f<T>(w[2 * i], 0) * up, to_f<T>(w[2 * i], 1) * up);
                qf[i][2 + h] = Elem<__half>::pack(to_f<T>(w[2 * i + 1], 0) * up, to_f<T>(w[2 * i + 1], 1) * up);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    qf[i][2 * j + h] = live ? __ldg(reinterpret_cast<const uint32_t *>(src + i * 16 + j * 8 + t * 2)) : 0u;
        }
    }
    h3b_win_row wr[2];
#pragma unroll
    for (int h = 0; h < 2; h++) wr[h] = h3b_win_of(a.win, e.pos0 + min(r_first + g + 8 * h, r_end - 1) / a.group, e.n);

    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    constexpr int MH = HALF_M ? 1 : 2;
    const int perm_t = ((t & 1) << 1) | (t >> 1);  // swap of the two bits: see the key order below
    bool ok = true;
    int gave_up = 0;

    auto step = [&](int it, auto slot_c) {
        constexpr int slot = decltype(slot_c)::value;
        const int tile = h3b_win_tile(tiles, first + it * WARPS), k0 = tile * U;
        ok = __all_sync(0xffffffffu, mbar_wait(&bar[slot], (it / STAGES) & 1, abort_word, a.status, H3B_ST_TIMEOUT_FULL));
        if (!ok) {
            gave_up = it;
            return;
        }
        const uint32_t kb = smem_u32(ring + slot * STAGE), vb = kb + HALF;
        float sc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
        if (KV8) {
            // key of column c of a tile: bits 0 and 2 of c swapped, so that the eight lanes of one shared-memory phase
            // (two columns) meet all eight 16-byte banks of the swizzled rows
            const int kr = (g & 2) | ((g & 1) << 2) | (g >> 2);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const uint32_t row = kb + (i * 8 + kr) * 128;
                const uint4 x = lds128(row + ((t ^ kr) << 4)), y = lds128(row + (((t + 4) ^ kr) << 4));
                const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                for (int k = 0; k < 8; k++)
                    mma16816<__half>(sc[i], qf[k][0], qf[k][1], qf[k][2], qf[k][3], widen2(w[k]), widen2(w[k] >> 16));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int key = i * 8 + (lane & 7), mat = lane >> 3;           // lane's row of matrix `mat` (16-byte piece of d)
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const int piece = k * 2 + mat;                              // of 16
                    uint32_t b0, b1, b2, b3;
                    ldsm4(kb + (piece >> 3) * (HALF / 2) + key * 128 + (((piece & 7) ^ (key & 7)) << 4), b0, b1, b2, b3);
                    mma16816<T>(sc[i], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b0, b1);
                    mma16816<T>(sc[i], qf[k + 1][0], qf[k + 1][1], qf[k + 1][2], qf[k + 1][3], b2, b3);
                }
            }
        }
        // exponents: score * scale (+ log2 of the value scale), masked ones -inf
        const float ks = ks_q[slot], vs = vs_q[slot];
        const float lvs = KV8 ? log2f(vs) : 0.0f, ivs = KV8 ? 1.0f / vs : 1.0f;
        const bool masked = !h3b_win_full(row_a, row_z, k0, U) || rows_q[slot] < 0;
        if (!KV8 && masked) {
            // a value that no row sees must not meet its zero probability (0 * NaN): such rows of the tile become zero
            const int j = k0 + lane;
            if (j > row_z.hi || (j < row_a.lo && j >= row_z.s)) {
#pragma unroll
                for (int c = 0; c < 16; c++)
                    *reinterpret_cast<uint4 *>(ring + slot * STAGE + HALF + (c >> 3) * (HALF / 2) + lane * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();          // the next copy into the stage comes behind these stores
            }
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < MH; h++) {
            const float f = KV8 ? row_scale[h] * ks : row_scale[h];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x = KV8 ? fmaf(sc[i][2 * h + j], f, lvs) : sc[i][2 * h + j] * f;
                    if (masked) {
                        const int key = k0 + i * 8 + (KV8 ? perm_t + 4 * j : 2 * t + j);
                        if (!h3b_win_sees(wr[h], key) || rows_q[slot] < 0) x = -INFINITY;
                    }
                    sc[i][2 * h + j] = x;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run[h], mx);
            // the maximum is followed only when it has grown by more than 2^8: P stays below 2^8, sums undo it
            const bool grow = m_new > m_run[h] + 8.0f || (m_run[h] == -INFINITY && m_new > -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
                float alpha = 1.0f;
                if (grow) {
                    alpha = m_run[h] == -INFINITY ? 0.0f : ex2_approx(m_run[h] - m_new);
                    m_run[h] = m_new;
                }
                l_run[h] *= alpha;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    o[i][2 * h] *= alpha;
                    o[i][2 * h + 1] *= alpha;
                }
            }
            const float m_use = m_run[h] == -INFINITY ? 0.0f : m_run[h];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float x = ex2_approx(sc[i][2 * h + j] - m_use);
                    sc[i][2 * h + j] = x;
                    sum += x;
                }
            l_run[h] += KV8 ? (sum == 0.0f ? 0.0f : sum * ivs) : sum;
        }
        // O += P V, 16 keys at a time
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
            uint32_t pf[4];
            if (KV8) {
                pf[0] = Elem<__half>::pack(sc[i][0], sc[i][1]);
                pf[1] = HALF_M ? 0u : Elem<__half>::pack(sc[i][2], sc[i][3]);
                pf[2] = Elem<__half>::pack(sc[i + 1][0], sc[i + 1][1]);
                pf[3] = HALF_M ? 0u : Elem<__half>::pack(sc[i + 1][2], sc[i + 1][3]);
                // lane: keys perm_t, perm_t + 4 of both tiles, d piece with bits 0 and 2 of g swapped (as for the keys)
                const int piece = (g & 2) | ((g & 1) << 2) | (g >> 2);
                uint4 x[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = (i + (r >> 1)) * 8 + perm_t + 4 * (r & 1);
                    x[r] = lds128(vb + key * 128 + ((piece ^ (key & 7)) << 4));
                    if (k0 + key >= e.n) x[r] = make_uint4(0u, 0u, 0u, 0u);    // stale bytes behind the sequence
                }
                const uint32_t w0[4] = {x[0].x, x[0].y, x[0].z, x[0].w}, w1[4] = {x[1].x, x[1].y, x[1].z, x[1].w};
                const uint32_t w2[4] = {x[2].x, x[2].y, x[2].z, x[2].w}, w3[4] = {x[3].x, x[3].y, x[3].z, x[3].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t lo0 = __byte_perm(w0[j], w1[j], 0x5140), hi0 = __byte_perm(w0[j], w1[j], 0x7362);
                    const uint32_t lo1 = __byte_perm(w2[j], w3[j], 0x5140), hi1 = __byte_perm(w2[j], w3[j], 0x7362);
                    mma16816<__half>(o[4 * j], pf[0], pf[1], pf[2], pf[3], widen2(lo0), widen2(lo1));
                    mma16816<__half>(o[4 * j + 1], pf[0], pf[1], pf[2], pf[3], widen2(lo0 >> 16), widen2(lo1 >> 16));
                    mma16816<__half>(o[4 * j + 2], pf[0], pf[1], pf[2], pf[3], widen2(hi0), widen2(hi1));
                    mma16816<__half>(o[4 * j + 3], pf[0], pf[1], pf[2], pf[3], widen2(hi0 >> 16), widen2(hi1 >> 16));
                }
            } else {
                pf[0] = Elem<T>::pack(sc[i][0], sc[i][1]);
                pf[1] = HALF_M ? 0u : Elem<T>::pack(sc[i][2], sc[i][3]);
                pf[2] = Elem<T>::pack(sc[i + 1][0], sc[i + 1][1]);
                pf[3] = HALF_M ? 0u : Elem<T>::pack(sc[i + 1][2], sc[i + 1][3]);
                const int key = i * 8 + (lane & 15);                            // matrices: keys 0-7 | 8-15 of two d pieces
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int piece = 2 * j + (lane >> 4);
                    uint32_t b0, b1, b2, b3;
                    ldsm4t(vb + (piece >> 3) * (HALF / 2) + key * 128 + (((piece & 7) ^ (key & 7)) << 4), b0, b1, b2, b3);
                    mma16816<T>(o[2 * j], pf[0], pf[1], pf[2], pf[3], b0, b1);
                    mma16816<T>(o[2 * j + 1], pf[0], pf[1], pf[2], pf[3], b2, b3);
                }
            }
        }
        __syncwarp();                                                           // every lane has read the stage
        if (it + STAGES < n_it) fetch(it + STAGES, slot);
    };
    for (int it = 0; it < n_it && ok; it += STAGES) {
        step(it, std::integral_constant<int, 0>{});
        if (ok && it + 1 < n_it) step(it + 1, std::integral_constant<int, 1>{});
        if (ok && it + 2 < n_it) step(it + 2, std::integral_constant<int, 2>{});
    }
    static_assert(STAGES == 3, "the loop above is unrolled by the ring");
    // a wait that gave up: the copies in flight (of this tile and the STAGES - 1 behind it) get a last, bounded chance to land
    if (!ok)
        for (int it = gave_up; it < min(n_it, gave_up + STAGES); it++)
            for (int spin = 0; spin < 100000 && !mbar_try_wait(&bar[it % STAGES], (it / STAGES) & 1); spin++) {}

    // ---- meet: warps of the CTA
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
        if (t == 0) {
            warp_ml[(warp * 16 + g + 8 * h) * 2] = m_run[h];
            warp_ml[(warp * 16 + g + 8 * h) * 2 + 1] = l_run[h];
        }
    }
    float *mine = reinterpret_cast<float *>(ring);                               // 16 x 128 f32 of this warp
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
        for (int h = 0; h < MH; h++) {
            const int r = g + 8 * h;
            if (KV8) {
                mine[r * 128 + perm_t * 16 + i] = o[i][2 * h];
                mine[r * 128 + 64 + perm_t * 16 + i] = o[i][2 * h + 1];
            } else {
                *reinterpret_cast<float2 *>(&mine[r * 128 + i * 8 + 2 * t]) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            }
        }
    __syncthreads();
    const int d = threadIdx.x;                                                   // THREADS = 128 = head size
    for (int r = 0; r < R; r++) {
        float m = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, warp_ml[(w * 16 + r) * 2]);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float mw = warp_ml[(w * 16 + r) * 2], lw = warp_ml[(w * 16 + r) * 2 + 1];
            const float c = mw == -INFINITY ? 0.0f : ex2_approx(mw - m);
            // a warp whose l is NaN saw something undefined: it counts even if it has no maximum
            l += lw != lw ? lw : c * lw;
            v += c * reinterpret_cast<const float *>(smem + w * STAGES * STAGE)[r * 128 + d];
        }
        acc[r * 128 + d] = v;
        if (d == 0) {
            acc_m[r] = m;
            acc_l[r] = l;
        }
    }
    // ---- CTAs of the cluster: each finishes some rows
    cluster_sync_all();
    const uint32_t acc_addr = smem_u32(acc);
    for (int r = rank; r < R; r += p.split) {
        float m = -INFINITY, l = 0.0f, v = 0.0f;
        for (int c = 0; c < p.split; c++) m = fmaxf(m, ld_cluster_f32(mapa_shared(acc_addr, c) + (16 * 128 + r) * 4));
        for (int c = 0; c < p.split; c++) {
            const uint32_t base = mapa_shared(acc_addr, c);
            const float mc = ld_cluster_f32(base + (16 * 128 + r) * 4), lc = ld_cluster_f32(base + (16 * 128 + 16 + r) * 4);
            const float w = mc == -INFINITY ? 0.0f : ex2_approx(mc - m);
            l += lc != lc ? lc : w * lc;
            v += w * ld_cluster_f32(base + (r * 128 + d) * 4);
        }
        const int qi = (r_first + r) / a.group, hd = (r_first + r) - qi * a.group;
        const h3b_win_row wr_r = h3b_win_of(a.win, e.pos0 + qi, e.n);
        const int seen = h3b_win_count(wr_r);
        const float res = seen ? v * (1.0f / l) : 0.0f;
        T *dst = reinterpret_cast<T *>(a.out) + (long long)(e.row0 + qi) * a.o_rs + (long long)(kvh * a.group + hd) * a.o_hs;
        const uint32_t w2 = Elem<T>::pack(res, res);
        reinterpret_cast<unsigned short *>(dst)[d] = (unsigned short)(w2 & 0xffffu);
        // a value that is not finite and that other rows of the tile see: such a row is computed again from its own keys
        if (!KV8 && __syncthreads_or(!(fabsf(res) < INFINITY))) {
            if (warp == 0) attn_row_by_warp<T, KV8>(a, s, e, qi, kvh * a.group + hd, lane);
        }
    }
    cluster_sync_all();                                                          // nobody leaves while its memory is read
}

// CTAs that share the keys of one (sequence, K/V head, 16 rows): as many as fill the chip once, but no fewer than
// `WARPS` tiles each (a ring is then filled once), and at most 8 (the portable cluster size).
static int few_split(const h3_cuda *cuda, size_t units, size_t tiles) {
    const size_t by_chip = units >= (size_t)cuda->sm_count ? 1 : (size_t)cuda->sm_count / units;
    const size_t by_work = std::max<size_t>(tiles / few::WARPS, 1);
    return (int)std::min<size_t>(std::min(by_chip, by_work), 8);
}

template <typename T, bool KV8> static int launch_few_t(h3_cuda *cuda, const FewParams &p, dim3 grid, bool half_m, char *error, size_t error_size) {
    void (*kernel)(const FewParams) = half_m ? k_attn_few<T, KV8, true> : k_attn_few<T, KV8, false>;
    H3B_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few::SMEM_BYTES), "attention smem attribute");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(few::THREADS);
    cfg.dynamicSmemBytes = few::SMEM_BYTES;
    cfg.stream = cuda->op_stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    H3B_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p), "k_attn_few launch");
    cuda->launches++;
    return 1;
}

// Keys that one sequence's rows can see at most, for the split (an estimate is enough).
static size_t window_keys(const h3b_win &w, size_t len, size_t rows) {
    const size_t reach = (size_t)w.left + (size_t)w.right + (size_t)w.block + rows;
    return std::min(len, reach >= (size_t)H3B_WIN_MAX ? len : reach + (size_t)w.sinks);
}

int launch_attn_few(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size) {
    FewParams p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    if (kv8) {
        const uint64_t n = (uint64_t)a.pages * a.kv_heads * a.page_blocks * KV8_BLOCK;
        if (h3b_encode_tmap_2d(&p.map_k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.kc, 128, n, 128, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_2d(&p.map_v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.vc, 128, n, 128, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "kv8_sdpa: cuTensorMapEncodeTiled failed");
    } else if (a.lk) {
        const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if (h3b_encode_tmap_3d(&p.map_k, dt, 2, a.k, 128, a.kv_heads, a.lk, a.k_hs * 2, a.k_rs * 2, 64, 1, 32, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_3d(&p.map_v, dt, 2, a.v, 128, a.kv_heads, a.lk, a.v_hs * 2, a.v_rs * 2, 64, 1, 32, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "sdpa_window: cuTensorMapEncodeTiled failed");
    }
    const size_t rows = (size_t)a.max_rows * a.group, mtiles = ceil_div(rows, 16);
    const size_t keys = window_keys(a.win, len, (size_t)a.max_rows);
    p.split = few_split(cuda, mtiles * a.kv_heads * a.n_seq, ceil_div(keys, kv8 ? few::UNIT8 : few::UNIT16));
    const dim3 grid((unsigned)(mtiles * p.split), (unsigned)a.kv_heads, (unsigned)a.n_seq);
    const bool half = rows <= 8;
    if (kv8) return f16 ? launch_few_t<__half, true>(cuda, p, grid, half, error, error_size)
                        : launch_few_t<__nv_bfloat16, true>(cuda, p, grid, half, error, error_size);
    return f16 ? launch_few_t<__half, false>(cuda, p, grid, half, error, error_size)
               : launch_few_t<__nv_bfloat16, false>(cuda, p, grid, half, error, error_size);
}

}  // namespace h3b
