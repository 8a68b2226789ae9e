// Windowed attention for few query rows per K/V head (one token of a stream, a handful of drafted ones, shared heads):
// the time is that of reading the keys and values once, so the whole chip has to read, and nothing else may wait.
//
// A warp works on all rows, up to 8 NT (query rows x heads of one K/V head; rows beyond them are zero), with m16n8k16
// tensor-core products whose 16 rows are KEYS, respectively dimensions: S^T = K Q^T and O^T += V^T P^T, so that nothing is
// padded from 1 to 16 rows (8 is the least) and the widened keys and values are the operands that are used once.  Q stays
// in registers, P goes from score fragments to operand fragments through one 8x8 transposition per 8 keys.  The running
// maximum is looked at by a vote and followed only when it has grown by more than ProbRange says.  A warp has a stage of its own
// for TMA copies: those of the next keys are under way while the values are used and the other way round, and a warp waits
// for nobody but its own copies.  Tiles are dealt out over the warps of a CTA and the CTAs of a cluster; the partial
// results (m, l, O) meet in shared memory, first of the CTA, then across the cluster, so a split over the keys needs
// neither a workspace nor a second launch.
//
// tcgen05 does not pay here: its smallest product has 64 rows, and S and P would go through tensor memory for 1 to 16.
//
// 8-bit cache: codes are widened to f16 in registers (E4M3 fits f16 exactly), Q goes to f16 under a power of two of its
// row's maximum (bf16 has more range than f16; what is 2^-38 below the row's largest element is lost), and neither K
// nor V is multiplied by its scale: the key scale multiplies 64 scores, and log2 of the value scale is added to
// their exponent, so P carries it (2^(x + log2 vs - m), in the range of f16 that ProbRange chooses) and the row sum takes it out again per 64 keys.  The order of
// the 128 products of a score and of the keys of a sum is free, so every lane takes the 16 bytes it reads as they lie:
// fragments need no shuffles, and the 128-byte swizzle of the copies keeps the reads free of bank conflicts.
//
// Measured (B200; the bytes are those of visible codes, scales, Q and output):
//   one token for each of 64 streams of up to 16,384 tokens, 56 heads over 8: 178 us = 6.6 TB/s, what a copy reaches.  With
//   the rows as the products' 16 rows it was 464 us, with twelve warps and shorter tiles 210: half of every product was
//   padding and a warp alone issues one instruction in four cycles.
//   five drafted tokens for 12 streams, 24 heads over 8 (15 rows), windows of 8,192: 46-47 us = 3.8 TB/s; twice the
//   products and exponentials per key.  Bound by latency: no unit is half busy (DRAM 48 %, issue 33 %, tensor 27 %), and of
//   7.6 cycles that a warp takes per instruction 2.1 are fixed latency, 1.3 loads and 1.0 barriers.  9 to 16 rows over the cache
//   are the one variant that spills (168 registers, 88 bytes stored and 68 loaded).
//   one stream of 24 heads: 8.2-8.4 us over 2,313 tokens, 6.8 over 640, 5.4 over 64, 3.6 over none: launch, look-ups one
//   behind the other (extents, page, copy) and the meeting of warps and CTAs.  One token over 4,160 of 16,384 16-bit keys,
//   24 heads: 12.6 us.
// A warp's sums of positive values drift low with the keys that it adds up (the tensor core cuts products to the accumulator's
// exponent): a stream over 96 warps (few streams) 4e-5 of the value at a million tokens, 2e-4 at 4 million, 1.0e-3 at 16;
// over 16 warps (64 streams) 2e-4 at a million; over 4 (max_len far too small) 5e-4, and 2e-3 at 4 million.
#include <algorithm>
#include <type_traits>

#include "h3b_attn_win.cuh"

namespace h3b {

namespace few {
// WIDE: one CTA of twelve warps on an SM, for a handful of (sequence, K/V head) pairs, whose clusters then reach the most
// SMs; else three CTAs of four warps, which fill the chip evenly and hide each other's beginnings and ends.
template <bool KV8, bool WIDE> struct Cfg {
    static constexpr int U = KV8 ? 64 : 32;         // keys of a tile: 8 KiB of keys, 8 KiB of values
    static constexpr int WARPS = WIDE ? 12 : 4, CTAS = WIDE ? 1 : 3, THREADS = WARPS * 32;
    static constexpr int HALF = U * 128 * (KV8 ? 1 : 2), STAGE = 2 * HALF;         // keys | values
    // a warp parks its sums in its stage at the end; pitch and order of a row such that its lanes meet all banks
    static constexpr int PITCH = KV8 ? 136 : 132;
    static_assert(STAGE >= 16 * PITCH * 4, "16 parked rows");
    // stages of the warps | partial results of the CTA (16 rows x 128 f32, m, l) | m, l of the warps | barriers
    static constexpr size_t SMEM_BYTES = 1024 + (size_t)WARPS * STAGE + 16 * 128 * 4 + 2 * 16 * 4 + WARPS * 16 * 8 + WARPS * 16 + 64;
};
}  // namespace few

struct FewParams {
    WinArgs a;
    CUtensorMap map_k, map_v;                      // 16-bit: {d, head, row} box {64, 1, U}; 8-bit: {128, rows} box {128, U}
    int split;                                     // CTAs of a cluster
};

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                               uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                                    uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// transposes an 8x8 matrix of 16-bit values: lane (g, t) has row g, columns 2t, 2t + 1
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
template <typename T> __device__ __forceinline__ float to_f(uint32_t pair, int hi) {
    if (Elem<T>::FMT == 1) return __uint_as_float(hi ? pair & 0xffff0000u : pair << 16);
    return __half2float(__ushort_as_half((unsigned short)(hi ? pair >> 16 : pair & 0xffffu)));
}

// One pass over the keys; true: values that are not finite may have reached rows that do not see them (16-bit; the whole
// cluster alike).  AGAIN: the pass after that, see OddValues.  NT: 8 NT rows.
template <typename T, bool KV8, int NT, bool WIDE, bool AGAIN> __device__ __forceinline__ bool few_pass(const FewParams &p) {
    using C = few::Cfg<KV8, WIDE>;
    using E = typename std::conditional<KV8, __half, T>::type;                     // operand type
    constexpr int U = C::U, WARPS = C::WARPS, STAGE = C::STAGE, HALF = C::HALF;
    constexpr int MT = U / 16;                                                     // score tiles of 16 keys
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *acc = reinterpret_cast<float *>(smem + WARPS * STAGE);                  // [16][128] of this CTA
    float *acc_m = acc + 16 * 128, *acc_l = acc_m + 16;
    float *warp_ml = acc_l + 16;                                                   // [WARPS][16][2]
    uint64_t *bars = reinterpret_cast<uint64_t *>(warp_ml + WARPS * 16 * 2);       // [WARPS][keys | values]
    volatile int *abort_word = reinterpret_cast<volatile int *>(bars + WARPS * 2);
    volatile int *again = abort_word + 1;                                          // 16-bit: the cluster goes over its keys a second time

    const WinArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)blockIdx.x, kvh = blockIdx.y, s = blockIdx.z;
    const SeqExt e = seq_ext<KV8>(a, s);
    const int R = e.nq * a.group;                                                  // rows = query * group + head of the group
    if (!R) return false;                                                          // the whole cluster alike
    const int p0 = e.pos0, p1 = e.pos0 + e.nq - 1;
    const h3b_win_tiles tiles = h3b_win_tiles_of(a.win, p0, p1, e.n, U);
    const h3b_win_row row_a = h3b_win_of(a.win, p0, e.n), row_z = h3b_win_of(a.win, p1, e.n);
    const int share = (tiles.count + p.split - 1) / p.split;
    const int first = rank * share + warp, last = min((rank + 1) * share, tiles.count);
    // (a first pass that gave up a wait may have copies under way still: no more of them)
    const int n_it = first < last && !(AGAIN && *abort_word) ? (last - first + WARPS - 1) / WARPS : 0;

    uint8_t *stage = smem + warp * STAGE;
    uint64_t *bar = bars + warp * 2;
    if (threadIdx.x == 0 && tiles.count) {         // (without keys there are no maps)
        tma_prefetch_desc(&p.map_k);
        tma_prefetch_desc(&p.map_v);
    }
    if (AGAIN && n_it && lane == 0) {
        mbar_inval(&bar[0]);
        mbar_inval(&bar[1]);
        mbar_init(&bar[0], 1);
        mbar_init(&bar[1], 1);
        mbar_fence_init();
    }
    if (!AGAIN && lane == 0) {
        mbar_init(&bar[0], 1);
        mbar_init(&bar[1], 1);
        if (warp == 0) *abort_word = 0, *again = 0;
        mbar_fence_init();
    }
    if (AGAIN) fence_proxy_async_smem();                                           // copies come where rows were parked
    __syncthreads();

    // ---- copies: lane 0 issues, all lanes together look up 32 tiles at a time
    int look_base = 0;
    int my_row = 0;                                // 8-bit: first row of the tile's codes, -1: page outside the pool
    float my_ks = 1.0f, my_vs = 1.0f, my_lvs = 0.0f, my_ivs = 1.0f;   // its scales; log2 and inverse of the value scale
    auto look_up = [&](int it0) {
        look_base = it0;
        if (KV8) {
            const int it = it0 + lane;
            if (it < n_it) {
                const int tile = h3b_win_tile(tiles, first + it * WARPS);
                const long long bi = kv8_block_index(a, s, tile * U / KV8_BLOCK, kvh);
                my_row = bi < 0 ? -1 : (int)(bi * KV8_BLOCK) + tile * U % KV8_BLOCK;
                my_ks = bi < 0 ? 1.0f : __ldg(a.ks + bi);
                my_vs = bi < 0 ? 1.0f : __ldg(a.vs + bi);
            }
        }
    };
    int next_row = 0;                              // of the tile whose keys were asked for last
    float next_ks = 1.0f, next_lvs = 0.0f, next_ivs = 1.0f;
    auto copy = [&](int it, int row, int which) {                                  // which: 0 keys, 1 values
        if (lane == 0) {
            uint8_t *dst = stage + which * HALF;
            mbar_expect_tx(&bar[which], HALF);
            const CUtensorMap *map = which ? &p.map_v : &p.map_k;
            if (KV8) {
                tma_load_2d(dst, map, &bar[which], 0, max(row, 0));
            } else {
                const int key = h3b_win_tile(tiles, first + it * WARPS) * U;
                tma_load_3d(dst, map, &bar[which], 0, kvh, key);
                tma_load_3d(dst + HALF / 2, map, &bar[which], 64, kvh, key);
            }
        }
    };
    auto logs = [&]() {
        if (KV8) {
            my_ks = kv8_read_scale(my_ks);           // (not where they are asked for: the first copies do not wait for them)
            my_vs = kv8_read_scale(my_vs);
            my_lvs = log2f(my_vs);
            my_ivs = 1.0f / my_vs;
        }
    };
    auto take_scales = [&](int src) {
        if (KV8) {
            next_ks = __shfl_sync(0xffffffffu, my_ks, src);
            next_lvs = __shfl_sync(0xffffffffu, my_lvs, src);
            next_ivs = __shfl_sync(0xffffffffu, my_ivs, src);
        }
    };
    auto fetch_keys = [&](int it) {                // page and scales of tile `it` (warp-uniform), then its keys
        if (it - look_base >= 32) {
            look_up(it);
            logs();
        }
        if (KV8) next_row = __shfl_sync(0xffffffffu, my_row, it - look_base);
        take_scales(it - look_base);
        copy(it, next_row, 0);
    };
    if (n_it) {                                    // the first copies do not wait for the scales
        look_up(0);
        if (KV8) next_row = __shfl_sync(0xffffffffu, my_row, 0);
        copy(0, next_row, 0);
        copy(0, next_row, 1);
        logs();
        take_scales(0);
    }

    // ---- Q as the other operand: lane (g, t) has row g of every 8.  16-bit keys: the product's own order of d.  8-bit:
    // lane t takes d = 16 t .. 16 t + 15 and 64 + 16 t .., the 16-byte pieces of a key that it reads.
    uint32_t qf[8][NT][2];
    float row_scale[NT][2];                        // rows 2t, 2t + 1: scale * log2(e), and what brings Q to f16
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = nt * 8 + g;
        const bool live = r < R;
        const int qi = live ? r / a.group : 0, hd = live ? r - qi * a.group : 0;
        const T *src = reinterpret_cast<const T *>(a.q) + (long long)(e.row0 + qi) * a.q_rs + (long long)(kvh * a.group + hd) * a.q_hs;
        float rs = a.scale_log2;
        if (KV8) {
            uint32_t w[16], pair = 0u;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (live) x = __ldg(reinterpret_cast<const uint4 *>(src + (c >> 1) * 64 + t * 16 + (c & 1) * 8));
                w[4 * c] = x.x; w[4 * c + 1] = x.y; w[4 * c + 2] = x.z; w[4 * c + 3] = x.w;
                pair = __vmaxu2(pair, abs_max8_pair(x));
            }
            uint32_t top = max(pair & 0xffffu, pair >> 16);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t bits = widen_abs<T>(top);
            int sh = 14 - ((int)(bits >> 23) - 127);
            sh = bits >= 0x7f800000u || bits == 0u ? 0 : max(min(sh, 120), -120);   // not finite: as it is, so that it reaches the result
            const float up = __uint_as_float((uint32_t)(127 + sh) << 23), down = __uint_as_float((uint32_t)(127 - sh) << 23);
            rs *= down;
#pragma unroll
            for (int i = 0; i < 8; i++)            // step i: words 2i (k 2t, 2t+1) and 2i + 1 (k 2t+8, 2t+9)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    qf[i][nt][j] = Elem<__half>::pack(to_f<T>(w[2 * i + j], 0) * up, to_f<T>(w[2 * i + j], 1) * up);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    qf[i][nt][j] = live ? __ldg(reinterpret_cast<const uint32_t *>(src + i * 16 + j * 8 + t * 2)) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 2; j++) row_scale[nt][j] = KV8 ? __shfl_sync(0xffffffffu, rs, (2 * t + j) * 4) : rs;
    }

    float o[8][NT][4];                             // O^T: 16 dimensions x 8 rows each
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) m_run[nt][0] = m_run[nt][1] = -INFINITY, l_run[nt][0] = l_run[nt][1] = 0.0f;
    // Rows of a tile in shared memory are 128 bytes under the 128-byte swizzle.  8-bit: row g of a 16-key tile is key
    // swap(g) (bits 0 and 2 exchanged), row g + 8 key 8 + swap(g), and a lane's 16 dimensions of a value are piece
    // swap(g), so that the eight lanes of one shared-memory phase meet all eight 16-byte banks.
    const int swap_g = (g & 2) | ((g & 1) << 2) | (g >> 2);
    const int swap_t = ((t & 1) << 1) | (t >> 1);  // swap(2t); swap(2t + 1) = swap_t + 4
    const uint32_t kb = smem_u32(stage), vb = kb + HALF;
    bool ok = true;

    for (int it = 0; it < n_it; it++) {
        const int k0 = h3b_win_tile(tiles, first + it * WARPS) * U;
        const float ks = next_ks, lvs = next_lvs, ivs = next_ivs;
        const bool absent = KV8 && next_row < 0;
        ok = __all_sync(0xffffffffu, mbar_wait(&bar[0], it & 1, abort_word, a.status, H3B_ST_TIMEOUT_FULL));
        if (!ok) break;
        float sc[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) sc[i][nt][0] = sc[i][nt][1] = sc[i][nt][2] = sc[i][nt][3] = 0.0f;
        if (KV8) {
            const uint32_t at0 = kb + swap_g * 128 + ((t ^ swap_g) << 4), at1 = kb + swap_g * 128 + (((t + 4) ^ swap_g) << 4);
            // two tiles at a time: their products do not depend on one another
#pragma unroll
            for (int i = 0; i < MT; i += 2)
#pragma unroll
                for (int h = 0; h < 2; h++) {      // half of the dimensions
                    uint32_t w[2][2][4];           // [tile][row half][word]
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const uint4 x = lds128((h ? at1 : at0) + ((i + u) * 16 + r * 8) * 128);
                            w[u][r][0] = x.x; w[u][r][1] = x.y; w[u][r][2] = x.z; w[u][r][3] = x.w;
                        }
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            uint32_t a0, a1, a2, a3;
                            widen4_e4m3(w[u][0][k], a0, a2);
                            widen4_e4m3(w[u][1][k], a1, a3);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma16816<E>(sc[i + u][nt], a0, a1, a2, a3, qf[4 * h + k][nt][0], qf[4 * h + k][nt][1]);
                        }
                }
        } else {
            const int key = lane & 15;
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const int piece = 2 * k + (lane >> 4);                          // 16-byte piece of d, of 16
                    uint32_t a0, a1, a2, a3;
                    ldsm4(kb + (piece >> 3) * (HALF / 2) + (i * 16 + key) * 128 + (((piece & 7) ^ (key & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma16816<E>(sc[i][nt], a0, a1, a2, a3, qf[k][nt][0], qf[k][nt][1]);
                }
        }
        __syncwarp();                                                               // every lane has read the keys
        if (it + 1 < n_it) fetch_keys(it + 1);

        // exponents: score * scale (+ log2 of the value scale), masked ones -inf; probabilities
        const bool masked = !h3b_win_full(row_a, row_z, k0, U) || absent;
        uint32_t pf[MT][NT][2];                                                     // P^T as operand: keys 2t.. and 2t + 8..
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            bool grow = false;
            float top[2], f[2], off[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (masked) {
                    const h3b_win_row wr = h3b_win_of(a.win, e.pos0 + min(nt * 8 + 2 * t + j, R - 1) / a.group, e.n);
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            if (!h3b_win_sees(wr, k0 + i * 16 + r * 8 + (KV8 ? swap_g : g)) || absent) sc[i][nt][2 * r + j] = -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < MT; i++) mx = fmaxf(mx, fmaxf(sc[i][nt][j], sc[i][nt][2 + j]));
                // factors are positive: the largest score has the largest exponent
                f[j] = KV8 ? row_scale[nt][j] * ks : row_scale[nt][j];
                off[j] = lvs;
                // a lane that sees nothing of the tile: its scales (perhaps NaN) have no part
                if (KV8 && mx == -INFINITY) f[j] = 1.0f, off[j] = 0.0f;
                mx = KV8 ? fmaf(mx, f[j], off[j]) : mx * f[j];
                top[j] = mx;
                grow |= mx > m_run[nt][j] + ProbRange<E>::LAG;                      // also at the first visible key: m_run = -inf
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float mx = top[j];
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float m_new = fmaxf(m_run[nt][j], mx);
                    const float alpha = m_run[nt][j] == -INFINITY ? 0.0f : ex2_approx(m_run[nt][j] - m_new);
                    m_run[nt][j] = m_new;
                    l_run[nt][j] *= alpha;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        o[i][nt][j] *= alpha;
                        o[i][nt][2 + j] *= alpha;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float m_use = m_run[nt][j] == -INFINITY ? 0.0f : m_run[nt][j] - ProbRange<E>::UP, c = (KV8 ? off[j] : 0.0f) - m_use;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float x = ex2_approx(fmaf(sc[i][nt][2 * r + j], f[j], c));
                        sc[i][nt][2 * r + j] = x;
                        sum += x;
                    }
                l_run[nt][j] += KV8 ? (sum == 0.0f ? 0.0f : sum * ivs) : sum;
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int r = 0; r < 2; r++) pf[i][nt][r] = transpose8(Elem<E>::pack(sc[i][nt][2 * r], sc[i][nt][2 * r + 1]));
        }

        ok = __all_sync(0xffffffffu, mbar_wait(&bar[1], it & 1, abort_word, a.status, H3B_ST_TIMEOUT_FULL));
        if (!ok) break;
        if (masked) {
            // a value that no row sees must not meet its zero probability (0 * NaN; behind a cached sequence lie stale
            // bytes): such rows of the tile become zero
#pragma unroll
            for (int i = 0; i < U; i += 32) {
                const int j = k0 + i + lane;
                if (i + lane < U && (j > row_z.hi || (j < row_a.lo && j >= row_z.s))) {
                    uint8_t *dst = stage + HALF + (i + lane) * 128;
#pragma unroll
                    for (int c = 0; c < (KV8 ? 8 : 16); c++)
                        *reinterpret_cast<uint4 *>(dst + (c >> 3) * (HALF / 2) + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();      // the next copy into the stage comes behind these stores
                } else if (AGAIN) {
                    uint8_t *row = stage + HALF + lane * 128;
#pragma unroll 4
                    for (int c = 0; c < 16; c++) {
                        uint4 *at = reinterpret_cast<uint4 *>(row + (c >> 3) * (HALF / 2) + (c & 7) * 16);
                        const uint4 w = *at;
                        *at = make_uint4(finite_or_zero<T>(w.x), finite_or_zero<T>(w.y), finite_or_zero<T>(w.z), finite_or_zero<T>(w.w));
                    }
                    fence_proxy_async_smem();
                }
            }
            __syncwarp();
        }
        // O^T += V^T P^T, 16 keys at a time
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if (KV8) {
                // column c of P^T is key swap(c): lane t has keys swap_t, swap_t + 4 and the same + 8
                uint4 x[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = swap_t + 4 * (r & 1);
                    x[r] = lds128(vb + (i * 16 + (r >> 1) * 8 + key) * 128 + ((swap_g ^ key) << 4));
                }
                const uint32_t w0[4] = {x[0].x, x[0].y, x[0].z, x[0].w}, w1[4] = {x[1].x, x[1].y, x[1].z, x[1].w};
                const uint32_t w2[4] = {x[2].x, x[2].y, x[2].z, x[2].w}, w3[4] = {x[3].x, x[3].y, x[3].z, x[3].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {      // dimensions 4j .. 4j + 3 of the lane's 16: rows g, g + 8 of products 2j, 2j + 1
                    uint32_t lo[4], hi[4];
                    widen4_e4m3(__byte_perm(w0[j], w1[j], 0x5140), lo[0], lo[1]);
                    widen4_e4m3(__byte_perm(w0[j], w1[j], 0x7362), lo[2], lo[3]);
                    widen4_e4m3(__byte_perm(w2[j], w3[j], 0x5140), hi[0], hi[1]);
                    widen4_e4m3(__byte_perm(w2[j], w3[j], 0x7362), hi[2], hi[3]);
#pragma unroll
                    for (int b = 0; b < 2; b++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            mma16816<E>(o[2 * j + b][nt], lo[2 * b], lo[2 * b + 1], hi[2 * b], hi[2 * b + 1], pf[i][nt][0], pf[i][nt][1]);
                }
            } else {
                const int key = i * 16 + (lane & 7) + ((lane >> 4) << 3);           // matrices: d 0-7 | 8-15, then keys + 8
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int piece = 2 * j + ((lane >> 3) & 1);
                    uint32_t a0, a1, a2, a3;
                    ldsm4t(vb + (piece >> 3) * (HALF / 2) + key * 128 + (((piece & 7) ^ (key & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma16816<E>(o[j][nt], a0, a1, a2, a3, pf[i][nt][0], pf[i][nt][1]);
                }
            }
        }
        __syncwarp();                                                               // every lane has read the values
        if (it + 1 < n_it) copy(it + 1, next_row, 1);
    }
    // a wait that gave up: the copies in flight (one on each barrier) get a last, bounded chance to land
    if (!ok)
        for (int i = 0; i < 4; i++)
            for (int spin = 0; spin < 1000 && !mbar_try_wait(&bar[i >> 1], i & 1); spin++) {}

    // ---- meet: warps of the CTA
    float *mine = reinterpret_cast<float *>(stage);                                 // 16 x 128 f32 of this warp
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = nt * 8 + 2 * t + j;
            float l = l_run[nt][j];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (g == 0) {
                warp_ml[(warp * 16 + r) * 2] = m_run[nt][j];
                warp_ml[(warp * 16 + r) * 2 + 1] = l;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (KV8) {
                    *reinterpret_cast<float2 *>(&mine[r * C::PITCH + i * 16 + swap_g * 2]) = make_float2(o[i][nt][j], o[i][nt][2 + j]);   // d = 16 swap_g + 2 i, + 1
                } else {
                    mine[r * C::PITCH + i * 16 + g] = o[i][nt][j];
                    mine[r * C::PITCH + i * 16 + g + 8] = o[i][nt][2 + j];
                }
            }
        }
    if (AGAIN) {
        // rows that see values which were taken out get them back
        const h3b_win_row wr = h3b_win_of(a.win, e.pos0 + min(lane & 15, R - 1) / a.group, e.n);
        OddValues x;
        x.clear();
        for (int it = 0; it < n_it; it++) {
            const int key = h3b_win_tile(tiles, first + it * WARPS) * U;
            if (!h3b_win_full(row_a, row_z, key, U)) x.template collect<T>(a, kvh, key, U, wr, lane < R, lane);
        }
        __syncwarp();
        for (int r = 0; r < R; r++)
            if (x.any(r))
#pragma unroll
                for (int i = 0; i < 4; i++) mine[r * C::PITCH + lane * 4 + i] += x.of(r, i);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * 128; i += C::THREADS) {
        const int r = i >> 7, dim = i & 127, at = r * C::PITCH + (KV8 ? ((dim & 14) << 3) + (dim >> 4 << 1) + (dim & 1) : dim);
        float m = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, warp_ml[(w * 16 + r) * 2]);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float mw = warp_ml[(w * 16 + r) * 2], lw = warp_ml[(w * 16 + r) * 2 + 1];
            const float c = mw == -INFINITY ? 0.0f : ex2_approx(mw - m);
            // a warp whose l is NaN saw something undefined: it counts even if it has no maximum
            l += lw != lw ? lw : c * lw;
            v += c * reinterpret_cast<const float *>(smem + w * STAGE)[at];
        }
        acc[i] = v;
        if ((i & 127) == 0) {
            acc_m[r] = m;
            acc_l[r] = l;
        }
    }
    // ---- CTAs of the cluster: each finishes some rows
    cluster_sync_all();
    const uint32_t acc_addr = smem_u32(acc);
    const int d = threadIdx.x;                                                   // threads 0..127: one dimension each
    bool odd = false;                                                            // not finite, with a finite sum of probabilities
    for (int r = rank; r < R; r += p.split) {
        const int qi = r / a.group, hd = r - qi * a.group;
        if (d < 128) {
            float mc[8], lc[8], vc[8], m = -INFINITY, l = 0.0f, v = 0.0f;            // at most 8 CTAs, all loads under way at once
#pragma unroll
            for (int c = 0; c < 8; c++) {
                if (c >= p.split) break;
                const uint32_t base = mapa_shared(acc_addr, c);
                mc[c] = ld_cluster_f32(base + (16 * 128 + r) * 4);
                lc[c] = ld_cluster_f32(base + (16 * 128 + 16 + r) * 4);
                vc[c] = ld_cluster_f32(base + (r * 128 + d) * 4);
            }
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (c < p.split) m = fmaxf(m, mc[c]);
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (c < p.split) {
                    const float w = mc[c] == -INFINITY ? 0.0f : ex2_approx(mc[c] - m);
                    l += lc[c] != lc[c] ? lc[c] : w * lc[c];
                    v += w * vc[c];
                }
            const float res = h3b_win_count(h3b_win_of(a.win, e.pos0 + qi, e.n)) ? within_type<T, KV8>(v * (1.0f / l)) : 0.0f;
            T *dst = reinterpret_cast<T *>(a.out) + (long long)(e.row0 + qi) * a.o_rs + (long long)(kvh * a.group + hd) * a.o_hs;
            reinterpret_cast<unsigned short *>(dst)[d] = (unsigned short)(Elem<T>::pack(res, res) & 0xffffu);
            odd |= !(fabsf(res) < INFINITY) && ordinary(l);
        }
    }
    if (!KV8 && !AGAIN && odd)                                                   // every CTA of the cluster has to know
        for (int c = 0; c < p.split; c++) st_cluster_u32(mapa_shared(smem_u32(const_cast<const int *>(again)), c), 1u);
    cluster_sync_all();                                                          // nobody leaves while its memory is read
    // rows that see the same hold what they see
    return !KV8 && !AGAIN && *again && (row_a.hi != row_z.hi || row_a.lo != row_z.lo || row_a.s != row_z.s);
}

// A function of its own, so that its registers are no concern of the first pass (as a loop around it, 9 to 18 % slower for 9 to
// 16 rows of 16-bit keys).
template <typename T, int NT, bool WIDE> __device__ __noinline__ void few_again(const FewParams &p) { few_pass<T, false, NT, WIDE, true>(p); }

template <typename T, bool KV8, int NT, bool WIDE> __global__ void __launch_bounds__(few::Cfg<KV8, WIDE>::THREADS, few::Cfg<KV8, WIDE>::CTAS)
k_attn_few(const __grid_constant__ FewParams p) {
    if (few_pass<T, KV8, NT, WIDE, false>(p) && !KV8) few_again<T, NT, WIDE>(p);
}

// How the keys of one (sequence, K/V head, row tile) are shared out.
struct FewPlan {
    bool wide;
    int split;                                     // CTAs of a cluster
};
// Measured on 148 SMs (us; an E4M3 cache unless said otherwise):
//   8 pairs of 100,000 keys: WIDE in clusters of 8 50, of 4 90; narrow of 8 81.  24 pairs of 20,000: WIDE of 5 28.2, narrow of
//   8 27.8, of 1 126.
//   One cluster more than the chip holds is a second wave (20,000 keys): 16 pairs, WIDE of 6 21.6, of 8 32.1; 18 pairs, of 6 22.8,
//   of 7 33.5; narrow, 52 pairs, of 7 47.2, of 8 62.7; 61 pairs, of 6 54.7, of 7 72.4; 107 pairs, of 3 92.0, of 4 107.6.
//   96 pairs of up to 12,000: narrow of 4 (384 CTAs, one wave) 33.6, of 1 77.6, of 5 41.7; WIDE 40.
//   512 pairs of up to 16,000: narrow of 4 157, of 1 182; 1536 pairs of up to 2,000: of 1 80.6, of 2 96.7.
// So: the largest clusters of which one wave takes all pairs, where there are any; beyond that shares of 32 tiles, below which a
// CTA's beginning and end cost more than even shares gain.
static FewPlan few_plan(const h3_cuda *cuda, size_t units, size_t tiles) {
    // the 8-bit kernels stand for the others too: a CTA of a size takes the same shared memory and threads in all of them
    static AttnClusters wide, narrow;
    auto room = [&](bool w, size_t n) {
        return w ? attn_clusters_of(cuda, wide, (const void *)k_attn_few<__half, true, 1, true>, few::Cfg<true, true>::THREADS, few::Cfg<true, true>::SMEM_BYTES, n)
                 : attn_clusters_of(cuda, narrow, (const void *)k_attn_few<__half, true, 1, false>, few::Cfg<true, false>::THREADS, few::Cfg<true, false>::SMEM_BYTES, n);
    };
    const size_t some = std::max<size_t>(tiles / 4, 1);                                 // a tile for every warp of four
    FewPlan p;
    p.wide = room(true, 6) >= units;
    size_t n = std::min<size_t>(some, 8);
    if (p.wide || room(false, 2) >= units)
        while (n > 1 && room(p.wide, n) < units) n--;
    else
        n = std::min<size_t>(std::max<size_t>(tiles / 32, 1), 4);
    p.split = (int)n;
    return p;
}

template <typename T, bool KV8, bool WIDE> static int launch_few_t(h3_cuda *cuda, const FewParams &p, dim3 grid, int nt, char *error, size_t error_size) {
    void (*kernel)(const FewParams) = nt == 1 ? k_attn_few<T, KV8, 1, WIDE> : k_attn_few<T, KV8, 2, WIDE>;
    using C = few::Cfg<KV8, WIDE>;
    static std::atomic<uint64_t> done[2];
    if (!smem_once(cuda, done[nt - 1], (const void *)kernel, C::SMEM_BYTES, "attention smem attribute", error, error_size)) return 0;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = cuda->op_stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    H3B_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p), "k_attn_few launch");
    cuda->launches++;
    return 1;
}

int launch_attn_few(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size) {
    FewParams p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    if (kv8) {
        const uint64_t n = (uint64_t)a.pages * a.kv_heads * a.page_blocks * KV8_BLOCK;
        if (h3b_encode_tmap_2d(&p.map_k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.kc, 128, n, 128, 128, few::Cfg<true, false>::U, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_2d(&p.map_v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.vc, 128, n, 128, 128, few::Cfg<true, false>::U, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "kv8_sdpa: cuTensorMapEncodeTiled failed");
    } else if (a.lk) {
        const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if (h3b_encode_tmap_3d(&p.map_k, dt, 2, a.k, 128, a.kv_heads, a.lk, a.k_hs * 2, a.k_rs * 2, 64, 1, few::Cfg<false, false>::U, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_3d(&p.map_v, dt, 2, a.v, 128, a.kv_heads, a.lk, a.v_hs * 2, a.v_rs * 2, 64, 1, few::Cfg<false, false>::U, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "sdpa_window: cuTensorMapEncodeTiled failed");
    }
    const size_t rows = (size_t)a.max_rows * a.group;
    const int nt = rows <= 8 ? 1 : 2;
    const size_t keys = attn_window_keys(a.win, len, (size_t)a.max_rows);
    const FewPlan plan = few_plan(cuda, (size_t)a.kv_heads * a.n_seq, ceil_div(keys, kv8 ? few::Cfg<true, false>::U : few::Cfg<false, false>::U));
    p.split = plan.split;
    const dim3 grid((unsigned)p.split, (unsigned)a.kv_heads, (unsigned)a.n_seq);
    int (*launch)(h3_cuda *, const FewParams &, dim3, int, char *, size_t);
    if (kv8) launch = f16 ? (plan.wide ? launch_few_t<__half, true, true> : launch_few_t<__half, true, false>)
                          : (plan.wide ? launch_few_t<__nv_bfloat16, true, true> : launch_few_t<__nv_bfloat16, true, false>);
    else launch = f16 ? (plan.wide ? launch_few_t<__half, false, true> : launch_few_t<__half, false, false>)
                      : (plan.wide ? launch_few_t<__nv_bfloat16, false, true> : launch_few_t<__nv_bfloat16, false, false>);
    return launch(cuda, p, grid, nt, error, error_size);
}

}  // namespace h3b
