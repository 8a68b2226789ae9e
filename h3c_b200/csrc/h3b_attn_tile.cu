// Windowed attention for many query rows per K/V head on tcgen05: the tensor core is the bound, so it has to be fed
// without a pause.
//
// One CTA per (256 rows of one K/V head = two 128-row tiles A and B, range of keys).  A row is a (query, head) pair of
// the K/V head's group, queries outermost: shared heads fill tiles with few queries, and K and V are read once for all
// heads of the group.  The key tiles (128 keys) that a CTA visits are the tiles of the sinks and of the union of its
// rows' windows (h3b_window.h); only a tile that some row does not see wholly pays for a mask.
//   warp 0       16-bit: K and V tiles by TMA, two-deep.  8-bit: idle
//   warp 1       MMA issuer: per key tile and row tile S = Q K^T (128x128x128) into TMEM, then O += P V with P from TMEM,
//                the two row tiles interleaved so that the tensor core works on one while the other is in its softmax
//   warps 4-7    softmax of tile A, warps 8-11 of tile B: one row per thread.  They bring Q to shared memory first, read
//                the 128 scores once, and write P back over the score columns in two halves of 64 keys; the accumulator
//                is rescaled only when the running maximum grew by more than 2^8
//   warps 12-15  8-bit: widen the codes of a tile from registers (asked for one tile ahead, 16 bytes per lane, whole
//                128-byte rows) to f16 in the swizzled layout that the MMAs read
// TMEM: S_A 0..127, S_B 128..255 (P overlays the first 64 columns of each), O_A 256..383, O_B 384..511.
//
// 8-bit cache: f16 operands whatever the type of Q (E4M3 fits f16 exactly; Q under a power of two of its row's maximum).
// Scales cost nothing per element: the key scale of 64 keys is part of the factor that the scores are multiplied by
// anyway, log2 of the value scale part of the offset that is subtracted anyway (P carries the value scale), and the row
// sum of 64 keys is divided by it once.
//
// Values that no row of the CTA sees are zeroed on their way (a probability of 0 times a NaN of stale memory is not 0);
// a row that comes out non-finite because of a value that only other rows of its tile see is computed again from its own
// keys.
//
// Few row tiles and many keys: the keys are split over the CTAs of a cluster, whose partial results meet in shared memory.
#include <algorithm>
#include <type_traits>

#include "h3b_attn_win.cuh"

namespace h3b {

namespace wtile {
constexpr int BM = 128, BN = 128, HD = 128;
constexpr int SLAB = 128 * 64 * 2, TILE = 2 * SLAB;       // 128 rows x 64 16-bit values under the 128-byte swizzle; two of them
constexpr int TMEM_COLS = 512;
constexpr uint32_t S_COL = 0, O_COL = 256;                // + 128 * row tile
constexpr int SOFTMAX_WARP = 4, WIDEN_WARP = 12;
constexpr int PART_ROW = 132;                             // floats of a parked row: 16-byte lanes of 8 rows hit all banks
constexpr int CODES = 128 * 128;                          // E4M3 codes of a tile
// Q_A Q_B | K0 K1 | V0 V1 (at the end: parked rows) | 8-bit: codes of a key and of a value tile | barriers | scales
template <bool KV8> constexpr size_t smem_bytes() { return 1024 + 6 * (size_t)TILE + (KV8 ? 2 * CODES : 0) + 512; }
static_assert(256 * PART_ROW * 4 + 2 * 256 * 4 <= 6 * TILE, "parked rows");
}  // namespace wtile

struct TileParams {
    WinArgs a;
    CUtensorMap map_k, map_v;                             // 16-bit: {d, head, row}, box {64, 1, 128}
    int split;                                            // CTAs of a cluster, each with a range of the key tiles
};

// largest of three, NaN if one is NaN
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t widen2_e4m3(uint16_t w) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
    return r;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float ld_cluster_f(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <bool KV8> struct TileCfg {
    static constexpr int THREADS = KV8 ? 512 : 384;
    // 8-bit: 512 threads start with 128 registers each, 72 + 2 * 184 + 72 = 4 * 128; 16-bit: 384 with 168, 88 + 2 * 208 = 3 * 168
    static constexpr int REG_ISSUE = KV8 ? 72 : 88, REG_SOFTMAX = KV8 ? 184 : 208, REG_WIDEN = 72;
};

// EMU: bit q set = the q-th group of four probabilities of every 32 on the FMA pipe (ex2_emu2)
template <typename T, bool KV8, uint32_t EMU>
__global__ void __launch_bounds__(TileCfg<KV8>::THREADS, 1) k_attn_tile(const __grid_constant__ TileParams p) {
    using namespace wtile;
    using C = TileCfg<KV8>;
    using E = typename std::conditional<KV8, __half, T>::type;          // operand type
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = smem, *sK = smem + 2 * TILE, *sV = smem + 4 * TILE, *sC = smem + 6 * TILE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sC + (KV8 ? 2 * CODES : 0));
    uint64_t *q_full = bars, *k_full = bars + 1, *v_full = bars + 3, *k_empty = bars + 5, *v_empty = bars + 7, *s_full = bars + 9,
             *p_full = bars + 11 /* [tile][half] */, *o_done = bars + 15, *v_raw = bars + 16;
    uint64_t *c_full = bars + 17 /* [keys, values] */, *c_empty = bars + 19;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 21);
    volatile int *abort_word = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float4 *scales = reinterpret_cast<float4 *>(bars + 24);               // [4]: key scale of either half, value scale of either half

    const WinArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % p.split, kvh = blockIdx.y, s = blockIdx.z;
    const SeqExt e = seq_ext<KV8>(a, s);
    const int r0 = ((int)blockIdx.x / p.split) * (2 * BM);
    const long long rows_all = (long long)e.nq * a.group;
    if (r0 >= rows_all) return;                                          // the whole cluster alike
    const int r_end = (int)(rows_all < r0 + 2 * BM ? rows_all : r0 + 2 * BM);
    const int n_tiles = r_end - r0 > BM ? 2 : 1;
    const h3b_win_tiles tiles = h3b_win_tiles_of(a.win, e.pos0 + r0 / a.group, e.pos0 + (r_end - 1) / a.group, e.n, BN);
    const h3b_win_row row_a = h3b_win_of(a.win, e.pos0 + r0 / a.group, e.n), row_z = h3b_win_of(a.win, e.pos0 + (r_end - 1) / a.group, e.n);
    const int share = (tiles.count + p.split - 1) / p.split;
    const int t_first = rank * share, n_kv = max(min(t_first + share, tiles.count) - t_first, 0);
    auto key_of = [&](int j) { return h3b_win_tile(tiles, t_first + j) * BN; };
    // no row of the CTA sees key j
    auto hidden = [&](int j) { return j > row_z.hi || (j < row_a.lo && j >= row_z.s); };

    if (threadIdx.x == 0) {
        mbar_init(q_full, 8);
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], KV8 ? 4 : 1);
            mbar_init(&v_full[i], KV8 ? 4 : 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
        }
        mbar_init(o_done, 1);
        mbar_init(v_raw, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&c_full[i], 1);
            mbar_init(&c_empty[i], 4);
        }
        *abort_word = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    bool ok = true;

    if (warp < SOFTMAX_WARP) {
        regs_dec<C::REG_ISSUE>();
        if (warp == 0 && !KV8) {
            // ------------------------------------------------------------ K and V by TMA
            uint32_t raw = 0;
            for (int j = 0; j < n_kv && ok; j++) {
                const int st = j & 1, key = key_of(j);
                const uint32_t ph = ((j >> 1) & 1) ^ 1;
                ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ph, abort_word, a.status, H3B_ST_TIMEOUT_EMPTY));
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(&k_full[st], TILE);
                    tma_load_3d(sK + st * TILE, &p.map_k, &k_full[st], 0, kvh, key);
                    tma_load_3d(sK + st * TILE + SLAB, &p.map_k, &k_full[st], 64, kvh, key);
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ph, abort_word, a.status, H3B_ST_TIMEOUT_EMPTY));
                if (!ok) break;
                // keys of the tile that no row sees (those behind the last key come as zeros)
                const int key_end = min(key + BN, e.n);
                const bool unseen = key_end - 1 > row_z.hi || (max(key, row_z.s) < min(key_end, row_a.lo));
                if (lane == 0) {
                    uint64_t *b = unseen ? v_raw : &v_full[st];
                    mbar_expect_tx(b, TILE);
                    tma_load_3d(sV + st * TILE, &p.map_v, b, 0, kvh, key);
                    tma_load_3d(sV + st * TILE + SLAB, &p.map_v, b, 64, kvh, key);
                }
                if (unseen) {
                    ok = __all_sync(0xffffffffu, mbar_wait(v_raw, raw & 1, abort_word, a.status, H3B_ST_TIMEOUT_FULL));
                    if (!ok) break;
                    raw++;
                    for (int i = lane; i < BN; i += 32)
                        if (hidden(key + i))
                            for (int c = 0; c < 16; c++)
                                *reinterpret_cast<uint4 *>(sV + st * TILE + (c >> 3) * SLAB + i * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[st]);
                }
            }
        } else if (warp == 0 && n_kv > 0) {
            // ------------------------------------------------------------ codes of the pages by bulk copies, 64 tokens each
            // (8 KiB that lie together).  Lanes look up the blocks of 16 tiles at a time.
            int look = 0, bi = -1;
            float bks = 1.0f, bvs = 1.0f;
            for (int j = 0; j < n_kv && ok; j++) {
                if (j % 16 == 0) {
                    look = j;
                    bi = -1;
                    const int jj = j + (lane >> 1);
                    if (jj < n_kv) {
                        const int blk = key_of(jj) / KV8_BLOCK + (lane & 1);
                        if (blk * KV8_BLOCK < e.n) bi = (int)kv8_block_index(a, s, blk, kvh);
                    }
                    bks = bi >= 0 ? __ldg(a.ks + bi) : 1.0f;
                    bvs = bi >= 0 ? __ldg(a.vs + bi) : 1.0f;
                }
                const int src = 2 * (j - look);
                const int b0 = __shfl_sync(0xffffffffu, bi, src), b1 = __shfl_sync(0xffffffffu, bi, src + 1);
                const float4 sc = make_float4(__shfl_sync(0xffffffffu, bks, src), __shfl_sync(0xffffffffu, bks, src + 1),
                                              __shfl_sync(0xffffffffu, bvs, src), __shfl_sync(0xffffffffu, bvs, src + 1));
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&c_empty[w], (j & 1) ^ 1, abort_word, a.status, H3B_ST_TIMEOUT_EMPTY));
                    if (!ok) break;
                    if (lane == 0) {
                        // scales of tile j: the softmax warps read them behind s_full(j); the slot is that of tile j - 4,
                        // whose scores were done with before the codes of tile j - 1 could be widened
                        if (w == 0) scales[j & 3] = sc;
                        const uint8_t *codes = w ? a.vc : a.kc;
                        // a block outside the pool (reported) or behind the last token is not read: its rows are hidden or invalid
                        mbar_expect_tx(&c_full[w], (b0 >= 0 ? CODES / 2 : 0) + (b1 >= 0 ? CODES / 2 : 0));
                        if (b0 >= 0) bulk_load(sC + w * CODES, codes + (long long)b0 * (CODES / 2), CODES / 2, &c_full[w]);
                        if (b1 >= 0) bulk_load(sC + w * CODES + CODES / 2, codes + (long long)b1 * (CODES / 2), CODES / 2, &c_full[w]);
                    }
                }
            }
        } else if (warp == 1 && n_kv > 0) {
            // ------------------------------------------------------------ MMA issuer
            // The whole warp walks the loop, converged; one lane, elected once, issues every tcgen05 instruction.  The
            // stage barriers of the next iteration are polled behind an issued block, while the queue drains.
            const bool lead = elect_one();
            constexpr uint32_t idesc_s = umma_idesc(1, Elem<E>::FMT, Elem<E>::FMT, BM, BN, 0, 0);
            constexpr uint32_t idesc_o = umma_idesc(1, Elem<E>::FMT, Elem<E>::FMT, BM, HD, 0, 1);
            constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);   // SBO 1024, version 1, 128-byte swizzle
            const uint32_t q_lo0 = ((smem_u32(sQ) & 0x3ffffu) >> 4) | (1u << 16), q_lo1 = q_lo0 + (TILE >> 4);
            const uint32_t k_lo0 = ((smem_u32(sK) & 0x3ffffu) >> 4) | (1u << 16);
            const uint32_t v_lo0 = ((smem_u32(sV) & 0x3ffffu) >> 4) | ((uint32_t)((SLAB >> 4) & 0x3fff) << 16);   // LBO = slab
            auto issue_s = [&](int t, int stage) {
                const uint32_t qa = t ? q_lo1 : q_lo0, kb = k_lo0 + (uint32_t)stage * (TILE >> 4);
                const uint32_t d_tmem = tmem_base + S_COL + 128u * t;
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t c = (uint32_t)(k >> 2) * (SLAB >> 4) + (uint32_t)(k & 3) * 2;
                    if (lead) umma_f16_ss_lh(d_tmem, qa + c, kb + c, DESC_HI, idesc_s, (uint32_t)(k != 0));
                }
                if (lead) tc_commit(&s_full[t]);
            };
            auto issue_pv = [&](int t, int stage, int half, bool first) {
                const uint32_t vb = v_lo0 + (uint32_t)stage * (TILE >> 4);
#pragma unroll
                for (int k = half * (BN / 32); k < (half + 1) * (BN / 32); k++)
                    if (lead)
                        umma_f16_ts_lh(tmem_base + O_COL + 128u * t, tmem_base + S_COL + 128u * t + (uint32_t)k * 8,
                                       vb + (uint32_t)k * (2048 >> 4), DESC_HI, idesc_o, (uint32_t)(!first || k != 0));
            };
            auto wait = [&](uint64_t *b, uint32_t parity, int code) {
                return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_word, a.status, code)) != 0;
            };
            ok = wait(q_full, 0, H3B_ST_TIMEOUT_OTHER) && wait(&k_full[0], 0, H3B_ST_TIMEOUT_FULL);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < n_tiles; t++) issue_s(t, 0);
                if (lead) tc_commit(&k_empty[0]);
                ok = wait(&v_full[0], 0, H3B_ST_TIMEOUT_FULL) && (n_kv < 2 || wait(&k_full[1], 0, H3B_ST_TIMEOUT_FULL));
            }
            auto step = [&](int j, auto stage_c) {
                constexpr int st = decltype(stage_c)::value, nx = st ^ 1;
                const bool more = j + 1 < n_kv;
                for (int t = 0; t < n_tiles && ok; t++) {
                    ok = wait(&p_full[2 * t], j & 1, H3B_ST_TIMEOUT_OTHER);
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(t, st, 0, j == 0);
                    ok = wait(&p_full[2 * t + 1], j & 1, H3B_ST_TIMEOUT_OTHER);
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(t, st, 1, false);
                    if (t == n_tiles - 1 && lead) tc_commit(&v_empty[st]);
                    if (more) {
                        issue_s(t, nx);
                        if (t == n_tiles - 1 && lead) tc_commit(&k_empty[nx]);
                    }
                }
                if (ok && more) {
                    ok = wait(&v_full[nx], ((j + 1) >> 1) & 1, H3B_ST_TIMEOUT_FULL);
                    if (ok && j + 2 < n_kv) ok = wait(&k_full[st], ((j + 2) >> 1) & 1, H3B_ST_TIMEOUT_FULL);
                    tc_fence_after();
                }
            };
            for (int j = 0; ok && j < n_kv; j += 2) {
                step(j, std::integral_constant<int, 0>{});
                if (ok && j + 1 < n_kv) step(j + 1, std::integral_constant<int, 1>{});
            }
            if (lead) tc_commit(o_done);
        }
        __syncwarp();
    } else if (warp < WIDEN_WARP) {
        // ---------------------------------------------------------------- softmax
        regs_inc<C::REG_SOFTMAX>();
        const int t = (warp - SOFTMAX_WARP) >> 2, q = warp & 3;          // row tile, TMEM lane quarter
        const int my = r0 + t * BM + q * 32 + lane;                      // row of this thread
        const bool live = my < r_end;
        const int qi = (live ? my : r_end - 1) / a.group, hd = (live ? my : r_end - 1) - qi * a.group;
        float row_scale = a.scale_log2;
        if (t < n_tiles && n_kv) {                                       // without keys the memory is the epilogue's at once
            // Q -> shared memory, sixteen lanes per 256-byte row (8-bit: f16 under a power of two of the row's maximum,
            // undone by row_scale)
            const long long mine = live ? (long long)(e.row0 + qi) * a.q_rs + (long long)(kvh * a.group + hd) * a.q_hs : -1;
            const int sub = lane >> 4, c = lane & 15;
            uint4 w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const long long off = __shfl_sync(0xffffffffu, mine, 2 * i + sub);
                w[i] = off >= 0 ? __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.q) + off) + c) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (KV8) {
                    uint32_t top = abs_max8<T>(w[i]);
#pragma unroll
                    for (int x = 1; x < 16; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const uint32_t bits = widen_abs<T>(top);
                    int sh = 14 - ((int)(bits >> 23) - 127);
                    sh = bits >= 0x7f800000u || bits == 0u ? 0 : max(min(sh, 120), -120);   // not finite: as it is
                    const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
                    const int down = __shfl_sync(0xffffffffu, 127 - sh, (lane & 1) * 16);
                    if ((lane >> 1) == i) row_scale *= __uint_as_float((uint32_t)down << 23);
                    uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float2 f;
                        if (Elem<T>::FMT == 1) f = make_float2(__uint_as_float(v[k] << 16), __uint_as_float(v[k] & 0xffff0000u));
                        else f = __half22float2(*reinterpret_cast<const __half2 *>(&v[k]));
                        v[k] = Elem<__half>::pack(f.x * up, f.y * up);
                    }
                    w[i] = make_uint4(v[0], v[1], v[2], v[3]);
                }
                const int row = q * 32 + 2 * i + sub;
                *reinterpret_cast<uint4 *>(sQ + t * TILE + (c >> 3) * SLAB + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = w[i];
            }
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);

        const uint32_t lane_base = (uint32_t)(q * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + S_COL + 128u * t, o_addr = tmem_base + lane_base + O_COL + 128u * t;
        const h3b_win_row wr = h3b_win_of(a.win, e.pos0 + qi, e.n);
        const h3b_win_row wa = h3b_win_of(a.win, e.pos0 + (r0 + t * BM) / a.group, e.n);
        const h3b_win_row wz = h3b_win_of(a.win, e.pos0 + (min(r0 + t * BM + BM, r_end) - 1) / a.group, e.n);
        float m_run = -INFINITY, l_run = 0.0f;
        ok = t < n_tiles;
        for (int j = 0; j < n_kv && ok; j++) {
            const int key = key_of(j);
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, abort_word, a.status, H3B_ST_TIMEOUT_TMEM_FULL));
            if (!ok) break;
            tc_fence_after();
            uint32_t sv[BN];
#pragma unroll
            for (int ch = 0; ch < BN / 32; ch++) tmem_ld_32x32b_x32(s_addr + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[ch * 32]));
            tmem_ld_wait();
            if (!h3b_win_full(wa, wz, key, BN)) {
#pragma unroll
                for (int ch = 0; ch < BN / 32; ch++) {
                    // bits of the 32 keys that the row sees
                    const int b = wr.hi - key - ch * 32, lo = wr.lo - key - ch * 32, sn = wr.s - key - ch * 32;
                    const uint32_t upto = b >= 31 ? 0xffffffffu : b < 0 ? 0u : (2u << b) - 1u;
                    const uint32_t from = lo <= 0 ? 0xffffffffu : lo > 31 ? 0u : 0xffffffffu << lo;
                    const uint32_t sink = sn <= 0 ? 0u : sn > 31 ? 0xffffffffu : (1u << sn) - 1u;
                    const uint32_t see = upto & (from | sink);
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (!(see >> i & 1u)) sv[ch * 32 + i] = 0xff800000u;
                }
            }
            float mxh[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float mxc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; i += 8)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        mxc[c] = max3_nan(mxc[c], __uint_as_float(sv[h * 64 + i + 2 * c]), __uint_as_float(sv[h * 64 + i + 2 * c + 1]));
                mxh[h] = max3_nan(max3_nan(mxc[0], mxc[1], mxc[2]), mxc[3], mxc[3]);
            }
            float f[2] = {row_scale, row_scale}, off[2] = {0.0f, 0.0f}, inv_vs[2] = {1.0f, 1.0f};
            float mx;
            if (KV8) {
                const float4 sc = scales[j & 3];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float vs = h ? sc.w : sc.z;
                    f[h] = row_scale * (h ? sc.y : sc.x);
                    off[h] = log2f(vs);
                    inv_vs[h] = 1.0f / vs;
                    // nothing of the 64 seen: its scales (of another sequence's tokens, or NaN) have no part
                    if (mxh[h] == -INFINITY) f[h] = 1.0f, off[h] = 0.0f, inv_vs[h] = 1.0f;
                    mxh[h] = fmaf(mxh[h], f[h], off[h]);
                }
                mx = max3_nan(mxh[0], mxh[1], mxh[1]);
            } else {
                mx = max3_nan(mxh[0], mxh[1], mxh[1]) * row_scale;
            }
            if (mx != mx) l_run = mx;                                    // undefined, and so is the row from here on
            const float m_new = fmaxf(m_run, mx);
            const bool grow = m_new > m_run + 8.0f || (m_run == -INFINITY && m_new > -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
                float alpha = 1.0f;
                if (grow) {
                    alpha = m_run == -INFINITY ? 0.0f : ex2_approx(m_run - m_new);
                    m_run = m_new;
                    l_run *= alpha;
                }
                // s_full of tile j came behind the P V product of tile j - 1: the accumulator is at rest
                if (j > 0) {
#pragma unroll 1
                    for (int ch = 0; ch < HD / 16; ch++) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_addr + ch * 16, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st_32x32b_x16(o_addr + ch * 16, o);
                    }
                }
            }
            const float m_use = m_run == -INFINITY ? 0.0f : m_run;
            float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
            auto chunk = [&](int ch, uint32_t (&packed)[16]) {
                const float fh = f[ch >> 1], c = KV8 ? off[ch >> 1] - m_use : -m_use;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float x0, x1, x2, x3;
                    fma2(x0, x1, __uint_as_float(sv[ch * 32 + i]), __uint_as_float(sv[ch * 32 + i + 1]), fh, c);
                    fma2(x2, x3, __uint_as_float(sv[ch * 32 + i + 2]), __uint_as_float(sv[ch * 32 + i + 3]), fh, c);
                    float p0, p1, p2, p3;
                    if ((EMU >> (i >> 2)) & 1u) {
                        ex2_emu2(p0, p1, x0, x1);
                        ex2_emu2(p2, p3, x2, x3);
                    } else {
                        p0 = ex2_approx(x0); p1 = ex2_approx(x1); p2 = ex2_approx(x2); p3 = ex2_approx(x3);
                    }
                    add2(l0, l1, p0, p1);
                    add2(l2, l3, p2, p3);
                    packed[i >> 1] = Elem<E>::pack(p0, p1);
                    packed[(i >> 1) + 1] = Elem<E>::pack(p2, p3);
                }
            };
            auto hand_over = [&](int half) {
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
            };
            uint32_t pk[16];
            chunk(0, pk);
            tmem_st_32x32b_x16(s_addr, pk);
            chunk(1, pk);
            tmem_st_32x32b_x16(s_addr + 16, pk);
            if (KV8) {
                l_run += ((l0 + l1) + (l2 + l3)) * inv_vs[0];
                l0 = l1 = l2 = l3 = 0.0f;
            }
            chunk(2, pk);
            hand_over(0);
            tmem_st_32x32b_x16(s_addr + 32, pk);
            chunk(3, pk);
            tmem_st_32x32b_x16(s_addr + 48, pk);
            hand_over(1);
            l_run += ((l0 + l1) + (l2 + l3)) * (KV8 ? inv_vs[1] : 1.0f);
        }
        if (t < n_tiles) {
            if (ok && n_kv) ok = __all_sync(0xffffffffu, mbar_wait(o_done, 0, abort_word, a.status, H3B_ST_TIMEOUT_OTHER));
            tc_fence_after();
            const bool seen = live && h3b_win_count(wr) > 0;
            if (p.split > 1) {
                // this CTA's share of the row: sums as they are, with their maximum and denominator
                const int slot = t * BM + q * 32 + lane;
                float *part = reinterpret_cast<float *>(smem) + slot * PART_ROW;
#pragma unroll 1
                for (int ch = 0; ch < HD / 32; ch++) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + ch * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4 *>(part + ch * 32 + i) =
                            n_kv ? make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]) : make_uint4(0u, 0u, 0u, 0u);
                }
                float *ml = reinterpret_cast<float *>(smem) + 2 * BM * PART_ROW;
                ml[slot] = m_run;
                ml[2 * BM + slot] = l_run;
            } else {
                const float inv_l = 1.0f / l_run;
                // Lane = row here; the rows of the warp are parked in (now free) tile memory and written out sixteen lanes
                // per 256-byte head slice.
                constexpr int STG_ROW = 256 + 16;
                uint8_t *stg = smem + (size_t)(warp - SOFTMAX_WARP) * 32 * STG_ROW;
                bool odd = false;
#pragma unroll 1
                for (int ch = 0; ch < HD / 32; ch++) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + ch * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t h[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const float x = __uint_as_float(o[i + 2 * u]) * inv_l, y = __uint_as_float(o[i + 2 * u + 1]) * inv_l;
                            if (!KV8) odd |= !(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY);
                            h[u] = Elem<T>::pack(x, y);
                        }
                        *reinterpret_cast<uint4 *>(stg + lane * STG_ROW + (ch * 32 + i) * 2) =
                            seen ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                __syncwarp();
                const int sub = lane >> 4, chunk = lane & 15;
#pragma unroll
                for (int k2 = 0; k2 < 16; k2++) {
                    const int rr = 2 * k2 + sub, row = r0 + t * BM + q * 32 + rr;
                    if (ok && row < r_end) {
                        const int qr = row / a.group;
                        T *dst = reinterpret_cast<T *>(a.out) + (long long)(e.row0 + qr) * a.o_rs + (long long)(kvh * a.group + row - qr * a.group) * a.o_hs;
                        *reinterpret_cast<uint4 *>(dst + chunk * 8) = *reinterpret_cast<const uint4 *>(stg + rr * STG_ROW + chunk * 16);
                    }
                }
                if (!KV8) {
                    __syncwarp();
                    uint32_t again = __ballot_sync(0xffffffffu, ok && seen && odd);
                    while (again) {
                        const int row = r0 + t * BM + q * 32 + (__ffs(again) - 1);
                        again &= again - 1;
                        attn_row_by_warp<T, KV8>(a, s, e, row / a.group, kvh * a.group + row % a.group, lane);
                    }
                }
            }
        }
    } else if (KV8) {
        // ---------------------------------------------------------------- widen the codes of a tile
        regs_dec<C::REG_WIDEN>();
        const int w4 = warp - WIDEN_WARP, sub = lane >> 3, piece = lane & 7;   // row within four, 16 codes of the row
        // 16 codes -> 32 bytes: pieces 2 * (piece & 3), + 1 of slab piece >> 2; lanes of the second slab write their second
        // piece first, so that the eight lanes of a row hit all banks
        const int second = piece >> 2, c = 2 * (piece & 3);
        auto widen = [&](uint8_t *tile, const uint8_t *codes, int key, bool unseen) {
            uint4 raw[8];
#pragma unroll
            for (int i = 0; i < 8; i++) raw[i] = *reinterpret_cast<const uint4 *>(codes + (i * 16 + w4 * 4 + sub) * 128 + piece * 16);
            if (unseen)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (hidden(key + i * 16 + w4 * 4 + sub)) raw[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int row = i * 16 + w4 * 4 + sub;
                const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                uint32_t h[8];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    h[2 * k] = widen2_e4m3((uint16_t)(v[k] & 0xffffu));
                    h[2 * k + 1] = widen2_e4m3((uint16_t)(v[k] >> 16));
                }
                const uint4 x = make_uint4(h[0], h[1], h[2], h[3]), y = make_uint4(h[4], h[5], h[6], h[7]);
                uint8_t *dst = tile + second * SLAB + row * 128;
                *reinterpret_cast<uint4 *>(dst + (((c + second) ^ (row & 7)) << 4)) = second ? y : x;
                *reinterpret_cast<uint4 *>(dst + (((c + 1 - second) ^ (row & 7)) << 4)) = second ? x : y;
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        for (int j = 0; j < n_kv && ok; j++) {
            const int st = j & 1, key = key_of(j);
            const uint32_t ph = ((j >> 1) & 1) ^ 1;
            const bool unseen = hidden(key + BN - 1) || hidden(key) || (key < row_a.lo && key + BN > row_z.s);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                ok = __all_sync(0xffffffffu, mbar_wait(&c_full[w], j & 1, abort_word, a.status, H3B_ST_TIMEOUT_FULL) &&
                                                 mbar_wait(w ? &v_empty[st] : &k_empty[st], ph, abort_word, a.status, H3B_ST_TIMEOUT_EMPTY));
                if (!ok) break;
                widen((w ? sV : sK) + st * TILE, sC + w * CODES, key, unseen);
                if (lane == 0) {
                    mbar_arrive(w ? &v_full[st] : &k_full[st]);
                    mbar_arrive(&c_empty[w]);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
    if (p.split > 1) {
        // ---- the shares meet: a warp finishes a row, a lane four of its dimensions
        cluster_sync_all();
        const uint32_t base = smem_u32(smem);
        const int rows = r_end - r0;
        for (int r = rank * (C::THREADS / 32) + warp; r < rows; r += p.split * (C::THREADS / 32)) {
            float m = -INFINITY, l = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < p.split; c++) m = fmaxf(m, ld_cluster_f(mapa_shared(base, c) + (2 * BM * PART_ROW + r) * 4));
            for (int c = 0; c < p.split; c++) {
                const uint32_t peer = mapa_shared(base, c);
                const float mc = ld_cluster_f(peer + (2 * BM * PART_ROW + r) * 4), lc = ld_cluster_f(peer + (2 * BM * PART_ROW + 2 * BM + r) * 4);
                const float w = mc == -INFINITY ? 0.0f : ex2_approx(mc - m);
                const float4 x = ld_cluster_f32x4(peer + (r * PART_ROW + lane * 4) * 4);
                l += lc != lc ? lc : w * lc;
                v.x += w * x.x; v.y += w * x.y; v.z += w * x.z; v.w += w * x.w;
            }
            const int qi = (r0 + r) / a.group, hd = (r0 + r) - qi * a.group;
            const bool seen = h3b_win_count(h3b_win_of(a.win, e.pos0 + qi, e.n)) > 0;
            const float inv = 1.0f / l;
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            const bool odd = !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY) || !(fabsf(v.z) < INFINITY) || !(fabsf(v.w) < INFINITY);
            if (!KV8 && seen && __any_sync(0xffffffffu, odd)) {
                attn_row_by_warp<T, KV8>(a, s, e, qi, kvh * a.group + hd, lane);
                continue;
            }
            T *dst = reinterpret_cast<T *>(a.out) + (long long)(e.row0 + qi) * a.o_rs + (long long)(kvh * a.group + hd) * a.o_hs;
            uint2 w = make_uint2(0u, 0u);
            if (seen) w = make_uint2(Elem<T>::pack(v.x, v.y), Elem<T>::pack(v.z, v.w));
            *reinterpret_cast<uint2 *>(dst + lane * 4) = w;
        }
        cluster_sync_all();                                              // nobody leaves while its memory is read
    }
}

template <typename T, bool KV8> static int launch_tile_t(h3_cuda *cuda, const TileParams &p, dim3 grid, char *error, size_t error_size) {
    void (*kernel)(const TileParams) = k_attn_tile<T, KV8, 0x11>;
    H3B_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wtile::smem_bytes<KV8>()), "attention smem attribute");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(TileCfg<KV8>::THREADS);
    cfg.dynamicSmemBytes = wtile::smem_bytes<KV8>();
    cfg.stream = cuda->op_stream;
    cfg.attrs = &attr;
    cfg.numAttrs = p.split > 1 ? 1 : 0;
    H3B_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p), "k_attn_tile launch");
    cuda->launches++;
    return 1;
}

int launch_attn_tile(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size) {
    TileParams p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    if (!kv8 && a.lk) {
        const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if (h3b_encode_tmap_3d(&p.map_k, dt, 2, a.k, 128, a.kv_heads, a.lk, a.k_hs * 2, a.k_rs * 2, 64, 1, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_3d(&p.map_v, dt, 2, a.v, 128, a.kv_heads, a.lk, a.v_hs * 2, a.v_rs * 2, 64, 1, 128, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "sdpa_window: cuTensorMapEncodeTiled failed");
    }
    const size_t mtiles = ceil_div((size_t)a.max_rows * a.group, 2 * wtile::BM);
    const size_t units = mtiles * a.kv_heads * a.n_seq;
    const size_t tiles = std::max<size_t>(ceil_div(attn_window_keys(a.win, len, std::min<size_t>(a.max_rows, 2 * wtile::BM)), wtile::BN), 1);
    p.split = units >= (size_t)cuda->sm_count ? 1 : (int)std::min(std::min<size_t>((size_t)cuda->sm_count / units, 8), std::max<size_t>(tiles / 2, 1));
    if (getenv("TILE_SPLIT")) p.split = atoi(getenv("TILE_SPLIT"));
    const dim3 grid((unsigned)(mtiles * p.split), (unsigned)a.kv_heads, (unsigned)a.n_seq);
    if (kv8) return f16 ? launch_tile_t<__half, true>(cuda, p, grid, error, error_size) : launch_tile_t<__nv_bfloat16, true>(cuda, p, grid, error, error_size);
    return f16 ? launch_tile_t<__half, false>(cuda, p, grid, error, error_size) : launch_tile_t<__nv_bfloat16, false>(cuda, p, grid, error, error_size);
}

}  // namespace h3b
