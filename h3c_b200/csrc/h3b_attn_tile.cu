// Windowed attention for many query rows per K/V head on tcgen05: the tensor core is the bound, so it has to be fed
// without a pause.
//
// A work item is (two row tiles A and B of one K/V head, range of keys).  A row is a (query, head) pair of the K/V head's
// group, queries outermost: shared heads fill tiles with few queries, and K and V are read once for all heads of the
// group.  A tile holds as many whole queries as fit 128 rows (126 rows for groups of 3, 6, 7), so that one TMA box of
// {64 dimensions, group, queries} brings half of its Q.  The key tiles (128 keys) that an item visits are the tiles of the
// sinks and of the union of its rows' windows (h3b_window.h); only a tile that some row does not see wholly pays for a mask.
// A CTA stays on its SM and takes item after item (cluster launch control hands it the CTAs that have not started yet,
// in grid order, so the chip balances itself), and the roles run ahead into the next item: its Q, K and V arrive while
// the last softmax and the stores of the current one are under way.  With one item per CTA, a window of 256 keys took
// 17 us per item, 8 of them waiting for Q and the first keys and 4 storing; frames of the 6,144-token step 234 us.
//   warp 0       16-bit: K and V tiles by TMA; 8-bit: the codes of a tile by bulk copies, one tile ahead
//   warp 1       MMA issuer: per key tile and row tile S = Q K^T (128x128x128) into TMEM, then O += P V with P from TMEM,
//                the two row tiles interleaved so that the tensor core works on one while the other is in its softmax
//   warp 2       Q of the next item by TMA as soon as the last S of the current one has been computed (by ordinary loads,
//                one warp takes 12 us for the 64 KiB, eight warps 7)
//   warp 3       the next item; 16-bit: zeroes the value rows of edge tiles that no row sees; 8-bit: helps to convert Q
//   warps 4-7    softmax of tile A, warps 8-11 of tile B: one row per thread.  They read the 128 scores once, write P back
//                over the score columns in two halves of 64 keys, and store the rows at the end; the accumulator is
//                rescaled only when the running maximum grew by more than ProbRange says
//   warps 12-15  8-bit: widen the codes of a tile to f16 in the swizzled layout that the MMAs read
// TMEM: S_A 0..127, S_B 128..255 (P overlays the first 64 columns of each), O_A 256..383, O_B 384..511.
//
// 8-bit cache: f16 operands whatever the type of Q (E4M3 fits f16 exactly; bf16 rows of Q go to f16 under a power of two of
// their maximum).  Scales cost nothing per element: the key scale of 64 keys is part of the factor that the scores are
// multiplied by anyway, log2 of the value scale part of the offset that is subtracted anyway (P carries the value scale),
// and the row sum of 64 keys is divided by it once.
//
// Values that no row of the item sees are zeroed on their way (a probability of 0 times a NaN of stale memory is not 0).
// 16-bit: an item with a row that comes out non-finite though its probabilities are finite is done a second time, as a further
// item of its CTA, with the values that are not finite taken out of the tiles that its rows see in part (OddValues).  The
// warp that hands out items learns of it with the third item after, or at the end, so that nothing waits for it in between.
//
// Few items and many keys: the keys are split over the CTAs of a cluster (one item each), whose partial results meet in
// shared memory.
//
// Measured (B200; TFLOP/s of visible pairs): frames of the 6,144-token step (24 heads, three frames and the first) 195-199 us
// = 1165-1190, 226-239 us in a long run at the 1000 W limit; 50,220-token video (eight frames back and the first) 7.6-7.8 ms =
// 1100-1125, at the limit all the time; full attention over 6,144 tokens 379-381 us against 360 of k_attn, which needs
// no edge, item and maximum-of-nothing arithmetic; 56 heads over 8, windows of 1,078 keys 76 us = 630 at 1,965 MHz,
// 93-95 right after work that had run into the power limit; a frame of
// 1,620 queries over 50,220 cached tokens 1.02-1.05 ms = 955-980; prompts and tokens of 9 sequences, windows of 2,048 and
// 64 sinks 127 us.  Per key tile of both row tiles, before the sums were folded (below): 3,230 cycles (16-bit), 3,780 (8-bit, where the widened tiles are
// written and the codes read beside the operands in shared memory), 2,048 of them products: the chain scores -> softmax ->
// P V -> next scores of a row tile bounds it, as in k_attn.
// Measured and rejected:
//   - warps of their own that divide and store finished rows: 16-bit the same within 1 %, 8-bit (the widening warps) 10 % slower;
//   - row tiles of the last, partly empty round as items of their own: 76.2 against 77.3 us (56 heads over 8), less than that case varies;
//   - a share of the exponentials on the FMA pipe (ex2_emu2): of eight, one 0.7 to 1.5 % slower, three 6 to 9, four 7 to 12;
//   - a widening loop unrolled over its four quarters: 2,115 against 1,713 us (a frame over 50,220 cached tokens; instruction cache);
//   - claiming the next item at the start of the current one: 175 against 133 us (ragged cache).
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
constexpr int FOLD = 256;                                 // key tiles that one accumulator takes
constexpr int PART_ROW = 132;                             // floats of a parked row: 16-byte lanes of 8 rows hit all banks
constexpr int CODES = 128 * 128;                          // E4M3 codes of a tile
// Q_A Q_B | K0 K1 | V0 V1 (at the end of a split: parked rows) | 8-bit: codes of a key and of a value tile | control
struct Control {
    uint64_t q_full, q_empty, q_raw, k_full[2], v_full[2], k_empty[2], v_empty[2], v_raw[2], s_full[2], p_full[4] /* [tile][half] */, o_done[2];
    uint64_t c_full[4], c_empty[4] /* codes of 64 keys: [keys | values][half] */, item_full[2], item_empty[2], clc_full;
    uint64_t rows_done[4];                                // softmax warps that are through with an item, by item modulo 4
    uint32_t tmem_base;
    int abort_word;
    int progress;                                         // tiles whose scores have been asked for
    int search;                                           // tiles gone through for values that are not finite
    int odd[4], cta_of[4];                                // by item modulo 4: it has rows that came out non-finite; CTA of the grid whose item it is
    alignas(16) uint32_t clc[4];
    alignas(16) int item[2][16];
    alignas(16) float4 scales[4];                         // of a tile: key scale of either half, log2 of the value scale of either half
    float2 inv_scales[4];                                 // 1 / value scale of either half
    int8_t q_shift[2][256];                               // 8-bit: rows of Q are here times 2^shift; by item
};
template <bool KV8> constexpr size_t smem_bytes() { return 1024 + 6 * (size_t)TILE + (KV8 ? 2 * CODES : 0) + sizeof(Control); }
static_assert(256 * PART_ROW * 4 + 2 * 256 * 4 <= 6 * TILE, "parked rows");
}  // namespace wtile

struct TileParams {
    WinArgs a;
    CUtensorMap map_q;                                    // {d, head, row}, box {64, group, queries of a tile}
    CUtensorMap map_k, map_v;                             // 16-bit: {d, head, row}, box {64, 1, 128}
    int split;                                            // CTAs of a cluster, each with a range of the key tiles
    int first, row_tiles;                                 // item of the grid's first CTA (cluster); row tiles of a sequence
    int heads_first;                                      // items run over the K/V heads first, then over the row tiles (else the other way round)
    int wide_stores;                                      // rows of the output are 32-byte aligned
    int bm;                                               // rows of a row tile: whole queries, at most 128
};

// largest of three, NaN if one is NaN
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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

// 32 bytes of one row
__device__ __forceinline__ void store32(void *dst, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// Cluster launch control: asks for a CTA of this grid that has not started; 16 bytes of answer land in shared memory.
__device__ __forceinline__ void clc_ask(uint32_t *answer, uint64_t *bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)),
                 "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool clc_answer(const uint32_t *answer, int &x) {
    uint32_t got, cx;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t.reg .b32 y, z;\n\tld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, _}, r;\n\t}"
        : "=&r"(got), "=&r"(cx) : "r"(smem_u32(answer)) : "memory");
    x = (int)cx;
    return got != 0;
}

template <bool KV8> struct TileCfg {
    static constexpr int THREADS = KV8 ? 512 : 384;
    // 8-bit: 512 threads start with 128 registers each, 48 + 2 * 200 + 64 = 4 * 128; 16-bit: 384 with 168, 88 + 2 * 208 = 3 * 168
    static constexpr int REG_ISSUE = KV8 ? 48 : 88, REG_SOFTMAX = KV8 ? 200 : 208, REG_WIDEN = 64;
    static constexpr int ITEM_READERS = KV8 ? 15 : 11;   // warps 0 to 2, softmax, widening
};

struct TileItem {
    int kvh, s, r0, r_end, row0, n, pos0, sink, from, n_kv, t_first;       // s: 8-bit: the sequence; 16-bit: 1 if done a second time
    int hi, lo, sn;                                       // some row sees key j: j <= hi and (j >= lo or j < sn)
    __device__ __forceinline__ int key(int j) const {                    // first key of the j-th tile
        const int i = t_first + j;
        return (i < sink ? i : from + i - sink) * wtile::BN;
    }
    __device__ __forceinline__ int row_tiles(int bm) const { return r_end - r0 > bm ? 2 : 1; }
};

// LONG: an item may have more than FOLD key tiles
template <typename T, bool KV8, bool LONG>
__global__ void __launch_bounds__(TileCfg<KV8>::THREADS, 1) k_attn_tile(const __grid_constant__ TileParams p) {
    using namespace wtile;
    using C = TileCfg<KV8>;
    using E = typename std::conditional<KV8, __half, T>::type;          // operand type
    constexpr bool CONVERT = KV8 && !std::is_same<T, __half>::value;    // Q has to become f16
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = smem, *sK = smem + 2 * TILE, *sV = smem + 4 * TILE, *sC = smem + 6 * TILE;
    Control &ctl = *reinterpret_cast<Control *>(sC + (KV8 ? 2 * CODES : 0));
    volatile int *abort_word = &ctl.abort_word;

    const WinArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % p.split;

    if (threadIdx.x == 0) {
        mbar_init(&ctl.q_full, CONVERT ? 2 : 1);
        mbar_init(&ctl.q_raw, 1);
        mbar_init(&ctl.q_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl.k_full[i], KV8 ? 4 : 1);
            mbar_init(&ctl.v_full[i], KV8 ? 4 : 1);
            mbar_init(&ctl.k_empty[i], 1);
            mbar_init(&ctl.v_empty[i], 1);
            mbar_init(&ctl.v_raw[i], 1);
            mbar_init(&ctl.s_full[i], 1);
            mbar_init(&ctl.o_done[i], 1);
            mbar_init(&ctl.p_full[2 * i], 4);
            mbar_init(&ctl.p_full[2 * i + 1], 4);
            for (int h = 0; h < 4; h += 2) {
                mbar_init(&ctl.c_full[h + i], 1);
                mbar_init(&ctl.c_empty[h + i], 4);
            }
            mbar_init(&ctl.item_full[i], 1);
            mbar_init(&ctl.item_empty[i], C::ITEM_READERS);
        }
        mbar_init(&ctl.clc_full, 1);
        for (int i = 0; i < 4; i++) {
            mbar_init(&ctl.rows_done[i], 8);
            ctl.odd[i] = 0;
        }
        ctl.abort_word = 0;
        ctl.progress = 0;
        ctl.search = 0;
        ctl.item[1][2] = -1;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(&ctl.tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    // rows behind the whole queries of a tile stay zero
    for (int i = threadIdx.x; i < 2 * (BM - p.bm) * 16; i += C::THREADS) {
        const int r = p.bm + (i >> 5), t = i >> 4 & 1, h = i & 15;
        *reinterpret_cast<uint4 *>(sQ + t * TILE + (h >> 3) * SLAB + r * 128 + (h & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = ctl.tmem_base;

    if (threadIdx.x == 32) tma_prefetch_desc(&p.map_q);
    if (!KV8 && threadIdx.x == 0 && a.lk) {                              // (without keys there are no maps)
        tma_prefetch_desc(&p.map_k);
        tma_prefetch_desc(&p.map_v);
    }
    // A bounded wait of one thread.  16-bit, long items: what its limit does not cover is a softmax warp that goes through the
    // tiles of an item's edges for values that are not finite (tens of millions of keys of one block, say).
    auto poll = [&](uint64_t *b, uint32_t parity, int code) -> bool {
        if (KV8 || !LONG) return mbar_wait(b, parity, abort_word, a.status, code);
        if (mbar_try_wait(b, parity)) return true;
        volatile int *search = &ctl.search;
        long long since = clock64();
        int seen = *search;
        for (uint32_t spins = 1;; spins++) {
            if (mbar_try_wait(b, parity)) return true;
            if (*abort_word) return false;
            if ((spins & 0x3ff) == 0 && clock64() - since > H3B_WAIT_CYCLES) {
                if (*search == seen) {
                    *abort_word = code;
                    if (a.status) atomicCAS(a.status, 0, code);
                    return false;
                }
                seen = *search;
                since = clock64();
            }
        }
    };
    // every wait: the whole warp together, bounded
    auto wait = [&](uint64_t *b, uint32_t parity, int code) -> bool { return __all_sync(0xffffffffu, poll(b, parity, code)) != 0; };
    // A wait that may last as long as an item, which has no bound of its own (one of 2^29 keys takes 8 s): its limit runs
    // from the last tile whose scores were asked for, so that it bounds a tile and not the item.  Only where that can be:
    // in every role it cost the 8-bit kernel 1,063 against 1,034 us (a frame over 50,220 cached tokens).
    auto wait_item = [&](auto done, int code) -> bool {
        volatile int *progress = &ctl.progress, *search = &ctl.search;
        long long since = clock64();
        int seen = *progress + (KV8 ? 0 : *search);
        bool fine = true;
        for (uint32_t spins = 1; fine && !done(); spins++) {
            if (*abort_word) fine = false;
            else if ((spins & 0xff) == 0) {
                const int now = *progress + (KV8 ? 0 : *search);
                if (now != seen) {
                    seen = now;
                    since = clock64();
                } else if (clock64() - since > H3B_WAIT_CYCLES) {
                    *abort_word = code;
                    if (a.status) atomicCAS(a.status, 0, code);
                    fine = false;
                }
            }
        }
        return __all_sync(0xffffffffu, fine) != 0;
    };
    // the k-th item of this CTA; false: no more (or a wait gave up)
    auto take_item = [&](int k, TileItem &it) -> bool {
        const int4 *src = reinterpret_cast<const int4 *>(ctl.item[k & 1]);
        const int4 x = src[0], y = src[1], z = src[2], w = src[3];
        it.kvh = x.x; it.s = x.y; it.r0 = x.z; it.r_end = x.w;
        it.row0 = y.x; it.n = y.y; it.pos0 = y.z; it.sink = y.w;
        it.from = z.x; it.n_kv = z.y; it.t_first = z.z; it.hi = z.w;
        it.lo = w.x; it.sn = w.y;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.item_empty[k & 1]);
        return it.r0 >= 0;
    };
    auto next_item = [&](int k, TileItem &it) -> bool { return wait(&ctl.item_full[k & 1], (k >> 1) & 1, H3B_ST_TIMEOUT_OTHER) && take_item(k, it); };
    // for those that have nothing to do, or are through, long before the item ends
    auto next_item_early = [&](int k, TileItem &it) -> bool {
        if (!LONG) return next_item(k, it);
        return wait_item([&] { return mbar_try_wait(&ctl.item_full[k & 1], (k >> 1) & 1); }, H3B_ST_TIMEOUT_OTHER) && take_item(k, it);
    };
    // what the first and the last row of an item see
    auto rows_of = [&](const TileItem &it, h3b_win_row &ra, h3b_win_row &rz) {
        ra = h3b_win_of(a.win, it.pos0 + it.r0 / a.group, it.n);
        rz = h3b_win_of(a.win, it.pos0 + (it.r_end - 1) / a.group, it.n);
    };
    // a tile has keys before `end` that no row sees (16-bit: what lies behind the last key comes as zeros)
    auto edge = [&](const TileItem &it, int key, int end) { return min(key + BN, end) - 1 > it.hi || max(key, it.sn) < min(key + BN, it.lo); };
    // 16-bit: a tile whose values pass through warp 3
    auto by_hand = [&](const TileItem &it, int key) {
        if (edge(it, key, it.n)) return true;
        if (!it.s) return false;
        h3b_win_row ra, rz;
        rows_of(it, ra, rz);
        return !h3b_win_full(ra, rz, key, BN);
    };
    bool ok = true;

    if (warp < SOFTMAX_WARP) {
        regs_dec<C::REG_ISSUE>();
        TileItem it;
        if (warp == 0) {
            // ------------------------------------------------------------ K and V
            int c = 0;                                                   // tiles so far
            for (int k = 0; ok && next_item(k, it); k++) {
                if (!KV8) {
                    for (int j = 0; j < it.n_kv && ok; j++, c++) {
                        const int st = c & 1, key = it.key(j);
                        const uint32_t ph = ((c >> 1) & 1) ^ 1;
                        ok = wait(&ctl.k_empty[st], ph, H3B_ST_TIMEOUT_EMPTY);
                        if (!ok) break;
                        if (lane == 0) {
                            mbar_expect_tx(&ctl.k_full[st], TILE);
                            tma_load_3d(sK + st * TILE, &p.map_k, &ctl.k_full[st], 0, it.kvh, key);
                            tma_load_3d(sK + st * TILE + SLAB, &p.map_k, &ctl.k_full[st], 64, it.kvh, key);
                        }
                        ok = wait(&ctl.v_empty[st], ph, H3B_ST_TIMEOUT_EMPTY);
                        if (!ok) break;
                        if (lane == 0) {
                            uint64_t *b = by_hand(it, key) ? &ctl.v_raw[st] : &ctl.v_full[st];
                            mbar_expect_tx(b, TILE);
                            tma_load_3d(sV + st * TILE, &p.map_v, b, 0, it.kvh, key);
                            tma_load_3d(sV + st * TILE + SLAB, &p.map_v, b, 64, it.kvh, key);
                        }
                    }
                } else {
                    // 64 tokens of a head lie together (8 KiB) and are asked for as soon as the widening warps are through with
                    // the same quarter of the tile before.  Lanes look up the blocks of 16 tiles at a time.
                    int bi = -1;
                    float bks = 1.0f, blvs = 0.0f, bivs = 1.0f;
                    for (int j = 0; j < it.n_kv && ok; j++, c++) {
                        if (j % 16 == 0) {
                            bi = -1;
                            if (j + (lane >> 1) < it.n_kv) {
                                // half of a tile may lie outside every row's window (before it, or behind the sinks): the page of such a
                                // half may be anything and is not looked up; the widening warps zero its rows
                                const int blk = it.key(j + (lane >> 1)) / KV8_BLOCK + (lane & 1);
                                if (h3b_win_any(it.hi, it.lo, it.sn, blk * KV8_BLOCK, KV8_BLOCK)) bi = (int)kv8_block_index(a, it.s, blk, it.kvh);
                            }
                            bks = bi >= 0 ? kv8_read_scale(__ldg(a.ks + bi)) : 1.0f;
                            const float vs = bi >= 0 ? kv8_read_scale(__ldg(a.vs + bi)) : 1.0f;
                            blvs = log2f(vs);
                            bivs = 1.0f / vs;
                        }
                        const int src = 2 * (j % 16);
                        const int b[2] = {__shfl_sync(0xffffffffu, bi, src), __shfl_sync(0xffffffffu, bi, src + 1)};
                        const float4 sc = make_float4(__shfl_sync(0xffffffffu, bks, src), __shfl_sync(0xffffffffu, bks, src + 1),
                                                      __shfl_sync(0xffffffffu, blvs, src), __shfl_sync(0xffffffffu, blvs, src + 1));
                        const float2 isc = make_float2(__shfl_sync(0xffffffffu, bivs, src), __shfl_sync(0xffffffffu, bivs, src + 1));
#pragma unroll
                        for (int w = 0; w < 4 && ok; w++) {
                            ok = wait(&ctl.c_empty[w], (c & 1) ^ 1, H3B_ST_TIMEOUT_EMPTY);
                            if (ok && lane == 0) {
                                // the softmax warps read the scales of tile c behind s_full(c); the slot is that of tile c - 4,
                                // whose scores were done with before the codes of tile c - 1 could be widened
                                if (w == 0) {
                                    ctl.scales[c & 3] = sc;
                                    ctl.inv_scales[c & 3] = isc;
                                }
                                // a block outside the pool (reported) or one that no row sees is not read: its rows are invalid or hidden
                                if (b[w & 1] >= 0) {
                                    mbar_expect_tx(&ctl.c_full[w], CODES / 2);
                                    bulk_load(sC + w * (CODES / 2), (w >> 1 ? a.vc : a.kc) + (long long)b[w & 1] * (CODES / 2), CODES / 2, &ctl.c_full[w]);
                                } else {
                                    mbar_arrive(&ctl.c_full[w]);
                                }
                            }
                        }
                    }
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA issuer
            // The whole warp walks the loop, converged; one lane, elected once, issues every tcgen05 instruction.  The
            // stage barriers of the next iteration are polled behind an issued block, while the queue drains.
            // Its waits are not voted on: nothing within an item is collective, and a lane that gives up alone meets the others
            // at the end of the item (theirs end too, since a wait that cannot be met looks at abort_word).
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
                    const uint32_t x = (uint32_t)(k >> 2) * (SLAB >> 4) + (uint32_t)(k & 3) * 2;
                    if (lead) umma_f16_ss_lh(d_tmem, qa + x, kb + x, DESC_HI, idesc_s, (uint32_t)(k != 0));
                }
                if (lead) tc_commit(&ctl.s_full[t]);
            };
            auto issue_pv = [&](int t, int stage, int half, bool first) {
                const uint32_t vb = v_lo0 + (uint32_t)stage * (TILE >> 4);
#pragma unroll
                for (int k = half * (BN / 32); k < (half + 1) * (BN / 32); k++)
                    if (lead)
                        umma_f16_ts_lh(tmem_base + O_COL + 128u * t, tmem_base + S_COL + 128u * t + (uint32_t)k * 8,
                                       vb + (uint32_t)k * (2048 >> 4), DESC_HI, idesc_o, (uint32_t)(!first || k != 0));
            };
            int c = 0, q = 0, pc[2] = {0, 0};                            // tiles, items with keys, tiles of either row tile so far
            for (int k = 0; ok && next_item(k, it); k++) {
                const int n_kv = it.n_kv, n_tiles = it.row_tiles(p.bm);
                if (!n_kv) continue;
                ok = poll(&ctl.q_full, q & 1, H3B_ST_TIMEOUT_OTHER) && poll(&ctl.k_full[c & 1], (c >> 1) & 1, H3B_ST_TIMEOUT_FULL);
                tc_fence_after();
                for (int t = 0; t < n_tiles && ok; t++) issue_s(t, c & 1);
                if (ok && lead) {
                    tc_commit(&ctl.k_empty[c & 1]);
                    if (n_kv == 1) tc_commit(&ctl.q_empty);
                }
                ok = ok && poll(&ctl.v_full[c & 1], (c >> 1) & 1, H3B_ST_TIMEOUT_FULL) &&
                     (n_kv < 2 || poll(&ctl.k_full[(c + 1) & 1], ((c + 1) >> 1) & 1, H3B_ST_TIMEOUT_FULL));
                auto step = [&](int j, auto stage_c) {
                    constexpr int st = decltype(stage_c)::value, nx = st ^ 1;
                    const bool more = j + 1 < n_kv;
                    for (int t = 0; t < n_tiles && ok; t++) {
                        const uint32_t ph = (uint32_t)((t ? pc[1] : pc[0]) + j) & 1;
                        ok = poll(&ctl.p_full[2 * t], ph, H3B_ST_TIMEOUT_OTHER);
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(t, st, 0, j == 0);
                        ok = poll(&ctl.p_full[2 * t + 1], ph, H3B_ST_TIMEOUT_OTHER);
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(t, st, 1, false);
                        if (t == n_tiles - 1 && lead) tc_commit(&ctl.v_empty[st]);
                        if (more) {
                            issue_s(t, nx);
                            if (t == n_tiles - 1 && lead) {
                                *reinterpret_cast<volatile int *>(&ctl.progress) = c + j + 2;
                                tc_commit(&ctl.k_empty[nx]);
                                if (j + 2 == n_kv) tc_commit(&ctl.q_empty);   // the last scores of the item
                            }
                        }
                    }
                    if (ok && more) {
                        ok = poll(&ctl.v_full[nx], ((c + j + 1) >> 1) & 1, H3B_ST_TIMEOUT_FULL);
                        if (ok && j + 2 < n_kv) ok = poll(&ctl.k_full[st], ((c + j + 2) >> 1) & 1, H3B_ST_TIMEOUT_FULL);
                        tc_fence_after();
                    }
                };
                for (int j = 0; ok && j < n_kv; j++) {
                    if ((c + j) & 1) step(j, std::integral_constant<int, 1>{});
                    else step(j, std::integral_constant<int, 0>{});
                }
                for (int t = 0; t < n_tiles; t++)
                    if (lead) tc_commit(&ctl.o_done[t]);
                c += n_kv;
                q++;
                pc[0] += n_kv;
                if (n_tiles == 2) pc[1] += n_kv;
                ok = __all_sync(0xffffffffu, ok) != 0;                   // here the lanes meet again
            }
        } else {
            // ------------------------------------------------------------ Q, items, value rows that nobody sees
            // Q of the q-th item with keys (warp 2)
            auto load_q = [&](const TileItem &x, int q) -> bool {
                if (!wait(&ctl.q_empty, (q & 1) ^ 1, H3B_ST_TIMEOUT_EMPTY)) return false;
                if (lane == 0) {
                    uint64_t *b = CONVERT ? &ctl.q_raw : &ctl.q_full;
                    const int n = x.row_tiles(p.bm);
                    mbar_expect_tx(b, (uint32_t)(n * p.bm * 256));
                    for (int t = 0; t < n; t++) {
                        const int row = x.row0 + (x.r0 + t * p.bm) / a.group;
                        tma_load_3d(sQ + t * TILE, &p.map_q, b, 0, x.kvh * a.group, row);
                        tma_load_3d(sQ + t * TILE + SLAB, &p.map_q, b, 64, x.kvh * a.group, row);
                    }
                }
                __syncwarp();
                return true;
            };
            // bf16 rows to f16 under a power of two of their maximum, which the softmax undoes; sixteen lanes per row, every
            // other pair of rows is this warp's
            auto convert_q = [&](const TileItem &x, int q) -> bool {
                if (!wait(&ctl.q_raw, q & 1, H3B_ST_TIMEOUT_FULL)) return false;
                const int sub = lane >> 4, ch = lane & 15, tiles = x.row_tiles(p.bm);
                for (int t = 0; t < tiles; t++) {
                    uint8_t *base = sQ + t * TILE + (ch >> 3) * SLAB;
#pragma unroll 4
                    for (int r0 = 2 * (warp & 1); r0 < BM; r0 += 4) {
                        const int r = r0 + sub;
                        uint4 *at = reinterpret_cast<uint4 *>(base + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                        const uint4 w = *at;
                        uint32_t top = abs_max8(w);
#pragma unroll
                        for (int y = 1; y < 16; y <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, y));
                        const uint32_t bits = widen_abs<T>(top);
                        int sh = 14 - ((int)(bits >> 23) - 127);
                        sh = bits >= 0x7f800000u || bits == 0u ? 0 : max(min(sh, 120), -120);   // not finite: as it is
                        const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
                        uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            v[i] = Elem<__half>::pack(__uint_as_float(v[i] << 16) * up, __uint_as_float(v[i] & 0xffff0000u) * up);
                        *at = make_uint4(v[0], v[1], v[2], v[3]);
                        if (ch == 0) ctl.q_shift[q & 1][t * BM + r] = (int8_t)sh;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl.q_full);
                return true;
            };
            int q = 0;
            if (warp == 2) {
                for (int k = 0; ok && next_item_early(k, it); k++)
                    if (it.n_kv) {
                        ok = load_q(it, q) && (!CONVERT || convert_q(it, q));
                        q++;
                    }
            } else {
                // item k of the CTA
                auto slot_free = [&](int k) -> bool { return wait(&ctl.item_empty[k & 1], ((k >> 1) & 1) ^ 1, H3B_ST_TIMEOUT_EMPTY); };
                auto publish = [&](int k, const TileItem &x) {
                    if (lane == 0) {
                        int4 *dst = reinterpret_cast<int4 *>(ctl.item[k & 1]);
                        dst[0] = make_int4(x.kvh, x.s, x.r0, x.r_end);
                        dst[1] = make_int4(x.row0, x.n, x.pos0, x.sink);
                        dst[2] = make_int4(x.from, x.n_kv, x.t_first, x.hi);
                        dst[3] = make_int4(x.lo, x.sn, 0, 0);
                        mbar_arrive(&ctl.item_full[k & 1]);
                    }
                };
                // what CTA x of the grid has to do; false: nothing
                auto describe = [&](int x, TileItem &d) -> bool {
                    const int i = p.first + x / p.split;
                    const int in_seq = a.kv_heads * p.row_tiles, j = i % in_seq;
                    d.s = KV8 ? i / in_seq : 0;
                    d.kvh = p.heads_first ? j % a.kv_heads : j / p.row_tiles;
                    // late rows first: under a window that is open to the left they see the most
                    d.r0 = (p.row_tiles - 1 - (p.heads_first ? j / a.kv_heads : j % p.row_tiles)) * (2 * p.bm);
                    const SeqExt e = seq_ext<KV8>(a, d.s);               // (16-bit: there is one)
                    const long long rows = (long long)e.nq * a.group;
                    if (d.r0 >= rows) return false;
                    d.r_end = (int)(rows < d.r0 + 2 * p.bm ? rows : d.r0 + 2 * p.bm);
                    d.row0 = e.row0; d.n = e.n; d.pos0 = e.pos0;
                    h3b_win_row ra, rz;
                    rows_of(d, ra, rz);
                    const h3b_win_tiles w = h3b_win_tiles_rows(ra, rz, BN);
                    d.hi = rz.hi; d.lo = ra.lo; d.sn = rz.s;
                    const int share = (w.count + p.split - 1) / p.split;
                    d.sink = w.sink; d.from = w.from;
                    d.t_first = rank * share;
                    d.n_kv = max(min(d.t_first + share, w.count) - d.t_first, 0);
                    return true;
                };
                int x = blockIdx.x, asked = 0;
                bool more = p.split == 1;                                // there may be another
                // the next item with rows in `d`; r0 = -1: none
                auto find = [&](bool own, TileItem &d) -> bool {
                    d.r0 = -1;
                    if (own && describe(x, d)) return true;
                    d.r0 = -1;
                    while (more) {
                        if (lane == 0) {
                            mbar_expect_tx(&ctl.clc_full, 16);
                            clc_ask(ctl.clc, &ctl.clc_full);
                        }
                        if (!wait(&ctl.clc_full, asked & 1, H3B_ST_TIMEOUT_OTHER)) return false;
                        asked++;
                        more = clc_answer(ctl.clc, x);
                        fence_proxy_async_smem();                        // the next answer comes behind this reading
                        __syncwarp();
                        if (more && describe(x, d)) return true;
                        d.r0 = -1;
                    }
                    return true;
                };
                // 16-bit: item `done` (the first that has not been looked at) has to be done a second time, as d
                int done = 0;
                auto second_time = [&](TileItem &d) -> bool {
                    volatile int *odd = &ctl.odd[done & 3];
                    const bool hit = *odd != 0;
                    const int from = *reinterpret_cast<volatile int *>(&ctl.cta_of[done & 3]);
                    __syncwarp();
                    if (lane == 0) *odd = 0;
                    done++;
                    if (!hit || !describe(from, d)) return false;
                    h3b_win_row ra, rz;
                    rows_of(d, ra, rz);
                    d.s = 1;
                    return ra.hi != rz.hi || ra.lo != rz.lo || ra.s != rz.s;   // rows that see the same hold what they see
                };
                TileItem next;                                           // found and not yet handed out (r0 = -1: none)
                // item k: one for the second time, the next one, or none
                auto choose = [&](int k) -> bool {
                    if (KV8) return find(k == 0, it) && slot_free(k);
                    if (next.r0 < 0 && !find(k == 0, next)) return false;
                    if (!slot_free(k)) return false;
                    // every warp has taken item k - 2, so the softmax warps are through with item k - 3
                    while (done + 3 <= k)
                        if (second_time(it)) return true;
                    while (next.r0 < 0 && done < k) {
                        if (!wait(&ctl.rows_done[done & 3], (done >> 2) & 1, H3B_ST_TIMEOUT_OTHER)) return false;
                        if (second_time(it)) return true;
                    }
                    if (lane == 0) ctl.cta_of[k & 3] = x;
                    __syncwarp();
                    it = next;
                    next.r0 = -1;
                    return true;
                };
                int c = 0, raw[2] = {0, 0};
                next.r0 = -1;
                ok = choose(0);
                if (ok) publish(0, it);
                for (int k = 1; ok && it.r0 >= 0; k++) {
                    if (CONVERT) {
                        if (it.n_kv) ok = convert_q(it, q++);
                    } else if (!KV8) {
                        for (int j = 0; j < it.n_kv && ok; j++) {
                            const int st = (c + j) & 1, key = it.key(j);
                            if (!by_hand(it, key)) continue;
                            // tiles that need no cleaning lie in between
                            if (LONG) ok = wait_item([&] { return mbar_try_wait(&ctl.v_raw[st], (st ? raw[1] : raw[0]) & 1); }, H3B_ST_TIMEOUT_FULL);
                            else ok = wait(&ctl.v_raw[st], (st ? raw[1] : raw[0]) & 1, H3B_ST_TIMEOUT_FULL);
                            if (!ok) break;
                            if (st) raw[1]++;
                            else raw[0]++;
                            for (int i = lane; i < BN; i += 32) {
                                uint8_t *row = sV + st * TILE + i * 128;
                                if (key + i > it.hi || (key + i < it.lo && key + i >= it.sn)) {
#pragma unroll
                                    for (int h = 0; h < 16; h++)
                                        *reinterpret_cast<uint4 *>(row + (h >> 3) * SLAB + ((h & 7) ^ (i & 7)) * 16) = make_uint4(0u, 0u, 0u, 0u);
                                } else if (it.s) {
#pragma unroll 4
                                    for (int h = 0; h < 16; h++) {
                                        uint4 *at = reinterpret_cast<uint4 *>(row + (h >> 3) * SLAB + ((h & 7) ^ (i & 7)) * 16);
                                        const uint4 w = *at;
                                        *at = make_uint4(finite_or_zero<T>(w.x), finite_or_zero<T>(w.y), finite_or_zero<T>(w.z), finite_or_zero<T>(w.w));
                                    }
                                }
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&ctl.v_full[st]);
                        }
                    }
                    // The next item is asked for when the scores of the last tile but one have been, some 5 us before the end:
                    // early enough for its first tiles, late enough that a CTA with a long item does not hold one back from
                    // CTAs that are through (asking at the start left some SMs with four items and others with one: 175 us
                    // instead of 133 for the ragged cache).
                    if (it.n_kv > 2) {
                        const int until = c + it.n_kv - 1;
                        ok = ok && wait_item([&] {
                            if (*reinterpret_cast<volatile int *>(&ctl.progress) >= until) return true;
                            __nanosleep(100);
                            return false;
                        }, H3B_ST_TIMEOUT_OTHER);
                    }
                    c += it.n_kv;
                    ok = ok && choose(k);
                    if (ok) publish(k, it);
                }
            }
        }
        __syncwarp();
    } else if (warp < WIDEN_WARP) {
        // ---------------------------------------------------------------- softmax
        regs_inc<C::REG_SOFTMAX>();
        const int t = (warp - SOFTMAX_WARP) >> 2, quarter = warp & 3;    // row tile, TMEM lane quarter
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + S_COL + 128u * t, o_addr = tmem_base + lane_base + O_COL + 128u * t;
        TileItem it;
        int c = 0, mine = 0, q = 0, mine_q = 0;                          // tiles and items with keys so far, and those of this row tile
        for (int k = 0; ok && next_item_early(k, it); k++) {
            const int n_kv = it.n_kv;
            // this warp's rows of the item are through (and, 16-bit, `odd`: one came out non-finite with a finite sum of probabilities)
            auto rows_done = [&](bool odd) {
                if (KV8) return;
                odd = __any_sync(0xffffffffu, odd);
                __syncwarp();                                            // what every lane has parked comes before the arrival
                if (lane == 0) {
                    if (odd && !it.s) *reinterpret_cast<volatile int *>(&ctl.odd[k & 3]) = 1;
                    mbar_arrive(&ctl.rows_done[k & 3]);
                }
            };
            if (t >= it.row_tiles(p.bm)) {
                c += n_kv;
                q += n_kv > 0;
                rows_done(false);
                continue;
            }
            const int slot = t * BM + quarter * 32 + lane;                      // place of this thread's row in the row tiles
            const int my = it.r0 + t * p.bm + quarter * 32 + lane;              // and the row
            const bool live = quarter * 32 + lane < p.bm && my < it.r_end;
            const int qi = (live ? my : it.r_end - 1) / a.group, hd = (live ? my : it.r_end - 1) - qi * a.group;
            const h3b_win_row wr = h3b_win_of(a.win, it.pos0 + qi, it.n);
            const h3b_win_row wa = h3b_win_of(a.win, it.pos0 + (it.r0 + t * p.bm) / a.group, it.n);
            const h3b_win_row wz = h3b_win_of(a.win, it.pos0 + (min(it.r0 + (t + 1) * p.bm, it.r_end) - 1) / a.group, it.n);
            float m_run = -INFINITY, l_run = 0.0f, row_scale = a.scale_log2;
            // The tensor core cuts each product to the accumulator's exponent (and two bits or so) before it adds it: a sum of
            // many keys comes out low, by 6e-9 of itself per key where nothing cancels (measured: 3.4e-4 at 65,536 keys, 6.5e-3
            // at a million; at 2^26 equal keys it stands still).  So it starts anew every FOLD tiles, and what it was is added
            // up here, in local memory: 128 KiB a CTA every 0.5 ms.  The bias stays at 1.5e-4 then (4 million keys of one CTA), for
            // code that costs a frame over 50,220 cached tokens 2 to 3 % (a loop of its own beside the rescaling 4).
            float far[HD], far_scale = 1.0f;                             // far_scale: what the maximum's growth makes of far
            for (int j = 0; j < n_kv; j++) {
                const int key = it.key(j);
                const bool whole = h3b_win_full(wa, wz, key, BN);        // no mask; decided before the scores are waited for
                ok = wait(&ctl.s_full[t], (mine + j) & 1, H3B_ST_TIMEOUT_TMEM_FULL);
                if (!ok) break;
                float4 scl;
                float2 inv;
                if (KV8) {
                    scl = ctl.scales[(c + j) & 3];
                    inv = ctl.inv_scales[(c + j) & 3];
                }
                if (CONVERT && j == 0) row_scale *= __uint_as_float((uint32_t)(127 - ctl.q_shift[q & 1][slot]) << 23);
                tc_fence_after();
                uint32_t sv[BN];
#pragma unroll
                for (int ch = 0; ch < BN / 32; ch++) tmem_ld_32x32b_x32(s_addr + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[ch * 32]));
                tmem_ld_wait();
                if (!whole) {
#pragma unroll
                    for (int ch = 0; ch < BN / 32; ch++) {
                        // bits of the 32 keys that the row sees
                        const int b = wr.hi - key - ch * 32, lo = wr.lo - key - ch * 32, sn = wr.s - key - ch * 32;
                        const uint32_t upto = b >= 31 ? 0xffffffffu : b < 0 ? 0u : (2u << b) - 1u;
                        const uint32_t from = lo <= 0 ? 0xffffffffu : lo > 31 ? 0u : 0xffffffffu << lo;
                        const uint32_t sink = sn <= 0 ? 0u : sn > 31 ? 0xffffffffu : (1u << sn) - 1u;
                        const uint32_t see = upto & (from | sink);
                        if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;
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
                        for (int x = 0; x < 4; x++)
                            mxc[x] = max3_nan(mxc[x], __uint_as_float(sv[h * 64 + i + 2 * x]), __uint_as_float(sv[h * 64 + i + 2 * x + 1]));
                    mxh[h] = max3_nan(max3_nan(mxc[0], mxc[1], mxc[2]), mxc[3], mxc[3]);
                }
                float f[2] = {row_scale, row_scale}, off[2] = {0.0f, 0.0f}, inv_vs[2] = {1.0f, 1.0f};
                float mx;
                if (KV8) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        f[h] = row_scale * (h ? scl.y : scl.x);
                        off[h] = h ? scl.w : scl.z;
                        inv_vs[h] = h ? inv.y : inv.x;
                        // nothing of the 64 seen: its scales (of tokens that others see, perhaps NaN) have no part
                        if (mxh[h] == -INFINITY) f[h] = 1.0f, off[h] = 0.0f, inv_vs[h] = 1.0f;
                        mxh[h] = fmaf(mxh[h], f[h], off[h]);
                    }
                    mx = max3_nan(mxh[0], mxh[1], mxh[1]);
                } else {
                    mx = max3_nan(mxh[0], mxh[1], mxh[1]) * row_scale;
                }
                if (mx != mx) l_run = mx;                                // undefined, and so is the row from here on
                const float m_new = fmaxf(m_run, mx);
                const bool grow = m_new > m_run + ProbRange<E>::LAG;     // also at the first visible key: m_run = -inf
                const bool fold = LONG && j && j % FOLD == 0;
                if (__any_sync(0xffffffffu, grow) || fold) {
                    float alpha = 1.0f;
                    if (grow) {
                        alpha = ex2_approx(m_run - m_new);
                        m_run = m_new;
                        l_run *= alpha;
                        if (LONG) far_scale *= alpha;
                    }
                    __syncwarp();
                    // s_full of tile j came behind the P V product of tile j - 1: the accumulator is at rest
                    if (j > 0) {
#pragma unroll 1
                        for (int ch = 0; ch < HD / 16; ch++) {
                            uint32_t o[16];
                            tmem_ld_32x32b_x16(o_addr + ch * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            if (fold) {
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    const float x = __uint_as_float(o[i]);
                                    far[ch * 16 + i] = j == FOLD ? x : fmaf(far[ch * 16 + i], far_scale, x);
                                    o[i] = 0u;
                                }
                            }
                            tmem_st_32x32b_x16(o_addr + ch * 16, o);
                        }
                    }
                    if (fold) far_scale = 1.0f;
                }
                const float m_use = m_run == -INFINITY ? 0.0f : m_run - ProbRange<E>::UP;
                float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
                auto chunk = [&](int ch, uint32_t (&packed)[16]) {
                    const float fh = f[ch >> 1], cc = KV8 ? off[ch >> 1] - m_use : -m_use;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float x0, x1, x2, x3;
                        fma2(x0, x1, __uint_as_float(sv[ch * 32 + i]), __uint_as_float(sv[ch * 32 + i + 1]), fh, cc);
                        fma2(x2, x3, __uint_as_float(sv[ch * 32 + i + 2]), __uint_as_float(sv[ch * 32 + i + 3]), fh, cc);
                        float p0, p1, p2, p3;
                        p0 = ex2_approx(x0); p1 = ex2_approx(x1); p2 = ex2_approx(x2); p3 = ex2_approx(x3);
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
                    if (lane == 0) mbar_arrive(&ctl.p_full[2 * t + half]);
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
            if (ok && n_kv) ok = wait(&ctl.o_done[t], mine_q & 1, H3B_ST_TIMEOUT_OTHER);
            if (!ok) break;
            c += n_kv;
            mine += n_kv;
            q += n_kv > 0;
            mine_q += n_kv > 0;
            tc_fence_after();
            const bool seen = live && h3b_win_count(wr) > 0;
            // done a second time: `add(x, r)` for every row r of the warp that sees values which were taken out
            auto give_back = [&](auto add) {
                h3b_win_row ra, rz;
                rows_of(it, ra, rz);
                OddValues x;
                x.clear();
                for (int j = 0; j < n_kv; j++) {
                    const int key = it.key(j);
                    if (h3b_win_full(ra, rz, key, BN)) continue;
                    x.template collect<T>(a, it.kvh, key, BN, wr, live, lane);
                    if (lane == 0) atomicAdd(&ctl.search, 1);
                }
                __syncwarp();                                            // the rows written above come first
                for (int r = 0; r < 32; r++)
                    if (x.any(r)) add(x, r);
            };
            if (LONG && n_kv > FOLD) {
#pragma unroll 1
                for (int ch = 0; ch < HD / 16; ch++) {
                    uint32_t o[16];
                    tmem_ld_32x32b_x16(o_addr + ch * 16, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = __float_as_uint(fmaf(far[ch * 16 + i], far_scale, __uint_as_float(o[i])));
                    tmem_st_32x32b_x16(o_addr + ch * 16, o);
                }
                tmem_st_wait();
            }
            if (p.split > 1) {
                // this CTA's share of the row: sums as they are, with their maximum and denominator
                float *part = reinterpret_cast<float *>(smem) + slot * PART_ROW;
                bool odd = false;
#pragma unroll 1
                for (int ch = 0; ch < HD / 32; ch++) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + ch * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4 *>(part + ch * 32 + i) =
                            n_kv ? make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]) : make_uint4(0u, 0u, 0u, 0u);
                    if (!KV8)
#pragma unroll
                        for (int i = 0; i < 32; i++) odd |= !(fabsf(__uint_as_float(o[i])) < INFINITY);
                }
                float *ml = reinterpret_cast<float *>(smem) + 2 * BM * PART_ROW;
                ml[slot] = m_run;
                ml[2 * BM + slot] = l_run;
                if (!KV8) {
                    if (it.s) give_back([&](const OddValues &x, int r) {
                        float4 *at = reinterpret_cast<float4 *>(reinterpret_cast<float *>(smem) + (t * BM + quarter * 32 + r) * PART_ROW + lane * 4);
                        const float4 y = *at;
                        *at = make_float4(y.x + x.of(r, 0), y.y + x.of(r, 1), y.z + x.of(r, 2), y.w + x.of(r, 3));
                    });
                    fence_proxy_async_smem();                            // done a second time, copies come where the rows are parked
                    rows_done(seen && n_kv && odd && ordinary(l_run));
                }
            } else {
                const float inv_l = 1.0f / l_run;
                T *dst = reinterpret_cast<T *>(a.out) + (long long)(it.row0 + qi) * a.o_rs + (long long)(it.kvh * a.group + hd) * a.o_hs;
                bool odd = false;
#pragma unroll 1
                for (int ch = 0; ch < HD / 32; ch++) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + ch * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 16) {
                        uint32_t h[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            const float x = __uint_as_float(o[i + 2 * u]) * inv_l, y = __uint_as_float(o[i + 2 * u + 1]) * inv_l;
                            if (!KV8) odd |= !(fabsf(x) <= largest<T>()) || !(fabsf(y) <= largest<T>());
                            h[u] = seen ? Elem<T>::pack(x, y) : 0u;
                        }
                        if (live) {
                            if (p.wide_stores) {
                                store32(dst + ch * 32 + i, h);
                            } else {
                                *reinterpret_cast<uint4 *>(dst + ch * 32 + i) = make_uint4(h[0], h[1], h[2], h[3]);
                                *reinterpret_cast<uint4 *>(dst + ch * 32 + i + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                            }
                        }
                    }
                }
                if (!KV8 && Elem<T>::FMT == 0 && __any_sync(0xffffffffu, odd)) {
                    // some row lies outside f16: what is finite goes back into it (in the loop above that cost 3 %)
                    odd = false;
#pragma unroll 1
                    for (int ch = 0; ch < HD / 16; ch++) {
                        uint32_t o[16], h[8];
                        tmem_ld_32x32b_x16(o_addr + ch * 16, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            const float x = __uint_as_float(o[2 * u]) * inv_l, y = __uint_as_float(o[2 * u + 1]) * inv_l;
                            odd |= !(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY);
                            h[u] = seen ? Elem<T>::pack(within_type<T, KV8>(x), within_type<T, KV8>(y)) : 0u;
                        }
                        if (live) {
                            *reinterpret_cast<uint4 *>(dst + ch * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                            *reinterpret_cast<uint4 *>(dst + ch * 16 + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                        }
                    }
                }
                if (!KV8) {
                    if (it.s) give_back([&](const OddValues &x, int r) {
                        const int row = __shfl_sync(0xffffffffu, qi, r), head = it.kvh * a.group + __shfl_sync(0xffffffffu, hd, r);
                        uint2 *at = reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + (long long)(it.row0 + row) * a.o_rs + (long long)head * a.o_hs + lane * 4);
                        const float4 y = load4(reinterpret_cast<const T *>(at));
                        *at = make_uint2(Elem<T>::pack(y.x + x.of(r, 0), y.y + x.of(r, 1)), Elem<T>::pack(y.z + x.of(r, 2), y.w + x.of(r, 3)));
                    });
                    rows_done(seen && odd && ordinary(l_run));
                }
            }
        }
    } else if (KV8) {
        // ---------------------------------------------------------------- widen the codes of a tile
        regs_dec<C::REG_WIDEN>();
        // Sixteen lanes per row: 8 codes in, one 16-byte piece of the f16 row out; the rows of a lane are 8 apart, so that its
        // place under the swizzle is the same in all of them.
        const int row0 = (warp - WIDEN_WARP) * 2 + (lane >> 4), ch = lane & 15;
        const uint32_t from = (uint32_t)(row0 * 128 + ch * 8), to = (uint32_t)((ch >> 3) * SLAB + row0 * 128 + (((ch & 7) ^ row0) << 4));
        TileItem it;
        int c = 0;
        for (int k = 0; ok && next_item(k, it); k++) {
            for (int j = 0; j < it.n_kv && ok; j++, c++) {
                const int st = c & 1, key = it.key(j);
                const uint32_t ph = ((c >> 1) & 1) ^ 1;
                const bool at_edge = edge(it, key, key + BN);    // stale bytes behind the last token among them
#pragma unroll 1                                                         // its code has to stay in the instruction caches beside the others'
                for (int w = 0; w < 4 && ok; w++) {                      // keys 0-63, 64-127, values 0-63, 64-127
                    ok = wait(&ctl.c_full[w], c & 1, H3B_ST_TIMEOUT_FULL) &&
                         (w & 1 || wait(w ? &ctl.v_empty[st] : &ctl.k_empty[st], ph, H3B_ST_TIMEOUT_EMPTY));
                    if (!ok) break;
                    const uint8_t *codes = sC + w * (CODES / 2) + from;
                    uint8_t *tile = (w >> 1 ? sV : sK) + st * TILE + (w & 1) * (64 * 128) + to;
                    uint2 raw[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) raw[i] = *reinterpret_cast<const uint2 *>(codes + i * (8 * 128));
                    if (at_edge)
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int x = key + (w & 1) * 64 + i * 8 + row0;
                            if (x > it.hi || (x < it.lo && x >= it.sn)) raw[i] = make_uint2(0u, 0u);
                        }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl.c_empty[w]);         // the codes are in registers
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        uint4 h;
                        widen4_e4m3(raw[i].x, h.x, h.y);
                        widen4_e4m3(raw[i].y, h.z, h.w);
                        *reinterpret_cast<uint4 *>(tile + i * (8 * 128)) = h;
                    }
                    if (w & 1) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(w >> 1 ? &ctl.v_full[st] : &ctl.k_full[st]);
                    }
                }
            }
        }
    }

    // A wait gave up: copies and products that are under way (microseconds) still write to this CTA's memory.  Whoever saw it
    // waits 1 ms before the others are let out.
    if (*abort_word)
        for (const long long since = clock64(); clock64() - since < 2000000;) __nanosleep(1000);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
    if (p.split > 1) {
        // ---- the shares meet: a warp finishes a row, a lane four of its dimensions
        const int *slot0 = ctl.item[ctl.item[0][2] < 0];                 // the one item (the first slot has the end if it was done twice)
        const int kvh = slot0[0], r0 = slot0[2], rows = *abort_word ? 0 : slot0[3] - slot0[2];
        SeqExt e;
        e.row0 = slot0[4]; e.n = slot0[5]; e.pos0 = slot0[6];
        cluster_sync_all();
        const uint32_t base = smem_u32(smem);
        for (int r = rank * (C::THREADS / 32) + warp; r0 >= 0 && r < rows; r += p.split * (C::THREADS / 32)) {
            const int slot = r < p.bm ? r : BM + r - p.bm;
            float m = -INFINITY, l = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < p.split; i++) m = fmaxf(m, ld_cluster_f(mapa_shared(base, i) + (2 * BM * PART_ROW + slot) * 4));
            for (int i = 0; i < p.split; i++) {
                const uint32_t peer = mapa_shared(base, i);
                const float mc = ld_cluster_f(peer + (2 * BM * PART_ROW + slot) * 4), lc = ld_cluster_f(peer + (2 * BM * PART_ROW + 2 * BM + slot) * 4);
                const float w = mc == -INFINITY ? 0.0f : ex2_approx(mc - m);
                const float4 x = ld_cluster_f32x4(peer + (slot * PART_ROW + lane * 4) * 4);
                l += lc != lc ? lc : w * lc;
                v.x += w * x.x; v.y += w * x.y; v.z += w * x.z; v.w += w * x.w;
            }
            const int qi = (r0 + r) / a.group, hd = (r0 + r) - qi * a.group;
            const bool seen = h3b_win_count(h3b_win_of(a.win, e.pos0 + qi, e.n)) > 0;
            const float inv = 1.0f / l;
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            T *dst = reinterpret_cast<T *>(a.out) + (long long)(e.row0 + qi) * a.o_rs + (long long)(kvh * a.group + hd) * a.o_hs;
            uint2 w = make_uint2(0u, 0u);
            if (seen) w = make_uint2(Elem<T>::pack(within_type<T, KV8>(v.x), within_type<T, KV8>(v.y)), Elem<T>::pack(within_type<T, KV8>(v.z), within_type<T, KV8>(v.w)));
            *reinterpret_cast<uint2 *>(dst + lane * 4) = w;
        }
        cluster_sync_all();                                              // nobody leaves while its memory is read
    }
}

template <typename T, bool KV8, bool LONG> static int launch_tile_t(h3_cuda *cuda, const TileParams &p, size_t items, char *error, size_t error_size) {
    void (*kernel)(const TileParams) = k_attn_tile<T, KV8, LONG>;
    static std::atomic<uint64_t> done;
    if (!smem_once(cuda, done, (const void *)kernel, wtile::smem_bytes<KV8>(), "attention smem attribute", error, error_size)) return 0;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(items * p.split));
    cfg.blockDim = dim3(TileCfg<KV8>::THREADS);
    cfg.dynamicSmemBytes = wtile::smem_bytes<KV8>();
    cfg.stream = cuda->op_stream;
    cfg.attrs = &attr;
    cfg.numAttrs = p.split > 1 ? 1 : 0;
    H3B_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p), "k_attn_tile launch");
    cuda->launches++;
    return 1;
}

// CTAs for each of `items` items that all run at once, at least two key tiles each
static int split_of(const h3_cuda *cuda, size_t items, size_t tiles) {
    static AttnClusters clusters;              // one CTA to an SM, in this variant as in the others
    size_t n = std::min<size_t>(std::max<size_t>(tiles / 2, 1), 8);
    while (n > 1 && attn_clusters_of(cuda, clusters, (const void *)k_attn_tile<__half, true, false>, TileCfg<true>::THREADS, wtile::smem_bytes<true>(), n) < items) n--;
    return (int)n;
}

int launch_attn_tile(h3_cuda *cuda, const WinArgs &a, int f16, bool kv8, size_t len, char *error, size_t error_size) {
    TileParams p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int queries = wtile::BM / a.group;
    p.bm = queries * a.group;
    if (h3b_encode_tmap_3d(&p.map_q, dt, 2, a.q, 128, a.heads, a.rows, a.q_hs * 2, a.q_rs * 2, 64, a.group, queries, CU_TENSOR_MAP_SWIZZLE_128B))
        return fail(error, error_size, "windowed attention: cuTensorMapEncodeTiled(Q) failed");
    if (!kv8 && a.lk) {
        if (h3b_encode_tmap_3d(&p.map_k, dt, 2, a.k, 128, a.kv_heads, a.lk, a.k_hs * 2, a.k_rs * 2, 64, 1, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
            h3b_encode_tmap_3d(&p.map_v, dt, 2, a.v, 128, a.kv_heads, a.lk, a.v_hs * 2, a.v_rs * 2, 64, 1, 128, CU_TENSOR_MAP_SWIZZLE_128B))
            return fail(error, error_size, "sdpa_window: cuTensorMapEncodeTiled failed");
    }
    const size_t sms = (size_t)cuda->sm_count, row_tiles = ceil_div((size_t)a.max_rows, 2 * (size_t)queries);
    const size_t items = row_tiles * a.kv_heads * a.n_seq;
    // (so many that passing over those without rows stays within the limit of a wait)
    if (items > (1u << 26)) return fail(error, error_size, "windowed attention: shape too large");
    const size_t tiles = std::max<size_t>(ceil_div(attn_window_keys(a.win, len, std::min<size_t>(a.max_rows, 2 * (size_t)queries)), wtile::BN), 1);
    p.row_tiles = (int)row_tiles;
    p.wide_stores = ((uintptr_t)a.out % 32 == 0) && (a.o_rs | a.o_hs) % 16 == 0;
    // Heads first puts the long items of all heads in front, which evens out the end; row tiles first lets neighbours share
    // keys in L2, which matters once all keys together do not fit it.  Measured (us, heads first | row tiles first): frames of
    // the 6,144-token step 198 | 210, ragged cache 126 | 131, 56 heads over 8 with 1,078-key windows 75.3 | 76.5; the other
    // way a frame over 50,220 cached tokens 1,006-1,016 | 985-1,001 and the 50,220-token video 8,525 | 7,650.
    p.heads_first = len * a.n_seq * a.kv_heads * (kv8 ? 256 : 512) <= (128u << 20);
    int (*launch)(h3_cuda *, const TileParams &, size_t, char *, size_t);
    // The most key tiles that an item can have, whatever the lengths on the device are: its rows' windows (their blocks may
    // begin a block apart) and the sinks, each rounded up to tiles, or all keys that there can be.  Up to FOLD of them need
    // neither folded sums nor waits of their own.  Measured (us, without | with them): ragged cache 127 | 131, 56 heads over 8
    // 75.7 | 76.6, frames of the 6,144-token step 195.8 | 196.9, 50,220-token video 7,630 | 7,685.
    const size_t capacity = kv8 ? (size_t)a.table_stride * a.page_blocks * KV8_BLOCK : (size_t)a.lk;
    const size_t reach = attn_window_keys(a.win, capacity, std::min<size_t>(a.max_rows, 2 * (size_t)queries) + (size_t)a.win.block);
    const bool is_long = reach / wtile::BN + 4 > (size_t)wtile::FOLD;
    if (kv8) launch = f16 ? (is_long ? launch_tile_t<__half, true, true> : launch_tile_t<__half, true, false>)
                          : (is_long ? launch_tile_t<__nv_bfloat16, true, true> : launch_tile_t<__nv_bfloat16, true, false>);
    else launch = f16 ? (is_long ? launch_tile_t<__half, false, true> : launch_tile_t<__half, false, false>)
                      : (is_long ? launch_tile_t<__nv_bfloat16, false, true> : launch_tile_t<__nv_bfloat16, false, false>);
    // Whole rounds of one item per SM run unsplit; what is left over, if it is less than half a round of one sequence's
    // long items, has its keys split so that it fills the chip too (a frame of 1,620 queries over 50,220 cached tokens,
    // 168 items: 1593 us unsplit, 1121 to 1249 split by 3 to 6 as a whole).
    const size_t rest = items % sms, whole = items - rest;
    const int n = rest ? split_of(cuda, rest, tiles) : 1;
    if (whole && (n < 2 || whole > 4 * sms || a.n_seq > 1 || tiles < 32)) {
        p.split = 1;
        return launch(cuda, p, items, error, error_size);
    }
    if (whole) {
        p.split = 1;
        if (!launch(cuda, p, whole, error, error_size)) return 0;
    }
    p.first = (int)whole;
    p.split = n;
    return !rest || launch(cuda, p, rest, error, error_size);
}

}  // namespace h3b
