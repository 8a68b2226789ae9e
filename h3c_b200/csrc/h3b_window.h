/* Which keys a query sees under a sliding window with sinks, and which key tiles a group of queries has to visit.
 * Plain C shared by the kernels (device), their host launchers and h3b_window_tiles (the host entry point that the
 * CPU tests walk).
 *
 * A query at position p belongs to the block that starts at b = p - p % block.  Key j of n is visible when
 *     j <= b + block - 1 + right   and   (j >= b - left or j < sinks).
 * lo and hi never decrease with p, which is what makes the union over a group of queries one range plus the sinks.
 *
 * All four numbers are clipped to H3B_WIN_MAX = 2^29 on the host (a side without a bound is clipped to it too), and
 * positions and key counts are below 2^29, so that every sum fits 31 bits. */
#ifndef H3B_WINDOW_H
#define H3B_WINDOW_H

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define H3B_HD __host__ __device__ __forceinline__
#else
#define H3B_HD inline
#endif

#define H3B_WIN_MAX (1 << 29)

typedef struct {
    int left, right, sinks, block;
} h3b_win;

typedef struct {
    int lo, hi, s; /* visible: j <= hi with j >= lo or j < s; hi = -1: nothing */
} h3b_win_row;

static H3B_HD h3b_win_row h3b_win_of(h3b_win w, int p, int n) {
    h3b_win_row r;
    const int b = p - p % w.block;
    const int hi = b + (w.block - 1) + w.right, lo = b - w.left;
    r.hi = p < 0 ? -1 : (hi < n - 1 ? hi : n - 1);
    r.lo = lo > 0 ? lo : 0;
    r.s = w.sinks < r.hi + 1 ? w.sinks : r.hi + 1;
    return r;
}

static H3B_HD int h3b_win_sees(h3b_win_row r, int j) { return j <= r.hi && (j >= r.lo || j < r.s); }

/* keys that the row sees */
static H3B_HD int h3b_win_count(h3b_win_row r) {
    const int from = r.lo > r.s ? r.lo : r.s, tail = r.hi + 1 - from;
    return (r.s > 0 ? r.s : 0) + (tail > 0 ? tail : 0);
}

/* Key tiles of `unit` keys that queries at positions p0..p1 (p0 <= p1) of a sequence of n keys have to visit: `sink`
 * tiles from 0 on, then tiles from `from` on; `count` in all. */
typedef struct {
    int sink, from, count;
} h3b_win_tiles;

/* a, z: rows of the first and the last query (of a query in front of token 0 only lo matters, which is that of token 0) */
static H3B_HD h3b_win_tiles h3b_win_tiles_rows(h3b_win_row a, h3b_win_row z, int unit) {
    h3b_win_tiles t;
    const int last = z.hi >= 0 ? z.hi / unit + 1 : 0, first = a.lo / unit;
    t.sink = z.s > 0 ? (z.s + unit - 1) / unit : 0;
    t.from = first > t.sink ? first : t.sink;
    t.count = t.sink + (last > t.from ? last - t.from : 0);
    return t;
}

static H3B_HD h3b_win_tiles h3b_win_tiles_of(h3b_win w, int p0, int p1, int n, int unit) {
    return h3b_win_tiles_rows(h3b_win_of(w, p0, n), h3b_win_of(w, p1, n), unit);
}

static H3B_HD int h3b_win_tile(h3b_win_tiles t, int i) { return i < t.sink ? i : t.from + i - t.sink; }

/* some query of a group sees some key of [k0, k0 + unit): hi of its last row, lo of its first, s of its last */
static H3B_HD int h3b_win_any(int hi, int lo, int s, int k0, int unit) {
    return k0 <= hi && (k0 + unit > lo || k0 < s);
}

/* every query at p0..p1 sees every key of [k0, k0 + unit): a is the row of p0, z of p1 */
static H3B_HD int h3b_win_full(h3b_win_row a, h3b_win_row z, int k0, int unit) {
    return k0 + unit - 1 <= a.hi && (k0 >= z.lo || k0 + unit <= a.s);
}

#endif
