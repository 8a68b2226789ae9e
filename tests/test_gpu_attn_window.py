"""Windowed attention with sinks, the paged 8-bit key/value cache and attention over it, against the definitions in 64
bits (torch float64 on the same inputs).

Tolerance, element by element, derived from the kernels' roundings.  With A = sum_j p_j |v_j| (p the exact
probabilities): every probability is rounded once to the 16-bit operand type (u = half a step: bf16 2^-8, f16 2^-11; the
8-bit cache always takes f16 probabilities), which moves the row by at most u A; the result is rounded once to the output
type, u_out |o| <= u_out A; what is computed in 32 bits (scores of 128 products, exponentials with a relative error of
at most 8.6e-5 < 2^-13, sums) adds less than 2^-12 A.  The probabilities are rounded under a maximum that may be stale by
2^8, which changes no relative error.  Values below 2^-24 of the row's maximum may underflow in f16: 2^-24 max|v| per key."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}


@pytest.fixture(scope="module")
def cuda():
    import h3c_b200
    c = h3c_b200.Cuda(0)
    yield c
    c.check()
    c.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def mask(pos, n, left, right, sinks, block):
    """[rows, n] of truth values, from the definition."""
    p = torch.as_tensor(pos, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")[None]
    b = p - p % block
    ok = (j >= b - left) | (j < sinks) if left >= 0 else torch.ones_like(j - p, dtype=torch.bool)
    if right >= 0:
        ok = ok & (j <= b + block - 1 + right)
    return ok & (p >= 0)


def attend(q, k, v, seen, scale):
    """q [rows, H, 128], k / v [n, KV, 128] -> (out, A) [rows, H * 128] in 64 bits; masked keys are left out entirely."""
    rows, heads = q.shape[0], q.shape[1]
    g = heads // k.shape[1]
    out, a = (torch.zeros(rows, heads, 128, dtype=torch.float64, device="cuda") for _ in range(2))
    if not k.shape[0]:
        return out.view(rows, -1), a.view(rows, -1)
    for h in range(heads):
        kk, vv = k[:, h // g].double(), v[:, h // g].double()
        live = seen.any(0)
        kk, vv, m = kk[live], vv[live], seen[:, live]
        if not kk.shape[0]:
            continue
        kk, vv = torch.where(torch.isfinite(kk), kk, 0.0), torch.where(torch.isfinite(vv), vv, 0.0)
        z = (q[:, h].double() @ kk.T) * scale
        z = z.masked_fill(~m, -math.inf)
        top = z.amax(1, keepdim=True)
        p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        t = p.sum(1, keepdim=True)
        p = p / torch.where(t > 0, t, 1.0)
        out[:, h], a[:, h] = p @ vv, p @ vv.abs()
    return out.view(rows, -1), a.view(rows, -1)


def close(got, want, a, v_max, dtype, p_dtype=None):
    tol = (U[p_dtype or dtype] + U[dtype] + 2.0 ** -12) * a + 2.0 ** -24 * v_max
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements off, worst {float((off - tol).max()):.3e} over the tolerance, at {bad.nonzero()[0].tolist()}"


def check_window(cuda, q, k, v, got=None, scale=None, **w):
    full = dict(left=-1, right=-1, sinks=0, block=1, q_pos=0) | w
    if got is None:
        got = cuda.sdpa_window(q, k, v, scale=scale, **full)
    q_pos = full.pop("q_pos")
    seen = mask(np.arange(q.shape[0]) + q_pos, k.shape[0], **full)
    want, a = attend(q, k, v, seen, 128 ** -0.5 if scale is None else scale)
    vf = v[torch.isfinite(v)]
    close(got, want, a, float(vf.abs().max()) if vf.numel() else 0.0, q.dtype)
    empty = ~seen.any(1)
    assert not got[empty].any()
    return got


# ------------------------------------------------------------------ 16-bit keys and values

WINDOWS = [dict(), dict(left=-1, right=0), dict(left=0, right=0), dict(left=5, right=0, sinks=2), dict(left=100, right=77, sinks=5),
           dict(left=64, right=0, sinks=64, block=64), dict(left=40, right=3, sinks=100, block=50), dict(left=0, right=0, block=1000),
           dict(left=300, right=-1, sinks=1), dict(left=-1, right=20, sinks=9)]


@pytest.mark.parametrize("w", WINDOWS, ids=str)
@pytest.mark.parametrize("lq, lk, heads, kv, q_pos, dtype", [
    (1, 1, 1, 1, 0, BF), (1, 700, 6, 2, 699, HF), (3, 129, 4, 4, 100, BF), (16, 400, 2, 1, 384, HF), (17, 300, 3, 3, 283, BF),
    (130, 515, 4, 2, 300, BF), (257, 257, 3, 1, 0, HF), (600, 600, 2, 2, 0, BF), (300, 900, 7, 1, 600, HF)])
def test_window(cuda, w, lq, lk, heads, kv, q_pos, dtype):
    g = gen(lq * 1000 + lk)
    q, k, v = normal(g, lq, heads, 128, dtype=dtype), normal(g, lk, kv, 128, dtype=dtype), normal(g, lk, kv, 128, dtype=dtype)
    check_window(cuda, q, k, v, q_pos=q_pos, **w)


@pytest.mark.parametrize("lq, lk, w", [(1, 20000, dict(left=4095, right=0, sinks=64)), (4, 33333, dict(left=-1, right=0)),
                                       (40, 9000, dict(left=-1, right=0)), (1000, 5000, dict(left=1500, right=0, sinks=10, block=250))])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_window_over_long_keys(cuda, lq, lk, w, dtype):
    g = gen(lk)
    q, k, v = normal(g, lq, 4, 128, dtype=dtype), normal(g, lk, 2, 128, dtype=dtype), normal(g, lk, 2, 128, dtype=dtype)
    check_window(cuda, q, k, v, q_pos=lk - lq, **w)


@pytest.mark.parametrize("lq, lk, heads, kv, w", [
    (6144, 6144, 24, 24, dict(left=2048, right=0, sinks=1024, block=1024)),     # several items for every SM
    (1531, 7919, 56, 8, dict(left=1000, right=77, sinks=5)),                     # 126-row tiles, a last round that is partly empty
    (1620, 9000, 24, 24, dict(left=-1, right=0, block=1620)),                    # whole rounds and a rest whose keys are split
    (1500, 9000, 3, 1, dict(left=-1, right=0)), (700, 300, 126, 14, dict(left=3, right=3))])
def test_window_full_size_sampled(cuda, lq, lk, heads, kv, w):
    g = gen(lq)
    q, k, v = normal(g, lq, heads, 128, dtype=BF), normal(g, lk, kv, 128, dtype=BF), normal(g, lk, kv, 128, dtype=BF)
    got = cuda.sdpa_window(q, k, v, q_pos=max(0, lk - lq), **w).view(lq, heads, 128)
    cuda.check()
    rows = torch.unique(torch.cat([torch.arange(0, lq, 97, device="cuda"), torch.arange(max(0, lq - 130), lq, 3, device="cuda"),
                                   torch.arange(0, min(lq, 260), 5, device="cuda")]))
    seen = mask(rows.cpu().numpy() + max(0, lk - lq), lk, w["left"], w["right"], w.get("sinks", 0), w.get("block", 1))
    for h in sorted({0, heads // 2, heads - 1}):
        kv_h = h // (heads // kv)
        want, a = attend(q[rows, h:h + 1], k[:, kv_h:kv_h + 1], v[:, kv_h:kv_h + 1], seen, 128 ** -0.5)
        close(got[rows, h], want, a, float(v.float().abs().max()), BF)


def test_window_without_bounds_is_the_frameworks_attention(cuda):
    g = gen(3)
    q, k, v = (normal(g, n, 4, 128, dtype=BF) for n in (500, 700, 700))
    a, b = cuda.sdpa_window(q, k, v).float(), cuda.sdpa(q, k, v).float()
    # two evaluations whose probabilities and results are each rounded to bf16
    assert float((a - b).abs().max()) <= 4 * U[BF] * float(v.float().abs().max())


def test_window_rows_that_see_nothing_are_zero(cuda):
    g = gen(4)
    for lq, lk in ((1, 5), (9, 100), (200, 64), (300, 40)):
        q, k, v = normal(g, lq, 2, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF)
        assert not cuda.sdpa_window(q, k, v, left=3, right=0, q_pos=lk + 10).any()       # wholly behind the keys
        check_window(cuda, q, k, v, left=3, right=0, q_pos=max(0, lk - 5))                # partly
        check_window(cuda, q, k, v, left=3, right=0, sinks=1, q_pos=lk + 10)              # a sink alone
    assert not cuda.sdpa_window(normal(g, 20, 2, 128, dtype=HF), torch.empty(0, 2, 128, dtype=HF, device="cuda"),
                                torch.empty(0, 2, 128, dtype=HF, device="cuda")).any()     # no keys at all
    assert cuda.sdpa_window(torch.empty(0, 2, 128, dtype=HF, device="cuda"), k.half(), v.half()).shape == (0, 256)


@pytest.mark.parametrize("lq", [1, 5, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_window_masked_keys_have_no_part_in_the_result(cuda, lq, bad):
    g = gen(5)
    lk, w = 777, dict(left=50, right=0, sinks=3, q_pos=500)
    q, k, v = normal(g, lq, 4, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF)
    want = check_window(cuda, q, k, v, **w)
    seen = mask(np.arange(lq) + 500, lk, 50, 0, 3, 1).any(0)
    k[~seen], v[~seen] = bad, bad
    got = cuda.sdpa_window(q, k, v, **w)
    assert torch.equal(got, want)
    # a key that some rows of a tile see and others do not: the others are as before
    if lq == 200:
        k2, v2 = k.clone(), v.clone()
        k2[520], v2[520] = float("nan"), float("nan")
        got = cuda.sdpa_window(q, k2, v2, **w)
        sees_it = mask(np.arange(lq) + 500, lk, 50, 0, 3, 1)[:, 520]
        assert got[sees_it].isnan().all()
        u = U[BF]
        assert float((got[~sees_it].float() - want[~sees_it].float()).abs().max()) <= 4 * u * float(v[seen].float().abs().max())
        v3 = v.clone()
        v3[520, :, 7] = bad
        got = cuda.sdpa_window(q, k, v3, **w)
        assert not torch.isfinite(got.view(lq, 4, 128)[sees_it][..., 7]).any()
        fine = got.view(lq, 4, 128).clone()
        fine[..., 7] = 0
        assert torch.isfinite(fine).all() and torch.isfinite(got[~sees_it]).all()


def test_window_visible_nan_reaches_the_rows_that_see_it(cuda):
    g = gen(6)
    for lq, lk in ((2, 300), (260, 300)):
        for where in (0, 3, 9, 130, 299):
            q, k, v = normal(g, lq, 2, 128, dtype=HF), normal(g, lk, 2, 128, dtype=HF), normal(g, lk, 2, 128, dtype=HF)
            k[where, 1, 5] = float("nan")
            got = cuda.sdpa_window(q, k, v, left=-1, right=0, q_pos=lk - lq).view(lq, 2, 128)
            sees = torch.arange(lk - lq, lk, device="cuda") >= where
            assert got[sees, 1].isnan().all() and torch.isfinite(got[~sees, 1]).all() and torch.isfinite(got[:, 0]).all()


def test_window_strides_orders_and_views(cuda):
    g = gen(7)
    w = dict(left=90, right=4, sinks=6, q_pos=100)
    for lq in (2, 150):
        fused = normal(g, 400, 6 + 2 + 2, 128, dtype=BF)                                  # one projection's rows
        q, k, v = fused[:lq, :6], fused[:, 6:8], fused[:, 8:]
        check_window(cuda, q, k, v, **w)
        heads_first = [normal(g, h, n, 128, dtype=BF).transpose(0, 1) for h, n in ((6, lq), (2, 400), (2, 400))]
        check_window(cuda, *heads_first, **w)
        wide = [normal(g, n, h, 136, dtype=BF)[..., 8:] for h, n in ((6, lq), (2, 400), (2, 400))]
        check_window(cuda, *wide, **w)
        every = [normal(g, 2 * n, h, 128, dtype=BF)[::2] for h, n in ((6, lq), (2, 400), (2, 400))]
        check_window(cuda, *every, **w)
        for first, wide in ((0, 6 * 128 + 64), (8, 6 * 128 + 24)):                          # out inside something larger, 16-byte aligned
            room = torch.full((lq + 5, wide), 3.0, dtype=BF, device="cuda")
            check_window(cuda, q, k, v, got=cuda.sdpa_window(q, k, v, out=room[:lq, first:first + 768], **w), **w)
            assert (room[lq:] == 3).all() and (room[:, :first] == 3).all() and (room[:, first + 768:] == 3).all()


@pytest.mark.parametrize("lq", [1, 150])
def test_window_offsets_past_32_bits(cuda, lq):
    g = gen(8)
    rows, stride = 1100, 2 ** 21 + 64                                                     # 2.3 G elements apart
    room = torch.empty(rows * stride + 1024, dtype=HF, device="cuda")
    k, v = (torch.as_strided(room, (rows, 2, 128), (stride, 128, 1), off) for off in (0, 512))
    k.copy_(normal(g, rows, 2, 128, dtype=HF))
    v.copy_(normal(g, rows, 2, 128, dtype=HF))
    q = normal(g, lq, 4, 128, dtype=HF)
    check_window(cuda, q, k, v, left=200, right=0, sinks=4, q_pos=rows - lq)


def test_window_large_scores_and_growing_maximum(cuda):
    g = gen(9)
    for lq in (2, 140):
        q, k, v = normal(g, lq, 2, 128, dtype=BF), normal(g, 1000, 2, 128, dtype=BF), normal(g, 1000, 2, 128, dtype=BF)
        k *= torch.linspace(0.01, 30, 1000, device="cuda")[:, None, None].to(BF)           # later keys dominate earlier ones
        # scores of up to some hundreds: their own f32 rounding (2^-24 of |q||k|) is exponentiated
        q64 = (q.double().abs().sum(-1).max() * k.double().abs().max() * 128 ** -0.5).item()
        assert q64 * 2.0 ** -24 * 8 < 2.0 ** -8
        got = cuda.sdpa_window(q, k, v, left=800, right=0, sinks=3, q_pos=1000 - lq)
        seen = mask(np.arange(lq) + 1000 - lq, 1000, 800, 0, 3, 1)
        want, a = attend(q, k, v, seen, 128 ** -0.5)
        close(got, want, a * (1 + q64 * 2.0 ** -24 * 8 / (2 * U[BF])), float(v.float().abs().max()), BF)


def test_window_argument_checks_in_python(cuda):
    import h3c_b200
    q, k = torch.zeros(4, 4, 128, dtype=BF, device="cuda"), torch.zeros(9, 2, 128, dtype=BF, device="cuda")
    for args in ((q.float(), k, k), (q, k.half(), k), (q, k, k[:5]), (q[..., :64], k, k), (q[0], k, k), (q, k.cpu(), k),
                 (q.transpose(0, 2).contiguous().transpose(0, 2), k, k), (q, k.expand(9, 2, 128).as_strided((9, 2, 128), (0, 128, 1)), k),
                 (q[:, :3], k, k)):
        with pytest.raises(h3c_b200.H3Error):
            cuda.sdpa_window(*args)
    for out in (torch.empty(4, 512, dtype=HF, device="cuda"), torch.empty(3, 512, dtype=BF, device="cuda"), torch.empty(4, 512, dtype=BF),
                torch.empty(512, 4, dtype=BF, device="cuda").t()):
        with pytest.raises(h3c_b200.H3Error):
            cuda.sdpa_window(q, k, k, out=out)


# ------------------------------------------------------------------ the 8-bit cache

def scale_of(top):
    """Smallest power of two 2^e, e >= -64, with top <= 448 * 2^e (64-bit)."""
    m, e = torch.frexp(top.double() / 448)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.exp2(torch.where(top > 0, e, -64).clamp(min=-64).double())


class Model:
    """The cache by its definition: one sequence after the other, block by block."""

    def __init__(self, cache):
        self.k, self.v = (t.view(torch.float8_e4m3fn).float().double() for t in (cache.k, cache.v))
        self.ks, self.vs = cache.k_scale.double(), cache.v_scale.double()
        self.page = cache.k.shape[2]

    def append(self, k, v, cu, start, table):
        for s in range(len(start)):
            n, at = cu[s + 1] - cu[s], start[s]
            done = 0
            while done < n:
                p = at + done
                take, o = min(64 - p % 64, n - done), p % 64
                pg, b = table[s][p // self.page], p % self.page // 64
                for x, codes, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    piece = x[cu[s] + done:cu[s] + done + take].double().transpose(0, 1)
                    sc = scale_of(piece.abs().amax((1, 2)))
                    blk = codes[pg, :, b * 64:(b + 1) * 64]
                    if o:
                        old = scales[pg, :, b].clone()
                        sc = torch.maximum(sc, old)
                        blk[:, :o] = (blk[:, :o] * (old / sc)[:, None, None]).float().to(torch.float8_e4m3fn).double()
                    blk[:, o:o + take] = (piece / sc[:, None, None]).float().to(torch.float8_e4m3fn).double()
                    scales[pg, :, b] = sc
                done += take

    def same_as(self, cache):
        for mine, his in ((self.k, cache.k), (self.v, cache.v), (self.ks, cache.k_scale), (self.vs, cache.v_scale)):
            his = his.view(torch.float8_e4m3fn).float() if his.dtype in (torch.uint8, torch.float8_e4m3fn) else his
            assert torch.equal(mine, his.double())

    def values(self, s, n, table):
        t = torch.as_tensor(table[s][:-(-n // self.page)], device="cuda").long()
        return tuple((c[t] * sc[t].repeat_interleave(64, -1)[..., None]).transpose(1, 2).reshape(-1, c.shape[1], 128)[:n]
                     for c, sc in ((self.k, self.ks), (self.v, self.vs)))


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device="cuda")


def pages_of(rng, lens, page, pool, width=None):
    """A page list for each sequence out of a shuffled pool; -1 behind its end."""
    order = rng.permutation(pool)
    need = [-(-int(n) // page) for n in lens]
    assert sum(need) <= pool
    width = width or max(max(need), 1)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table


def filled(cuda, rng, g, lens, page, kv, dtype=BF, spread=True):
    """A cache of `lens` tokens per sequence, put there by the operator in two calls; with its model."""
    pool = sum(-(-int(n) // page) for n in lens) + 3
    cache = cuda.kv8_cache(pool, page, kv)
    table = pages_of(rng, lens, page, pool)
    model = Model(cache)
    first = [int(rng.integers(0, n + 1)) for n in lens]
    for rows, start in ((first, [0] * len(lens)), ([n - f for n, f in zip(lens, first)], first)):
        cu = np.concatenate([[0], np.cumsum(rows)])
        k, v = normal(g, int(cu[-1]), kv, 128, dtype=torch.float32), normal(g, int(cu[-1]), kv, 128, dtype=torch.float32)
        if spread:                                   # rows of very different size: scales grow, codes become subnormal
            k, v = (x * torch.exp2(torch.randint(-9, 5, (x.shape[0], 1, 1), generator=g, device="cuda").float()) for x in (k, v))
        k, v = k.to(dtype), v.to(dtype)
        cuda.kv8_append(cache, k, v, i32(cu), i32(start), i32(table), max_rows=max(rows))
        model.append(k, v, cu, start, table)
    return cache, table, model


@pytest.mark.parametrize("lens, page, kv, dtype", [([1], 64, 1, BF), ([64], 64, 2, HF), ([65, 0, 1, 63], 64, 3, BF), ([500, 77, 130], 128, 2, HF),
                                                   ([1000, 3, 64, 640, 129], 192, 5, BF), ([300] * 40, 256, 1, BF)])
def test_append_gives_the_codes_and_scales_of_the_definition(cuda, lens, page, kv, dtype):
    rng, g = np.random.default_rng(sum(lens)), gen(sum(lens))
    cache, _, model = filled(cuda, rng, g, lens, page, kv, dtype)
    cuda.check()
    model.same_as(cache)


def test_append_token_by_token_and_over_again(cuda):
    rng, g = np.random.default_rng(5), gen(5)
    cache = cuda.kv8_cache(6, 64, 2)
    table = pages_of(rng, [140, 100], 64, 6)
    model = Model(cache)
    for t in range(100):
        k, v = (normal(g, 2, 2, 128, dtype=BF) * (1 + 0.2 * t) for _ in range(2))
        cuda.kv8_append(cache, k, v, i32([0, 1, 2]), i32([t + 40, t]), i32(table), max_rows=1)
        model.append(k, v, [0, 1, 2], [t + 40, t], table)
    model.same_as(cache)
    k, v = normal(g, 30, 2, 128, dtype=BF) * 0.01, normal(g, 30, 2, 128, dtype=BF)          # a draft is taken back: from token 70 on
    cuda.kv8_append(cache, k, v, i32([0, 0, 30]), i32([0, 70]), i32(table), max_rows=30)
    model.append(k, v, [0, 0, 30], [0, 70], table)
    model.same_as(cache)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    cuda.kv8_append(cache, k, v, i32([0, 0, 30]), i32([0, 70]), i32(table), max_rows=30)    # the same rows again change nothing
    for a, b in zip(before, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
        assert torch.equal(a, b)


def test_append_borders_of_the_scale(cuda):
    cache = cuda.kv8_cache(1, 64, 1)
    for dtype, tops in ((BF, [448.0, 450.0, 224.0, 1.0, 1.75, 1.7578125, 1e-30, 1e-20, 3.3e38, 0.0, 2.0 ** -133]),
                        (HF, [448.0, 448.25, 65504.0, 6e-8, 0.875, 0.8755, 0.0])):
        for top in tops:
            k = torch.zeros(64, 1, 128, dtype=dtype, device="cuda")
            k[17, 0, 99], k[3, 0, 1] = -top, top / 3
            cuda.kv8_append(cache, k, k, i32([0, 64]), i32([0]), i32([[0]]), max_rows=64)
            model = Model(cuda.kv8_cache(1, 64, 1))
            model.append(k, k, [0, 64], [0], [[0]])
            model.same_as(cache)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_of_a_value_that_is_not_finite(cuda, bad):
    g = gen(8)
    cache = cuda.kv8_cache(3, 64, 2)
    k, v = normal(g, 150, 2, 128, dtype=BF), normal(g, 150, 2, 128, dtype=BF)
    k[70, 1, 9] = bad
    table = i32([[2, 0, 1]])
    cuda.kv8_append(cache, k, v, i32([0, 150]), i32([0]), table, max_rows=150)
    assert cache.k_scale.isnan().sum() == 1 and cache.k_scale[0, 1, 0].isnan() and not cache.v_scale.isnan().any()
    assert not cache.k.view(torch.uint8)[0, 1].any()
    q = normal(g, 150, 2, 128, dtype=BF)
    for rows in (150, 3):
        out = cuda.kv8_sdpa(cache, q[150 - rows:], i32([0, rows]), i32([150]), table, max_rows=rows, max_len=150, left=20).view(rows, 2, 128)
        pos = torch.arange(150 - rows, 150, device="cuda")
        sees = (pos >= 64) & (pos - 20 <= 127)
        assert out[sees, 1].isnan().all() and torch.isfinite(out[~sees, 1]).all() and torch.isfinite(out[:, 0]).all()
    # further tokens of the block keep it so; the block started again is clean
    cuda.kv8_append(cache, k[:5], v[:5], i32([0, 5]), i32([100]), table, max_rows=5)
    assert cache.k_scale[0, 1, 0].isnan()
    cuda.kv8_append(cache, k[:64], v[:64], i32([0, 64]), i32([64]), table, max_rows=64)
    assert torch.isfinite(cache.k_scale).all()


def check_cache(cuda, cache, table, model, q, cu, lens, got=None, scale=None, **w):
    full = dict(left=-1, right=0, sinks=0, block=1) | w
    rows = max(int(cu[s + 1] - cu[s]) for s in range(len(lens)))
    if got is None:
        got = cuda.kv8_sdpa(cache, q, i32(cu), i32(lens), i32(table), max_rows=rows, max_len=max(max(lens), 1), scale=scale, **full)
        cuda.check()
    for s, n in enumerate(lens):
        r0, r1 = int(cu[s]), int(cu[s + 1])
        if r0 == r1:
            continue
        k, v = model.values(s, n, table)
        seen = mask(np.arange(n - (r1 - r0), n), n, **full)
        want, a = attend(q[r0:r1], k, v, seen, 128 ** -0.5 if scale is None else scale)
        # one E4M3 code may underflow under its block's maximum: nothing further, values are exact products
        close(got[r0:r1], want, a, float(v.abs().max()) if n else 0.0, q.dtype, HF)
        assert not got[r0:r1][~seen.any(1)].any()
    return got


CACHE_WINDOWS = [dict(), dict(left=0), dict(left=70, sinks=3), dict(left=100, right=20, sinks=130), dict(left=-1, right=-1),
                 dict(left=64, block=64, sinks=1), dict(left=33, block=50, right=1, sinks=70)]


@pytest.mark.parametrize("w", CACHE_WINDOWS, ids=str)
@pytest.mark.parametrize("rows, lens, heads, kv, page, dtype", [
    ([1], [1], 1, 1, 64, BF), ([1, 1, 1], [5, 300, 64], 4, 4, 64, HF), ([1] * 5, [700, 1, 64, 65, 2000], 14, 2, 128, BF),
    ([4, 1, 0, 3], [400, 7, 90, 3], 6, 2, 64, BF), ([16, 2], [500, 129], 3, 3, 192, HF), ([5, 8], [333, 444], 10, 2, 64, BF),
    ([40, 1, 77], [700, 200, 77], 4, 2, 64, BF), ([130, 300], [130, 900], 6, 1, 128, HF), ([257], [1025], 2, 2, 256, BF),
    ([20, 33], [400, 1000], 7, 1, 64, HF)])
def test_cache_attention(cuda, w, rows, lens, heads, kv, page, dtype):
    rng, g = np.random.default_rng(sum(lens)), gen(sum(lens) + heads)
    cache, table, model = filled(cuda, rng, g, lens, page, kv, dtype, spread=False)
    cu = np.concatenate([[0], np.cumsum(rows)])
    check_cache(cuda, cache, table, model, normal(g, int(cu[-1]), heads, 128, dtype=dtype), cu, lens, **w)


@pytest.mark.parametrize("rows, lens", [([1, 2], [900, 300]), ([64, 100], [300, 900])])
def test_cache_attention_over_blocks_of_very_different_scales(cuda, rows, lens):
    rng, g = np.random.default_rng(2), gen(2)
    cache, table, model = filled(cuda, rng, g, lens, 64, 2, BF, spread=True)
    cache.v_scale *= torch.exp2(torch.randint(-30, 30, cache.v_scale.shape, generator=g, device="cuda").float())   # powers of two stay so
    model = Model(cache)
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = normal(g, int(cu[-1]), 4, 128, dtype=BF) * 0.2
    got = cuda.kv8_sdpa(cache, q, i32(cu), i32(lens), i32(table), max_rows=max(rows), max_len=max(lens))
    for s, n in enumerate(lens):
        k, v = model.values(s, n, table)
        r0, r1 = cu[s], cu[s + 1]
        seen = mask(np.arange(n - (r1 - r0), n), n, -1, 0, 0, 1)
        want, a = attend(q[r0:r1], k, v, seen, 128 ** -0.5)
        # what a key adds is held in f16 next to the largest probability * scale: 2^-24 of the row's largest |v| scale
        close(got[r0:r1], want, a, 448 * float(model.vs.max()) * 2.0, BF, HF)


def test_cache_attention_with_large_and_small_queries(cuda):
    rng, g = np.random.default_rng(3), gen(3)
    cache, table, model = filled(cuda, rng, g, [500], 64, 2, BF, spread=False)
    for rows in (2, 150):
        for size in (1e-30, 1e-4, 40.0):
            q = normal(g, rows, 4, 128, dtype=BF) * size
            check_cache(cuda, cache, table, model, q, [0, rows], [500], scale=128 ** -0.5 / size)


def test_cache_attention_of_evicted_pages_and_stale_memory(cuda):
    """Pages wholly outside the window may hold any index; tokens behind the length may hold any bytes."""
    rng, g = np.random.default_rng(4), gen(4)
    for rows in (1, 90):
        cache, table, model = filled(cuda, rng, g, [1000, 210], 64, 2, BF, spread=False)
        cu = [0, rows, 2 * rows]
        q = normal(g, 2 * rows, 4, 128, dtype=BF)
        want = check_cache(cuda, cache, table, model, q, cu, [1000, 210], left=100, sinks=70)
        bad = table.copy()
        bad[0, 2:(1000 - rows - 100) // 64] = 1 << 30
        bad[1, 4:] = -7
        cache.k.view(torch.uint8)[table[1, 3], :, 210 - 192:] = 0x7f                    # NaN patterns behind token 210
        cache.v.view(torch.uint8)[table[1, 3], :, 210 - 192:] = 0xff
        got = cuda.kv8_sdpa(cache, q, i32(cu), i32([1000, 210]), i32(bad), max_rows=rows, max_len=1000, left=100, sinks=70)
        cuda.check()
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows, lens, heads, kv, w", [
    ([1620], [9000], 24, 24, dict(block=1620)), ([700, 1, 333, 701, 64, 2, 500, 90, 17], [9000, 1000, 333, 8000, 64, 5000, 700, 3000, 2000], 24, 6, dict(left=2047, sinks=64)),
    ([1] * 64, [100 + 117 * i for i in range(64)], 28, 4, dict()), ([300] * 20, [300 + 50 * i for i in range(20)], 12, 4, dict(left=500))])
def test_cache_full_size_sampled(cuda, rows, lens, heads, kv, w):
    rng, g = np.random.default_rng(sum(lens)), gen(sum(lens))
    pool = sum(-(-n // 64) for n in lens) + 1
    cache = cuda.kv8_cache(pool, 64, kv)
    table = pages_of(rng, lens, 64, pool)
    cu_k = np.concatenate([[0], np.cumsum(lens)])
    k, v = normal(g, int(cu_k[-1]), kv, 128, dtype=BF), normal(g, int(cu_k[-1]), kv, 128, dtype=BF)
    cuda.kv8_append(cache, k, v, i32(cu_k), i32([0] * len(lens)), i32(table), max_rows=max(lens))
    model = Model(cache)
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = normal(g, int(cu[-1]), heads, 128, dtype=BF)
    got = cuda.kv8_sdpa(cache, q, i32(cu), i32(lens), i32(table), max_rows=max(rows), max_len=max(lens), **w).view(-1, heads, 128)
    cuda.check()
    full = dict(left=-1, right=0, sinks=0, block=1) | w
    for s, n in enumerate(lens):
        kk, vv = model.values(s, n, table)
        pick = torch.unique(torch.cat([torch.arange(0, rows[s], 61, device="cuda"), torch.arange(max(0, rows[s] - 3), rows[s], device="cuda")]))
        seen = mask(n - rows[s] + pick.cpu().numpy(), n, **full)
        for h in {s % heads, heads - 1}:
            kv_h = h // (heads // kv)
            want, a = attend(q[cu[s]:cu[s + 1]][pick, h:h + 1], kk[:, kv_h:kv_h + 1], vv[:, kv_h:kv_h + 1], seen, 128 ** -0.5)
            close(got[cu[s]:cu[s + 1]][pick, h], want, a, float(vv.abs().max()), BF, HF)


def test_cache_sequences_that_share_pages(cuda):
    rng, g = np.random.default_rng(6), gen(6)
    cache, table, model = filled(cuda, rng, g, [640], 64, 2, BF, spread=False)
    both = np.concatenate([table, table])
    q = normal(g, 2, 4, 128, dtype=BF)
    got = check_cache(cuda, cache, both, model, q, [0, 1, 2], [640, 320])
    assert not torch.equal(got[0], got[1])


def test_cache_rows_of_no_sequence_are_left_as_they_are(cuda):
    rng, g = np.random.default_rng(7), gen(7)
    cache, table, model = filled(cuda, rng, g, [100, 90], 64, 1, BF, spread=False)
    for rows in (1, 30):
        q = normal(g, 2 * rows + 9, 2, 128, dtype=BF)
        out = torch.full((2 * rows + 9, 256), 5.0, dtype=BF, device="cuda")
        cuda.kv8_sdpa(cache, q, i32([4, 4 + rows, 4 + 2 * rows]), i32([100, 90]), i32(table), max_rows=rows, max_len=100, out=out)
        check_cache(cuda, cache, table, model, q, [4, 4 + rows, 4 + 2 * rows], [100, 90], got=out)
        assert (out[:4] == 5).all() and (out[4 + 2 * rows:] == 5).all()


def test_cache_lengths_shorter_than_the_rows_and_max_len_as_a_guess(cuda):
    rng, g = np.random.default_rng(9), gen(9)
    for rows, heads in ((6, 2), (50, 4)):
        cache, table, model = filled(cuda, rng, g, [300, 4], 64, 2, BF, spread=False)
        q = normal(g, 2 * rows, heads, 128, dtype=BF)
        cu = [0, rows, 2 * rows]
        a = check_cache(cuda, cache, table, model, q, cu, [300, 4])                    # rows in front of token 0 are zero
        for guess in (1, 64, 100000):
            b = cuda.kv8_sdpa(cache, q, i32(cu), i32([300, 4]), i32(table), max_rows=rows, max_len=guess)
            assert float((a.float() - b.float()).abs().max()) <= 4 * U[BF] * float(model.values(0, 300, table)[1].abs().max())
        none = cuda.kv8_sdpa(cache, q, i32(cu), i32([0, 0]), i32(table), max_rows=rows, max_len=1)
        assert not none.any()


@pytest.mark.parametrize("bits", [8, 16])
def test_long_sums_do_not_drift(cuda, bits):
    """Positive values, so that nothing cancels, of one page again and again: the weights of one page.  The bound: P in f16
    and the rounding of the output half a step each; products cut to 2^-25 of the sum, and the sum to 2^-23 of itself per 16
    keys, over the 32,768 keys of one accumulator; 2^-14 for scores and exponentials."""
    page, reps = 16384, 256 if bits == 8 else 16
    g, heads = gen(12), 32
    cache = cuda.kv8_cache(1, page, 1)
    cache.k_scale.fill_(1)
    cache.v_scale.fill_(1)
    cache.k.copy_(torch.randn(1, 1, page, 128, device="cuda", generator=g).to(torch.float8_e4m3fn))
    cache.v.copy_((1 + torch.rand(1, 1, page, 128, device="cuda", generator=g)).to(torch.float8_e4m3fn))
    k, v = cache.k[0, 0].double(), cache.v[0, 0].double()
    if bits == 8:                                              # one CTA: 4 million tokens
        q = (0.5 * torch.randn(8, heads, 128, device="cuda", generator=g)).to(HF)
        table = torch.zeros(1, reps, dtype=torch.int32, device="cuda")
        got = cuda.kv8_sdpa(cache, q, i32([0, 8]), i32([page * reps]), table, max_rows=8, max_len=1, right=-1)
    else:                                                      # as many items as fill the chip: 262,144 keys each
        q = (0.5 * torch.randn(1280, heads, 128, device="cuda", generator=g)).to(HF)
        kk, vv = (x.to(HF).repeat(reps, 1)[:, None].contiguous() for x in (cache.k[0, 0], cache.v[0, 0]))
        got = cuda.sdpa_window(q, kk, vv)
    cuda.check()
    some = slice(0, q.shape[0] * heads, max(1, q.shape[0] // 8))
    want = torch.softmax(q.reshape(-1, 128)[some].double() @ k.T * 128 ** -0.5, -1) @ v
    worst = float((got.view(-1, 128)[some].double() / want - 1).abs().max())
    assert worst <= 2 * 2.0 ** -11 + 32768 * (2.0 ** -25 + 2.0 ** -27) + 2.0 ** -14, worst


def test_an_item_that_runs_longer_than_a_wait_may(cuda):
    """200 million tokens of one sequence (one page, listed again and again) that a small max_len leaves to one CTA: some
    1.6 million key tiles, about 3 s, while a wait gives up after 4e9 cycles, some 2 s, without any progress.  Keys of zero
    make every probability 1, so that a row's sums are its keys times a power of two: exact in one accumulator (32,768 keys)
    and, as multiples of 32,768 (64) below 2^39 (2^30), in what adds them up, but for the last tile, where one rounding of
    2^-24 is less than half a step of the output."""
    n, page, rows, heads = 200_000_000, 65536, 8, 32
    cache = cuda.kv8_cache(1, page, 1)
    values = 2.0 ** (torch.arange(128, device="cuda") % 5 - 3) * (1 - 2 * (torch.arange(128, device="cuda") % 2))
    cache.k_scale.fill_(1)
    cache.v_scale.fill_(1)
    cache.v.copy_(values.expand(1, 1, page, 128).to(torch.float8_e4m3fn))
    table = torch.zeros(1, -(-n // page), dtype=torch.int32, device="cuda")
    q = normal(gen(3), rows, heads, 128, dtype=BF)
    out = cuda.kv8_sdpa(cache, q, i32([0, rows]), i32([n]), table, max_rows=rows, max_len=1)
    cuda.check()
    assert torch.equal(out.float().view(rows, heads, 128), values.float().expand(rows, heads, 128))


def test_bad_extents_and_pages_are_reported_and_touch_nothing(cuda):
    import h3c_b200
    rng, g = np.random.default_rng(10), gen(10)
    for rows in (2, 40):
        cache, table, model = filled(cuda, rng, g, [200, 200], 64, 2, BF, spread=False)
        q = normal(g, 2 * rows, 4, 128, dtype=BF)
        cu, lens = [0, rows, 2 * rows], [200, 200]
        before = [t.clone() for t in (cache.k.view(torch.uint8), cache.k_scale)]
        x = normal(g, 2 * rows, 2, 128, dtype=BF)
        for bad_cu, bad_len, bad_table in (([0, rows, 3 * rows], lens, table), ([0, -1, rows], lens, table), ([2, 1, rows], lens, table),
                                           (cu, [200, 99999], table), (cu, [-1, 200], table), (cu, lens, np.full_like(table, 10 ** 6)),
                                           (cu, lens, np.full_like(table, -1))):
            cuda.kv8_sdpa(cache, q, i32(bad_cu), i32(bad_len), i32(bad_table), max_rows=rows, max_len=200)
            with pytest.raises(h3c_b200.H3Error, match="outside the call's arrays"):
                cuda.check()
        for bad_cu, bad_start, bad_table in (([0, 0, 3 * rows], [0, 0], table), ([0, 0, rows], [0, 99999], table), ([0, 0, rows], [0, -3], table),
                                             ([0, 0, rows], [0, 0], np.full_like(table, 10 ** 6)), ([0, 0, rows], [0, 0], np.full_like(table, -1))):
            cuda.kv8_append(cache, x, x, i32(bad_cu), i32(bad_start), i32(bad_table), max_rows=rows)
            with pytest.raises(h3c_b200.H3Error, match="outside the call's arrays"):
                cuda.check()
        assert torch.equal(before[0], cache.k.view(torch.uint8)) and torch.equal(before[1], cache.k_scale)
        check_cache(cuda, cache, table, model, q, cu, lens)


def test_cache_pool_past_32_bits(cuda):
    rng, g = np.random.default_rng(11), gen(11)
    pool = 2 ** 31 // (64 * 4 * 128) + 2000                                             # code offsets beyond 2^31 bytes
    cache = cuda.kv8_cache(pool, 64, 4)
    table = np.arange(pool - 10, pool, dtype=np.int32)[None]
    model = None
    for rows in (1, 100):
        k, v = normal(g, 600, 4, 128, dtype=BF), normal(g, 600, 4, 128, dtype=BF)
        cuda.kv8_append(cache, k, v, i32([0, 600]), i32([0]), i32(table), max_rows=600)
        small = type(cache)(*(t[pool - 10:].clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        model = Model(small)
        again = Model(cuda.kv8_cache(10, 64, 4))
        again.append(k, v, [0, 600], [0], table - (pool - 10))
        again.same_as(small)
        q = normal(g, rows, 8, 128, dtype=BF)
        got = cuda.kv8_sdpa(cache, q, i32([0, rows]), i32([600]), i32(table), max_rows=rows, max_len=600)
        check_cache(cuda, small, table - (pool - 10), model, q, [0, rows], [600], got=got)


# ------------------------------------------------------------------ as a program uses them

def test_a_stream_of_frames_through_the_cache(cuda):
    """Frames of 40 tokens: each is appended, then attends to the frames before it, itself and the first one."""
    rng, g = np.random.default_rng(12), gen(12)
    frame, frames, heads, kv = 40, 9, 6, 2
    cache, table = cuda.kv8_cache(8, 64, kv), rng.permutation(8)[None, :6].astype(np.int32)
    model = Model(cache)
    for f in range(frames):
        k, v, q = (normal(g, frame, h, 128, dtype=BF) for h in (kv, kv, heads))
        cuda.kv8_append(cache, k, v, i32([0, frame]), i32([f * frame]), i32(table), max_rows=frame)
        model.append(k, v, [0, frame], [f * frame], table)
        model.same_as(cache)
        check_cache(cuda, cache, table, model, q, [0, frame], [(f + 1) * frame], left=3 * frame, sinks=frame, block=frame)
    # the frames' values at once, as 16-bit tensors: the same windows
    k, v = model.values(0, frame * frames, table)
    check_window(cuda, normal(g, frame * frames, heads, 128, dtype=BF), k.to(BF), v.to(BF), left=3 * frame, right=0, sinks=frame, block=frame)


@pytest.mark.parametrize("rows", [1, 70])
def test_captured_decode_loop_follows_the_tables(cuda, rows):
    rng, g = np.random.default_rng(13), gen(13)
    kv, heads, n = 2, 4, 3
    cache, table = cuda.kv8_cache(40, 64, kv), i32(rng.permutation(40)[:36].reshape(n, 12))
    model = Model(cache)
    lens, cu = torch.zeros(n, dtype=torch.int32, device="cuda"), i32(np.arange(n + 1) * rows)
    k, v, q = (torch.zeros(n * rows, h, 128, dtype=BF, device="cuda") for h in (kv, kv, heads))

    def step():
        cuda.kv8_append(cache, k, v, cu, lens, table, max_rows=rows)
        lens.add_(rows)
        return cuda.kv8_sdpa(cache, q, cu, lens, table, max_rows=rows, max_len=700, left=300, sinks=4), \
            cuda.sdpa_window(q, k, v, left=10, right=0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(side):
            cuda.use_stream(side)
            step()
            lens.zero_()
            graphs = []
            for _ in range(2):                       # two captured graphs on one handle
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = step()
                graphs.append((graph, out))
            lens.zero_()
            for i in range(9):
                for t, h in ((k, kv), (v, kv), (q, heads)):
                    t.copy_(normal(g, n * rows, h, 128, dtype=BF))
                graph, (out, near) = graphs[i % 2]
                graph.replay()
                side.synchronize()
                model.append(k, v, cu.tolist(), [i * rows] * n, table.tolist())
                model.same_as(cache)
                check_cache(cuda, cache, table.cpu().numpy(), model, q, cu.tolist(), [(i + 1) * rows] * n, got=out, left=300, sinks=4)
                check_window(cuda, q, k, v, got=near, left=10, right=0)
    finally:
        torch.cuda.synchronize()
        cuda.use_stream(torch.cuda.current_stream())


def test_two_graphs_replayed_at_once(cuda):
    """Nothing is shared between two captured calls but the handle: their replays may overlap."""
    g = gen(17)
    rng = np.random.default_rng(17)
    cache, table, _ = filled(cuda, rng, g, [3000], 64, 4, BF, spread=False)
    side = [torch.cuda.Stream() for _ in range(2)]
    table, lens = i32(table), i32([3000])
    graphs, outs, wants = [], [], []
    try:
        for s, rows in zip(side, (3, 300)):
            q = normal(g, rows, 8, 128, dtype=BF)
            k, v = normal(g, 2000, 8, 128, dtype=BF), normal(g, 2000, 8, 128, dtype=BF)
            cu = i32([0, rows])
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                cuda.use_stream(s)
                step = lambda: (cuda.kv8_sdpa(cache, q, cu, lens, table, max_rows=rows, max_len=3000, left=1500),  # noqa: E731
                                cuda.sdpa_window(q, k, v, left=900, right=0, q_pos=2000 - rows, sinks=3))
                wants.append([o.clone() for o in step()])
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    outs.append(step())
                graphs.append((graph, q, k, v, cu))
        torch.cuda.synchronize()
        for _ in range(20):
            for s, (graph, *_) in zip(side, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, wants):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        torch.cuda.synchronize()
        cuda.use_stream(torch.cuda.current_stream())


def test_another_stream_than_the_current_one(cuda):
    """The handle works on its own stream while torch's current stream is another: outputs come from its memory."""
    g = gen(14)
    q, k, v = (normal(g, n, 4, 128, dtype=BF) for n in (100, 3000, 3000))
    cache = cuda.kv8_cache(50, 64, 4)
    table, cu, lens, zero = i32([np.arange(50)]), i32([0, 3000]), i32([3000]), i32([0])
    want = cuda.sdpa_window(q, k, v, left=500, sinks=5, right=0, q_pos=2900)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        cuda.use_stream(side)
        got = [cuda.sdpa_window(q, k, v, left=500, sinks=5, right=0, q_pos=2900) for _ in range(20)]
        cuda.kv8_append(cache, k, v, cu, zero, table, max_rows=3000)
        over = cuda.kv8_sdpa(cache, q, i32([0, 100]), lens, table, max_rows=100, max_len=3000)
        side.synchronize()
        assert all(torch.equal(o, want) for o in got)
        model = Model(cuda.kv8_cache(50, 64, 4))
        side.synchronize()
        model.append(k, v, [0, 3000], [0], table.tolist())
        model.same_as(cache)
        check_cache(cuda, cache, table.cpu().numpy(), model, q, [0, 100], [3000], got=over)
    finally:
        torch.cuda.synchronize()
        cuda.use_stream(torch.cuda.current_stream())


def test_two_handles_at_once(cuda):
    import h3c_b200
    g = gen(15)
    q, k, v = (normal(g, n, 8, 128, dtype=HF) for n in (3, 9000, 9000))
    want = cuda.sdpa_window(q, k, v, left=-1, right=0, q_pos=8997)
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles = [h3c_b200.Cuda(0) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for h, s in zip(handles, streams):
        h.use_stream(s)
    for _ in range(10):
        got += [h.sdpa_window(q, k, v, left=-1, right=0, q_pos=8997) for h in handles]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
    for h in handles:
        h.check()
        h.close()


def test_results_do_not_change_from_run_to_run(cuda):
    rng, g = np.random.default_rng(16), gen(16)
    cache, table, _ = filled(cuda, rng, g, [5000, 800], 64, 2, BF, spread=False)
    for rows in (1, 60):
        q = normal(g, 2 * rows, 6, 128, dtype=BF)
        outs = [cuda.kv8_sdpa(cache, q, i32([0, rows, 2 * rows]), i32([5000, 800]), i32(table), max_rows=rows, max_len=5000) for _ in range(5)]
        assert all(torch.equal(o, outs[0]) for o in outs)
