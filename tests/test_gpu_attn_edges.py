"""Windowed attention and the 8-bit cache at the edges of their contracts: pages that no row needs, values that are not
finite, probabilities far below the largest, scales of zero, orders of the cache's operands.  Definitions in 64 bits and
tolerances as in test_gpu_attn_window.py unless a test derives its own."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_attn_window import BF, HF, Model, check_cache, check_window, close, cuda, filled, gen, i32, mask, normal, pages_of  # noqa: E402, F401


# ------------------------------------------------------------------ pages that no row needs

@pytest.mark.parametrize("page", [64, 192])
@pytest.mark.parametrize("left, right, sinks, block", [(100, 0, s, 1) for s in (0, 1, 64, 65, 128)] + [
    (0, 0, 64, 1), (36, 0, 0, 1), (164, 0, 3, 1), (30, 0, 65, 50), (-1, 0, 0, 1), (0, 0, 0, 64)])
@pytest.mark.parametrize("rows, n", [(1, 1000), (7, 960), (40, 1000), (40, 1065), (64, 512), (300, 1000)])
def test_pages_that_no_row_needs_are_not_looked_at(cuda, rows, n, left, right, sinks, block, page):
    """A page without any visible key may be given to another sequence: its entry may hold any index.  Windows begin in odd
    and in even blocks of 64 tokens, sinks end in both."""
    rng, g = np.random.default_rng(n + sinks), gen(n + rows)
    cache, table, model = filled(cuda, rng, g, [n], page, 2, BF, spread=False)
    w = dict(left=left, right=right, sinks=sinks, block=block)
    q = normal(g, rows, 4, 128, dtype=BF)
    want = check_cache(cuda, cache, table, model, q, [0, rows], [n], **w)
    seen = mask(np.arange(n - rows, n), n, left, right, sinks, block).any(0).cpu().numpy()
    needed = np.array([seen[p * page:(p + 1) * page].any() for p in range(table.shape[1])])
    for index in (-1, 1 << 30):
        evicted = np.where(needed, table[0], index).astype(np.int32)[None]
        got = cuda.kv8_sdpa(cache, q, i32([0, rows]), i32([n]), i32(evicted), max_rows=rows, max_len=n, **w)
        cuda.check()
        assert torch.equal(got, want)


# ------------------------------------------------------------------ 16-bit values that are not finite

def place(v, where, g):
    """Puts values that are not finite into a copy of v [n, KV, 128]; returns it."""
    v, n = v.clone(), v.shape[0]
    inf, nan = float("inf"), float("nan")
    if where == "one":
        v[n // 2 + 3, 0, 77] = inf
    elif where == "first":
        v[0, :, 5], v[1, 0, 6] = -inf, nan
    elif where == "last":
        v[n - 1, 0, 0], v[n - 2, 0, 0], v[n - 3, 0, 127] = inf, -inf, nan
    elif where == "some":
        hit = torch.rand(v.shape, generator=g, device="cuda") < 3e-4
        pick = torch.tensor([inf, -inf, nan], device="cuda", dtype=v.dtype)[torch.randint(0, 3, v.shape, generator=g, device="cuda")]
        v = torch.where(hit, pick, v)
    elif where == "column":
        v[:, 0, 64] = inf
    elif where == "all":
        v[:] = nan
    return v


def check_odd_values(cuda, q, k, v, where, g, **w):
    """Against the same call with zeros in place of the values that are not finite: a row that sees none in a dimension is
    the same to the bit, one that sees some is what their sum is (probabilities here are far from underflow)."""
    full = dict(left=-1, right=-1, sinks=0, block=1, q_pos=0) | w
    odd = place(v, where, g)
    got = cuda.sdpa_window(q, k, odd, **full)
    cuda.check()
    fine = torch.isfinite(odd)
    want = cuda.sdpa_window(q, k, torch.where(fine, odd, 0), **full)
    q_pos = full.pop("q_pos")
    lq, heads, kv = q.shape[0], q.shape[1], k.shape[1]
    keys = (~fine).any(2).any(1).nonzero()[:, 0]
    for rows in torch.arange(lq, device="cuda").split(2000):
        p = rows[:, None] + q_pos                              # the definition, for the keys that have such values
        b = p - p % full["block"]
        seen = (keys <= b + full["block"] - 1 + full["right"]) if full["right"] >= 0 else keys[None] >= 0
        seen = (seen & ((keys >= b - full["left"]) | (keys < full["sinks"])) if full["left"] >= 0 else seen.expand(len(rows), -1)).float()
        x = odd[keys].permute(1, 0, 2)                          # [KV, keys, 128]
        nan, pos, neg = ((seen @ y.float()) > 0 for y in (x.isnan(), x == float("inf"), x == -float("inf")))   # [KV, rows, 128]
        nan, inf = nan | (pos & neg), torch.where(pos, float("inf"), -float("inf"))
        per_head = want[rows].view(-1, heads, 128).permute(1, 0, 2).float().reshape(kv, heads // kv, -1, 128)
        per_head = torch.where(nan[:, None], float("nan"), torch.where((pos | neg)[:, None], inf[:, None], per_head))
        expect = per_head.reshape(heads, -1, 128).permute(1, 0, 2).reshape(len(rows), -1)
        assert torch.equal(got[rows].float().nan_to_num(nan=12345.0), expect.nan_to_num(nan=12345.0))


ODD = ["one", "first", "last", "some", "column", "all"]


@pytest.mark.parametrize("where", ODD)
@pytest.mark.parametrize("lq, lk, heads, kv, dtype, w", [
    (200, 777, 4, 2, BF, dict(left=50, right=0, sinks=3, q_pos=500)), (600, 600, 2, 2, HF, dict(left=-1, right=0)),
    (300, 900, 7, 1, BF, dict(left=100, right=30, sinks=9, q_pos=600)), (512, 512, 2, 2, BF, dict(left=128, right=0, sinks=64, block=64)),
    (17, 300, 1, 1, BF, dict(left=-1, right=-1)),                               # every row sees every key
    (40, 9000, 4, 2, BF, dict(left=-1, right=0, q_pos=8960)),                   # keys split over a cluster
    (130, 2000, 3, 1, HF, dict(left=700, right=0, sinks=200, q_pos=1870)),
    (9000, 9000, 4, 4, BF, dict(left=5, right=0)),                              # many short items for a CTA
    (1620, 9000, 24, 24, BF, dict(left=-1, right=0, block=1620, q_pos=7380)),   # whole rounds, then a rest that is split
    (2500, 6000, 16, 2, HF, dict(left=-1, right=0, q_pos=3500)),
    # up to 16 rows for a K/V head
    (5, 777, 4, 2, BF, dict(left=50, right=0, sinks=3, q_pos=386)), (16, 400, 2, 2, HF, dict(left=-1, right=0, q_pos=384)),
    (1, 500, 6, 6, BF, dict(left=-1, right=0, q_pos=499)), (8, 20000, 4, 2, BF, dict(left=-1, right=0, q_pos=9996)),
    (3, 30000, 24, 24, HF, dict(left=9000, right=5, sinks=40, q_pos=15000)), (2, 3001, 7, 1, BF, dict(left=0, right=0, block=2, sinks=3, q_pos=1502)),
    (4, 200, 300, 100, BF, dict(left=20, right=0, q_pos=100))])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(cuda, lq, lk, heads, kv, dtype, w, where):
    g = gen(lq + lk)
    q, k, v = normal(g, lq, heads, 128, dtype=dtype), normal(g, lk, kv, 128, dtype=dtype), normal(g, lk, kv, 128, dtype=dtype)
    check_odd_values(cuda, q, k, v, where, g, **w)


@pytest.mark.parametrize("where", ["one", "first", "column"])
def test_values_that_are_not_finite_among_very_many_keys(cuda, where):
    """Items of more keys than one accumulator takes, of one sequence each: 40 rows over 70,000 and 1,000 over 300,000 keys."""
    g = gen(20)
    for lq, lk in ((40, 70000), (1000, 300000)):
        q, k, v = (normal(g, n, 1, 128, dtype=BF) for n in (lq, lk, lk))
        check_odd_values(cuda, q, k, v, where, g, left=-1, right=0, q_pos=lk - lq)
        check_odd_values(cuda, q, k, v, where, g, left=-1, right=0, q_pos=lk // 2)   # half of the keys are behind every row


def timed(fn):
    fn()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    fn()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b)


@pytest.mark.parametrize("w", [dict(left=2048, right=0, sinks=1024, block=1024), dict(left=2047, right=0, sinks=64)], ids=str)
def test_a_value_that_is_not_finite_costs_a_second_pass_and_no_more(cuda, w):
    """6,144 tokens by frames (whose rows see the same, so that nothing is done twice) and by tokens: one infinity in a key that
    stays visible, one dimension of infinities, some values, all of them.  Each item is done twice at most; the bound leaves
    room for the search, the rows written once more, and a busy machine."""
    g = gen(21)
    q, k, v = (normal(g, 6144, 24, 128, dtype=BF) for _ in range(3))
    base = min(timed(lambda: cuda.sdpa_window(q, k, v, **w)) for _ in range(5))
    for where in ("one", "first", "column", "some", "all"):
        odd = place(v, where, g)
        took = min(timed(lambda: cuda.sdpa_window(q, k, odd, **w)) for _ in range(5))
        print(f"{where}: {took:.3f} ms, {base:.3f} without")
        assert took < 16 * base                                              # (up to 6 measured)
    cuda.check()


# ------------------------------------------------------------------ probabilities far below the largest

def tail_tolerance(a, n, dtype, p_dtype, v_max, lost):
    """Half a step of P and of the output, 2^-12 for what is computed in 32 bits (all relative to a = sum p |v|); products that
    are cut to 2^-25 of an accumulator and its sum to 2^-27 of itself, over the up to 32,768 keys of one; and at the bottom of
    P's range `lost` of the largest |v| per key."""
    u = {BF: 2.0 ** -8, HF: 2.0 ** -11}
    return (u[p_dtype] + u[dtype] + 2.0 ** -12 + min(n, 32768) * (2.0 ** -25 + 2.0 ** -27)) * a + n * lost * v_max


def tail_of(n, step, loud):
    """One key of weight 1 and n - 1 of 2^-step (scale ln 2, so that a score counts in powers of two); values: the heavy key
    `loud` in dimensions 0 to 63 and nothing in the others, the rest 1 everywhere.  (q, k, v, out, sum p |v|) in 64 bits."""
    k, v = torch.zeros(n, 128, dtype=torch.float64, device="cuda"), torch.ones(n, 128, dtype=torch.float64, device="cuda")
    q = torch.zeros(128, dtype=torch.float64, device="cuda")
    heavy = 5
    k[heavy, 9], q[9] = 26.0, step / 26.0
    v[heavy, :64], v[heavy, 64:] = loud, 0.0
    q = q.to(BF).double()                                          # eight bits: exact in both types
    w = 2.0 ** (q[9] * 26.0)
    return q, k, v, (w * v[heavy] + (n - 1)) / (w + n - 1)


@pytest.mark.parametrize("n", [50220, 262144])
@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_flat_tail_far_below_the_largest_probability(cuda, n, rows, dtype):
    """2^-25.2 each: together 0.1 % of the row at 50,220 keys and 0.7 % at 262,144, and the whole result where the heavy
    key's value is zero."""
    q, k, v, want = tail_of(n, 25.2, 1.0)
    q, k, v = q.to(dtype).expand(rows, 2, 128).contiguous(), k.to(dtype)[:, None].contiguous(), v.to(dtype)[:, None].contiguous()
    got = cuda.sdpa_window(q, k, v, scale=float(np.log(2.0))).view(-1, 128).double()
    assert ((got - want).abs() <= tail_tolerance(want, n, dtype, dtype, 1.0, 2.0 ** -34 if dtype is HF else 0.0)).all(), (got - want).abs().amax(0)
    cache = cuda.kv8_cache(-(-n // 256), 256, 1)
    table = torch.arange(-(-n // 256), dtype=torch.int32, device="cuda")[None]
    cuda.kv8_append(cache, k, v, i32([0, n]), i32([0]), table, max_rows=n)
    got = cuda.kv8_sdpa(cache, q, i32([0, rows]), i32([n]), table, max_rows=rows, max_len=n, right=-1, scale=float(np.log(2.0))).view(-1, 128).double()
    cuda.check()
    assert ((got - want).abs() <= tail_tolerance(want, n, dtype, HF, 1.0, 2.0 ** -34)).all(), (got - want).abs().amax(0)


@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_loud_block_of_the_cache_does_not_drown_the_others(cuda, rows, dtype):
    """The heavy key's block has values 2^6 louder than the rest, whose 50,219 keys hold 6 % of the row at 2^-19.5 each and are the
    whole result in the dimensions where the heavy key is silent.  P carries the scale, so a key loses at most 2^-34 of
    the loud one's."""
    n = 50220
    q, k, v, want = tail_of(n, 19.5, 64.0)
    q, k, v = q.to(dtype).expand(rows, 2, 128).contiguous(), k.to(dtype)[:, None].contiguous(), v.to(dtype)[:, None].contiguous()
    cache = cuda.kv8_cache(-(-n // 64), 64, 1)
    table = torch.arange(-(-n // 64), dtype=torch.int32, device="cuda")[None]
    cuda.kv8_append(cache, k, v, i32([0, n]), i32([0]), table, max_rows=n)
    assert cache.v_scale[0, 0, 0] == 2.0 ** 6 * cache.v_scale[1, 0, 0]
    got = cuda.kv8_sdpa(cache, q, i32([0, rows]), i32([n]), table, max_rows=rows, max_len=n, right=-1, scale=float(np.log(2.0))).view(-1, 128).double()
    cuda.check()
    assert ((got - want).abs() <= tail_tolerance(want, n, dtype, HF, 64.0, 2.0 ** -34)).all(), (got - want).abs().amax(0)


# ------------------------------------------------------------------ scales of zero

@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("w", [dict(), dict(left=70, sinks=3), dict(left=0)], ids=str)
def test_a_scale_of_zero_counts_as_the_smallest_one(cuda, rows, w):
    """A new cache holds zeros, and a block of zeros quantised by its largest magnitude has a scale of zero: its tokens are
    zeros that take their share of the softmax."""
    rng, g = np.random.default_rng(rows), gen(rows)
    n = 500
    fresh = cuda.kv8_cache(9, 64, 2)
    q = normal(g, rows, 4, 128, dtype=BF)
    assert not cuda.kv8_sdpa(fresh, q, i32([0, rows]), i32([n]), i32([np.arange(9)]), max_rows=rows, max_len=n, **w).any()
    cache, table, _ = filled(cuda, rng, g, [n], 64, 2, BF, spread=False)
    for page, k_too in ((0, True), (3, False), (6, True), (7, True)):      # 7: the last page, partly filled
        for codes, scales in ((cache.v, cache.v_scale), (cache.k, cache.k_scale)):
            if scales is cache.v_scale or k_too:
                codes.view(torch.uint8)[table[0, page]] = 0
                scales[table[0, page]] = 0
    check_cache(cuda, cache, table, Model(cache), q, [0, rows], [n], **w)
    cache.v_scale.masked_fill_(cache.v_scale == 0, 2.0 ** -80)              # and so does any below it
    check_cache(cuda, cache, table, Model(cache), q, [0, rows], [n], **w)


def test_append_behind_tokens_under_a_scale_of_zero(cuda):
    g = gen(3)
    cache = cuda.kv8_cache(1, 64, 1)
    model = Model(cache)
    zero, k = torch.zeros(10, 1, 128, dtype=BF, device="cuda"), normal(g, 10, 1, 128, dtype=BF)
    for x, start in ((zero, 7), (k, 20)):                                    # tokens 0 to 6 were never written
        cuda.kv8_append(cache, x, x, i32([0, 10]), i32([start]), i32([[0]]), max_rows=10)
        model.append(x, x, [0, 10], [start], [[0]])
        model.same_as(cache)


# ------------------------------------------------------------------ how keys are split over clusters

def test_streams_that_just_miss_a_cluster_size_do_not_take_a_second_wave(cuda):
    """One token for `n` streams of 20,000 tokens and one K/V head: a count for which the next larger clusters would not all fit
    the chip at once takes no longer than some more streams in the smaller ones (a second wave: 1.3 to 1.5 times as long)."""
    n_keys, page = 20000, 256
    per, streams = -(-n_keys // page), 54
    cache = cuda.kv8_cache(streams * per, page, 1)
    cache.k.view(torch.uint8).random_(0, 120)
    cache.v.view(torch.uint8).random_(0, 120)
    cache.k_scale.fill_(2.0 ** -8)
    cache.v_scale.fill_(2.0 ** -8)
    table = torch.arange(streams * per, dtype=torch.int32, device="cuda").view(streams, per)
    q = normal(gen(1), streams, 7, 128, dtype=BF)
    side = torch.cuda.Stream()

    def took(n):
        args = q[:n], torch.arange(n + 1, dtype=torch.int32, device="cuda"), i32([n_keys] * n), table[:n]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cuda.use_stream(side)
            try:
                step = lambda: cuda.kv8_sdpa(cache, *args, max_rows=1, max_len=n_keys)  # noqa: E731
                step()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    for _ in range(20):
                        step()
                best = math.inf
                for _ in range(10):
                    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    a.record(side)
                    graph.replay()
                    b.record(side)
                    side.synchronize()
                    best = min(best, a.elapsed_time(b))
                return best
            finally:
                side.synchronize()
                cuda.use_stream(torch.cuda.default_stream())

    times = {n: took(n) for n in (16, 18, 19, 52, 54)}
    cuda.check()
    assert times[16] < 1.15 * times[19] and times[18] < 1.15 * times[19] and times[52] < 1.15 * times[54], times


# ------------------------------------------------------------------ memory of a cache

def test_memory_of_a_new_cache_waits_for_the_current_stream(cuda):
    """A cache made while the handle works on another stream than the current one: its memory comes from the handle's
    stream and is not given out again there while the caller's own work on the current stream still reads it."""
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        cuda.use_stream(side)
        cache = cuda.kv8_cache(301, 64, 3)
        side.synchronize()
        before = {t.data_ptr() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)}
        total = lambda: sum(t.float().sum() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))  # noqa: E731
        total()                                                              # (its kernels are loaded)
        torch.cuda.synchronize()
        torch.cuda._sleep(400_000_000)                                       # some 0.2 s on the current stream, then
        read, done = total(), torch.cuda.Event()
        done.record()
        del cache
        again = cuda.kv8_cache(301, 64, 3)
        now = {t.data_ptr() for t in (again.k, again.v, again.k_scale, again.v_scale)}
        assert not done.query()                                              # the caller's work is still under way
        assert not before & now
        with torch.cuda.stream(side):
            for t in (again.k.view(torch.uint8), again.v.view(torch.uint8), again.k_scale, again.v_scale):
                t.fill_(1)
        assert float(read) == 0
    finally:
        torch.cuda.synchronize()
        cuda.use_stream(torch.cuda.current_stream())


# ------------------------------------------------------------------ orders of the cache's operands

def orders(g, rows, heads, dtype):
    """Views of a [rows, heads, 128] tensor in other orders, with the same values in each."""
    x = normal(g, rows, heads, 128, dtype=dtype)
    fused = normal(g, rows, heads + 5, 128, dtype=dtype)                    # part of one projection's rows
    fused[:, 3:3 + heads] = x
    heads_first = x.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((rows, heads, 136), 9.0, dtype=dtype, device="cuda")
    wide[..., 8:] = x
    every = torch.full((2 * rows, heads, 128), 9.0, dtype=dtype, device="cuda")
    every[::2] = x
    return x, {"fused": fused[:, 3:3 + heads], "heads first": heads_first, "wide": wide[..., 8:], "every second row": every[::2]}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.uint8])
def test_append_of_rows_in_other_orders(cuda, dtype, codes):
    import h3c_b200
    rng, g = np.random.default_rng(1), gen(1)
    rows, start, page, kv = [70, 1, 130], [30, 64, 200], 128, 3
    cu = np.concatenate([[0], np.cumsum(rows)])
    table = pages_of(rng, [a + b for a, b in zip(rows, start)], page, 9)
    (k, ks), (v, vs) = orders(g, int(cu[-1]), kv, dtype), orders(g, int(cu[-1]), kv, dtype)
    pairs = [(k, v)] + [(ks[a], vs[b]) for a, b in zip(ks, reversed(vs))] + [(ks["fused"], v), (k, vs["wide"])]
    want = None
    for kk, vv in pairs:
        made = cuda.kv8_cache(9, page, kv)
        cache = h3c_b200.KvCache8(made.k.view(codes), made.v.view(codes), made.k_scale, made.v_scale)
        if want is None:
            want = Model(cache)
            want.append(k, v, cu, start, table)
        cuda.kv8_append(cache, kk, vv, i32(cu), i32(start), i32(table), max_rows=max(rows))
        cuda.check()
        want.same_as(cache)


@pytest.mark.parametrize("rows, lens, heads, kv", [([1, 3], [300, 70], 6, 2), ([40, 150], [400, 150], 6, 2), ([30, 9], [300, 90], 7, 1), ([33], [333], 4, 4)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_cache_attention_of_queries_and_outputs_in_other_orders(cuda, rows, lens, heads, kv, dtype):
    import h3c_b200
    rng, g = np.random.default_rng(2), gen(2)
    cache, table, model = filled(cuda, rng, g, lens, 64, kv, dtype, spread=False)
    cu = np.concatenate([[0], np.cumsum(rows)])
    n, w = int(cu[-1]), dict(left=50, sinks=2)
    q, others = orders(g, n, heads, dtype)
    want = check_cache(cuda, cache, table, model, q, cu, lens, **w)
    args = dict(max_rows=max(rows), max_len=max(lens), **w)
    codes = h3c_b200.KvCache8(cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)
    for c, qq in [(cache, x) for x in others.values()] + [(codes, q)]:
        assert torch.equal(cuda.kv8_sdpa(c, qq, i32(cu), i32(lens), i32(table), **args), want)
    for first, width in ((0, heads * 128 + 64), (8, heads * 128 + 24), (16, heads * 128 + 16)):   # 16- and 32-byte stores
        room = torch.full((n + 3, width), 3.0, dtype=dtype, device="cuda")
        out = room[1:n + 1, first:first + heads * 128]
        got = cuda.kv8_sdpa(cache, q, i32(cu), i32(lens), i32(table), out=out, **args)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
        room[1:n + 1, first:first + heads * 128] = 3.0
        assert (room == 3).all()


# ------------------------------------------------------------------ values that are not finite, in the calls of a program

@pytest.mark.parametrize("where", ["one", "first", "some"])
@pytest.mark.parametrize("lq, w", [(3, dict(left=60, right=0, sinks=6, q_pos=198)), (150, dict(left=90, right=4, sinks=6, q_pos=100)),
                                   (60, dict(left=3, right=0, q_pos=350)), (9, dict(left=3, right=0, sinks=1, q_pos=395))])   # rows behind the keys
def test_values_that_are_not_finite_in_views_and_outputs_of_other_orders(cuda, lq, w, where):
    g = gen(lq)
    fused = normal(g, 400, 6 + 2 + 2, 128, dtype=BF)
    q, k = fused[:lq, :6], fused[:, 6:8]
    fused[:, 8:] = place(fused[:, 8:], where, g)
    v = fused[:, 8:]
    check_odd_values(cuda, q, k, torch.where(torch.isfinite(v), v, 1.0), where, g, **w)
    want = cuda.sdpa_window(q.contiguous(), k.contiguous(), v.contiguous(), **w)
    room = torch.full((lq, 6 * 128 + 24), 3.0, dtype=BF, device="cuda")
    out = cuda.sdpa_window(q, k, v, out=room[:, 8:8 + 768], **w)
    assert torch.equal(out.float().nan_to_num(nan=12345.0), want.float().nan_to_num(nan=12345.0))
    assert (room[:, :8] == 3).all() and (room[:, 776:] == 3).all()


@pytest.mark.parametrize("lq, lk", [(2, 3000), (300, 700), (40, 9000)])
def test_a_captured_call_follows_values_that_are_not_finite(cuda, lq, lk):
    """Whether there is a second pass is decided on the device: a graph captured over ordinary values, replayed over others."""
    g = gen(lq)
    q, k, v = normal(g, lq, 4, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF), normal(g, lk, 2, 128, dtype=BF)
    fine, w = v.clone(), dict(left=-1, right=0, q_pos=lk - lq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(side):
            cuda.use_stream(side)
            cuda.sdpa_window(q, k, v, **w)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = cuda.sdpa_window(q, k, v, **w)
            for where in ("none", "last", "some", "none", "all", "none"):
                v.copy_(place(fine, where, g))
                graph.replay()
                got = out.clone()
                want = cuda.sdpa_window(q, k, v, **w)
                assert torch.equal(got.float().nan_to_num(nan=12345.0), want.float().nan_to_num(nan=12345.0))
                assert bool(torch.isfinite(got).all()) == (where == "none")
            side.synchronize()
    finally:
        torch.cuda.synchronize()
        cuda.use_stream(torch.cuda.current_stream())
    cuda.check()


@pytest.mark.parametrize("rows", [2, 70])
def test_outputs_by_head_through_the_c_entry_points(cuda, rows):
    """[heads, rows, 128] outputs, which the Python entry points do not offer."""
    import h3c_b200
    from h3c_b200 import lib as l
    rng, g = np.random.default_rng(5), gen(5)
    cache, table, model = filled(cuda, rng, g, [300], 64, 2, BF, spread=False)
    q, cu, lens, pages = normal(g, rows, 4, 128, dtype=BF), i32([0, rows]), i32([300]), i32(table)
    want = check_cache(cuda, cache, table, model, q, [0, rows], [300], left=40)
    out = torch.full((4, rows + 1, 128), 3.0, dtype=BF, device="cuda")
    h3c_b200.call("h3b_kv8_sdpa_dev", cuda.h, cache.packed, l.KV8_SDPA_ARGS.pack(
        q.data_ptr(), out.data_ptr(), cu.data_ptr(), lens.data_ptr(), pages.data_ptr(), 512, 128, 128, (rows + 1) * 128, rows, 4, table.shape[1], 1,
        rows, 300, 40, 0, 0, 1, 128 ** -0.5, l.BF16))
    cuda.check()
    assert torch.equal(out[:, :rows].transpose(0, 1).reshape(rows, -1), want) and (out[:, rows] == 3).all()
    k, v = normal(g, 200, 2, 128, dtype=BF), normal(g, 200, 2, 128, dtype=BF)
    v[150, 0, 3] = float("inf")                                              # seen by some rows: a second pass writes there too
    want = cuda.sdpa_window(q, k, v, left=40, right=0, q_pos=149)
    h3c_b200.call("h3b_sdpa_window_dev", cuda.h, l.SDPA_WINDOW_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 512, 128, 256, 128, 256, 128, 128, (rows + 1) * 128, rows, 200, 4, 2, 128, 149, 40, 0,
        0, 1, 128 ** -0.5, l.BF16))
    cuda.check()
    assert torch.equal(out[:, :rows].transpose(0, 1).reshape(rows, -1).float().nan_to_num(nan=9.5), want.float().nan_to_num(nan=9.5))
    assert not torch.isfinite(want).all() and (out[:, rows] == 3).all()


@pytest.mark.parametrize("w", [dict(left=-1, right=0), dict(left=200, right=0, sinks=9), dict(left=-1, right=-1)], ids=str)
@pytest.mark.parametrize("lq, heads, kv", [(8, 3, 3), (9, 3, 3), (16, 3, 3), (17, 3, 3), (2, 8, 2), (3, 8, 2), (4, 8, 2)])
def test_window_on_both_sides_of_the_choice_of_kernels(cuda, lq, heads, kv, w):
    for lk in (17, 64, 255, 256, 257, 600):
        g = gen(lk)
        q, k, v = normal(g, lq, heads, 128, dtype=HF), normal(g, lk, kv, 128, dtype=HF), normal(g, lk, kv, 128, dtype=HF)
        check_window(cuda, q, k, v, q_pos=max(0, lk - lq), **w)


@pytest.mark.parametrize("lq, lk, w", [(1, 700, dict()), (9, 700, dict(left=300, right=0, q_pos=600)), (300, 700, dict(left=300, right=0, q_pos=400)),
                                       (40, 9000, dict(left=-1, right=0, q_pos=8960))])   # keys split over a cluster
def test_means_of_the_largest_f16_values_stay_finite(cuda, lq, lk, w):
    """Values clamped to the type's range, as programs in f16 do: a mean of 65504 is 65504, not infinity.  One key in 37 has the
    largest score, the others one whose probability next to it, 1/2 + 2^-12 + 2^-15, is rounded up by 2^-12 - 2^-15: the mean
    comes out high by 2^-11.3 of itself, and from 2^-12 on it is rounded to infinity."""
    g = gen(lq)
    q, k = torch.zeros(lq, 4, 128, dtype=HF, device="cuda"), torch.zeros(lk, 2, 128, dtype=HF, device="cuda")
    q[..., 7] = 1
    k[::37, :, 7] = 1
    v = torch.full((lk, 2, 128), 65504.0, dtype=HF, device="cuda")
    v[:, 1] = -65504.0
    w = w | dict(scale=-math.log(0.5 + 2.0 ** -12 + 2.0 ** -15))
    got = cuda.sdpa_window(q, k, v, **w)
    want = torch.where(torch.arange(512, device="cuda") < 256, 65504.0, -65504.0).double().expand(lq, -1)
    close(got, want, want.abs(), 65504.0, HF)
    v[lk - 1, 0, 3] = float("inf")                                           # a value that is infinite stays so
    got = cuda.sdpa_window(q, k, v, **w).view(lq, 4, 128)
    sees = mask(np.arange(lq) + w.get("q_pos", 0), lk, w.get("left", -1), w.get("right", -1), 0, 1)[:, lk - 1]
    assert (got[sees][:, :2, 3] == float("inf")).all() and torch.isfinite(got[~sees]).all() and int(torch.isinf(got).sum()) == 2 * int(sees.sum())
