"""Windowed attention with sinks, and attention over a paged 8-bit key/value cache with its append: sizes, plain forms
and 64-bit definitions.

    h3c_b200.Cuda.sdpa_window   16-bit Q, K, V of one sequence; sliding window per token or per frame, first keys stay visible
    h3c_b200.Cuda.kv8_append    K / V rows of many sequences into the pages of an E4M3 cache, one scale per 64 tokens and head
    h3c_b200.Cuda.kv8_sdpa      queries of many sequences over that cache, with the same windows

A query at position p belongs to the block (frame) that starts at b = p - p % block.  It sees key j if
j <= b + block - 1 + right and (j >= b - left or j < sinks); a negative left or right does not bound that side.
A row that sees nothing is zero.

The cache holds codes [pages, kv_heads, page_tokens, 128] (E4M3) and scales [pages, kv_heads, page_tokens / 64] (f32,
powers of two): value = code * scale.  The scale of 64 tokens of a head is the smallest power of two 2^e, e >= -64, with
absmax <= 448 * 2^e; tokens put behind others of the same 64 may raise it, and the codes that are there are then
rounded again under the new scale.
"""
import math

import numpy as np
import torch

own = False

D = 128          # head size of every attention operator here
BLOCK = 64       # tokens that share a scale
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of a stream over its last 4096 keys and 64 first ones
        dict(name="window_token", op="window", dtype="bf16", lq=1, lk=16384, heads=24, kv_heads=24, q_pos=16383, left=4095, right=0, sinks=64, block=1, fused=0),
        # the 6,144-token step (6 frames of 32 x 32): each frame sees itself, the two before it and the first one
        dict(name="window_frames_6144", op="window", dtype="bf16", lq=6144, lk=6144, heads=24, kv_heads=24, q_pos=0, left=2048, right=0, sinks=1024, block=1024, fused=0),
        # the 50,220-token video (31 frames of 30 x 54): eight frames back and the first one
        dict(name="window_video_50220", op="window", dtype="bf16", lq=50220, lk=50220, heads=24, kv_heads=24, q_pos=0, left=12960, right=0, sinks=1620, block=1620, fused=0),
        # shared K/V heads, views of one fused projection, odd sizes, a window to both sides
        dict(name="window_shared_heads", op="window", dtype="f16", lq=1531, lk=7919, heads=56, kv_heads=8, q_pos=6200, left=1000, right=77, sinks=5, block=1, fused=1),
        # one new token for each of 64 streams
        dict(name="append_tokens", op="append", dtype="bf16", seqs=64, max_rows=1, max_start=2000, kv_heads=8, page=64),
        # a finished chunk of video goes into the cache behind what is there
        dict(name="append_chunk", op="append", dtype="bf16", seqs=1, max_rows=6144, max_start=4860, kv_heads=24, page=256),
        # prompts and drafts of many requests at once
        dict(name="append_ragged", op="append", dtype="f16", seqs=37, max_rows=301, max_start=1500, kv_heads=5, page=128),
        # one token, one short stream: latency
        dict(name="cache_token", op="cache", dtype="bf16", seqs=1, max_rows=1, max_len=2313, ragged=0, heads=24, kv_heads=24, page=64, left=-1, right=0, sinks=0, block=1),
        # one token for each of 64 streams of up to 16,384 tokens, seven query heads to a K/V head
        dict(name="cache_tokens", op="cache", dtype="bf16", seqs=64, max_rows=1, max_len=16384, ragged=1, heads=56, kv_heads=8, page=64, left=-1, right=0, sinks=0, block=1),
        # a few drafted tokens for each of 12 streams, window and sinks
        dict(name="cache_drafts", op="cache", dtype="f16", seqs=12, max_rows=5, max_len=30011, ragged=1, heads=24, kv_heads=8, page=128, left=8191, right=0, sinks=16, block=1),
        # the next frame of the 50,220-token video over all the frames before it and itself
        dict(name="cache_frame", op="cache", dtype="bf16", seqs=1, max_rows=1620, max_len=50220, ragged=0, heads=24, kv_heads=24, page=256, left=-1, right=0, sinks=0, block=1620),
        # prompts and tokens in one call, window and sinks
        dict(name="cache_mixed", op="cache", dtype="f16", seqs=9, max_rows=701, max_len=9001, ragged=1, heads=24, kv_heads=6, page=64, left=2047, right=0, sinks=64, block=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16"])
    kind = rng.choice(["window", "window", "append", "cache", "cache", "cache"])
    if kind == "append":
        kv, seqs = rng.choice([1, 2, 5, 8, 12, 24]), _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, 6144 * 24 // (kv * seqs)) if seqs > 1 else 6144)
        return dict(op="append", dtype=dtype, seqs=seqs, max_rows=min(rows, 6144), max_start=_log(rng, 1, max(2, min(5000, 300000 // (kv * seqs)))), kv_heads=kv, page=rng.choice([64, 128, 192, 256]))
    kv = rng.choice([1, 2, 4, 6, 8, 24])
    heads = kv * (1 if kv == 24 else rng.choice([1, 2, 3, 4, 7]))
    block = rng.choice([1, 1, 1, rng.randint(2, 1620)])
    left = rng.choice([-1, _log(rng, 1, 8192)])
    right = rng.choice([0, 0, 0, _log(rng, 1, 500), -1])
    sinks = rng.choice([0, _log(rng, 1, 600)])
    if kind == "window":
        lk = _log(rng, 1, 20000)
        lq = rng.choice([1, _log(rng, 1, 64), min(lk, _log(rng, 1, 8000))])
        q_pos = rng.choice([0, max(0, lk - lq), rng.randint(0, lk)])
        return dict(op="window", dtype=dtype, lq=lq, lk=lk, heads=heads, kv_heads=kv, q_pos=q_pos, left=left, right=right, sinks=sinks, block=block, fused=rng.randint(0, 1))
    seqs = _log(rng, 1, 48)
    most = max(64, min(40000, 6000000 // (kv * seqs)))
    max_len = _log(rng, 40, most)
    rows = rng.choice([1, 1, _log(rng, 1, 16), _log(rng, 16, 1000)])
    rows = max(1, min(rows, max_len, 2000000000 // (max_len * heads * seqs)))
    return dict(op="cache", dtype=dtype, seqs=seqs, max_rows=rows, max_len=max_len, ragged=rng.randint(0, 1), heads=heads, kv_heads=kv, page=rng.choice([64, 128, 192, 256]), left=left, right=right, sinks=sinks, block=block)


# ---- which sequence has how many rows and tokens (host numbers, the same for every seed)

def _extents(case):
    """rows of each sequence in this call, and the tokens its cache holds before it (append) or with it (cache)."""
    r = np.random.RandomState(sum((i + 1) * v for i, v in enumerate(case[k] for k in sorted(case) if isinstance(case[k], int))) % (1 << 31))
    n, most = case["seqs"], case["max_rows"]
    if case["op"] == "append":
        rows = r.randint(max(1, most // 4), most + 1, n) if n > 1 else np.array([most])
        start = r.randint(0, case["max_start"] + 1, n) if n > 1 else np.array([case["max_start"]])
        return rows.astype(np.int64), start.astype(np.int64)
    if not case["ragged"]:
        return np.full(n, most), np.full(n, case["max_len"])
    rows = r.randint(1, most + 1, n)
    rows[0] = most
    low = min(case["max_len"], max(most, case["max_len"] // 16))
    lens = r.randint(low, case["max_len"] + 1, n)
    lens[n // 2] = case["max_len"]
    return rows.astype(np.int64), lens.astype(np.int64)


def _bounds(p, n, case):
    """(lo, hi, sinks) of queries at positions p over n keys: visible are j <= hi with j >= lo or j < sinks."""
    b = p - p % case["block"]
    hi = (b + case["block"] - 1 + case["right"]) if case["right"] >= 0 else (p * 0 + n - 1)
    lo = (b - case["left"]) if case["left"] >= 0 else p * 0
    if isinstance(p, np.ndarray):
        hi, lo = np.minimum(hi, n - 1), np.maximum(lo, 0)
        return lo, hi, np.minimum(case["sinks"], hi + 1)
    hi, lo = torch.minimum(hi, torch.as_tensor(n - 1, device=p.device)), lo.clamp(min=0)
    return lo, hi, hi * 0 + case["sinks"]


def _pairs(p, n, case):
    """visible (query, key) pairs, and keys that at least one query sees."""
    lo, hi, s = _bounds(p, n, case)
    some = hi >= 0
    pairs = np.where(some, np.maximum(hi - np.maximum(lo, s) + 1, 0) + np.maximum(np.minimum(s, hi + 1), 0), 0).sum()
    if not some.any():
        return 0, 0
    lo, hi, s = int(lo[some].min()), int(hi[some].max()), int(s[some].max())
    return int(pairs), max(0, hi + 1 - max(lo, s)) + s


def work(case):
    if case["op"] == "window":
        pairs, keys = _pairs(np.arange(case["lq"], dtype=np.int64) + case["q_pos"], case["lk"], case)
        return {"bytes": 2 * D * (2 * case["lq"] * case["heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * D * case["heads"] * pairs}
    rows, lens = _extents(case)
    if case["op"] == "append":  # rows in 16 bits in, codes and scales out
        return {"bytes": int(rows.sum()) * case["kv_heads"] * 2 * (2 * D + D) + int((rows // BLOCK + 1).sum()) * case["kv_heads"] * 8, "flops": 0}
    pairs = keys = 0
    for nq, n in zip(rows, lens):
        a, b = _pairs(n - nq + np.arange(nq, dtype=np.int64), n, case)
        pairs, keys = pairs + a, keys + b
    return {"bytes": keys * case["kv_heads"] * 2 * (D + 4 / BLOCK) + int(rows.sum()) * case["heads"] * 4 * D, "flops": 4 * D * case["heads"] * pairs}


# ---- inputs

def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _channels(gen, heads):
    """Key channels differ in size as they do behind a learned norm weight: a few are several times the others."""
    c = torch.exp(0.3 * torch.randn(heads, D, generator=gen, device="cuda"))
    return torch.where(torch.rand(heads, D, generator=gen, device="cuda") < 0.02, 4 * c, c) * 0.8


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, kv = DTYPES[case["dtype"]], case["kv_heads"]
    s = {"case": case}
    if case["op"] == "window":
        h, lq, lk = case["heads"], case["lq"], case["lk"]
        if case["fused"]:  # K and V are parts of one projection's rows
            both = _normal(gen, lk, 2 * kv, D, dtype=dt)
            s["q"], s["k"], s["v"] = _normal(gen, lq, h, D, dtype=dt), both[:, :kv], both[:, kv:]
        else:
            s["q"], s["k"], s["v"] = (_normal(gen, n, m, D, dtype=dt) for n, m in ((lq, h), (lk, kv), (lk, kv)))
        return s
    rows, tokens = _extents(case)
    page, n = case["page"], case["seqs"]
    need = -(-(tokens + (rows if case["op"] == "append" else 0)) // page)
    total, width = int(need.sum()), int(need.max())
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    at = np.cumsum(need) - need
    idx = np.minimum(at[:, None] + np.arange(width)[None], total - 1)
    table = order[torch.from_numpy(idx).cuda()]
    s["table"] = torch.where(torch.from_numpy(np.arange(width)[None] < need[:, None]).cuda(), table, torch.tensor(-1, dtype=torch.int32, device="cuda")).contiguous()
    s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()
    s["tokens"] = torch.from_numpy(tokens.astype(np.int32)).cuda()
    k, v = (torch.empty(total, kv, page, D, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.empty(total, kv, page // BLOCK, device="cuda") for _ in range(2))
    chan = _channels(gen, kv)
    for codes, scales, c in ((k, ks, chan[:, None]), (v, vs, 1.0)):
        for i in range(0, total, 4096):
            x = torch.randn(len(codes[i:i + 4096]), kv, page, D, generator=gen, device="cuda") * c
            blocks = x.view(-1, kv, page // BLOCK, BLOCK * D)
            m, e = torch.frexp(blocks.abs().amax(-1))
            sc = torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875))
            scales[i:i + 4096] = sc
            codes[i:i + 4096] = (blocks / sc[..., None]).view(x.shape).to(torch.float8_e4m3fn)
    s |= {"k_codes": k, "v_codes": v, "k_scale": ks, "v_scale": vs}
    total_rows = int(rows.sum())
    if case["op"] == "append":
        s["k"] = (torch.randn(total_rows, kv, D, generator=gen, device="cuda") * chan).to(dt)
        s["v"] = _normal(gen, total_rows, kv, D, dtype=dt)
    else:
        s["q"] = _normal(gen, total_rows, case["heads"], D, dtype=dt)
    return s


# ---- one pass

_kept = {}


def _cuda():
    """The current device's handle, on the current stream (whose number is cheap to look up)."""
    device = torch.cuda.current_device()
    raw, kept = torch._C._cuda_getCurrentRawStream(device), _kept.get(device)
    if kept is None or kept[0] != raw:
        import h3c_b200
        cuda = kept[1] if kept else h3c_b200.Cuda(device)
        cuda.use_stream(torch.cuda.current_stream())
        kept = _kept[device] = raw, cuda, h3c_b200.KvCache8
    return kept[1:]


def run(s):
    c = s["case"]
    if own:
        cuda, cache_of = _cuda()
        if c["op"] == "window":
            return cuda.sdpa_window(s["q"], s["k"], s["v"], left=c["left"], right=c["right"], sinks=c["sinks"], block=c["block"], q_pos=c["q_pos"])
        cache = cache_of(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        if c["op"] == "cache":
            return cuda.kv8_sdpa(cache, s["q"], s["cu"], s["tokens"], s["table"], max_rows=c["max_rows"], max_len=c["max_len"], left=c["left"], right=c["right"], sinks=c["sinks"], block=c["block"])
        cuda.kv8_append(cache, s["k"], s["v"], s["cu"], s["tokens"], s["table"], max_rows=c["max_rows"])
        return {"k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "window":
        return _plain_window(s, c)
    return _plain_cache(s, c) if c["op"] == "cache" else _plain_append(s, c)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end

def _softmax_pv(scores, seen, v):
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _plain_window(s, c):
    """Queries in pieces of a frame (or 1024): each piece takes the keys up to its last visible one, from its first."""
    g, kv, n = c["heads"] // c["kv_heads"], c["kv_heads"], c["lk"]
    k, v = s["k"].float().permute(1, 2, 0), s["v"].float().permute(1, 0, 2)
    out = torch.empty(c["lq"], c["heads"], D, device="cuda", dtype=s["q"].dtype)
    step = c["block"] if c["block"] > 256 else 1024
    for i in range(0, c["lq"], step):
        q = s["q"][i:i + step].float()
        at = np.arange(len(q), dtype=np.int64) + i + c["q_pos"]
        lo, hi, first = _bounds(at, n, c)
        lo, hi, first = int(lo.min()), int(hi.max()) + 1, min(int(first.max()), n)
        first = max(0, min(first, lo, hi))
        pos = torch.cat([torch.arange(first, device="cuda"), torch.arange(min(lo, hi), hi, device="cuda")])
        kk, vv = torch.cat([k[..., :first], k[..., min(lo, hi):hi]], -1), torch.cat([v[:, :first], v[:, min(lo, hi):hi]], 1)
        if not len(pos):
            out[i:i + step] = 0
            continue
        a, b, f = _bounds(torch.from_numpy(at).cuda(), n, c)
        seen = (pos <= b[:, None]) & ((pos >= a[:, None]) | (pos < f[:, None]))
        q = (q * D ** -0.5).view(len(q), kv, g, D).permute(1, 2, 0, 3).reshape(kv, g * len(at), D)
        o = _softmax_pv((q @ kk).view(kv, g, len(at), -1), seen, vv[:, None])
        out[i:i + step] = o.permute(2, 0, 1, 3).reshape(len(at), c["heads"], D).to(out.dtype)
    return out.view(c["lq"], c["heads"] * D)


def _plain_cache(s, c):
    """All sequences padded to the longest: gathered pages times scales, scores, softmax, product."""
    n, kv, g, page = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    table = s["table"].clamp(min=0).long()
    lens, cu = s["tokens"].long(), s["cu"].long()

    def values(codes, scales):  # [seqs, kv, tokens, D]
        x = codes[table].float().view(n, -1, kv, page // BLOCK, BLOCK, D) * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(n, kv, -1, D)

    k, v = values(s["k_codes"], s["k_scale"]), values(s["v_codes"], s["v_scale"])
    row = torch.arange(c["max_rows"], device="cuda")
    count = cu[1:] - cu[:-1]
    real = row < count[:, None]
    at = torch.where(real, cu[:-1, None] + row, 0)
    q = s["q"].float()[at].view(n, -1, kv, g, D).permute(0, 2, 3, 1, 4) * D ** -0.5
    lo, hi, first = _bounds((lens - count)[:, None] + row, lens[:, None], c)
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= hi[..., None]) & ((key >= lo[..., None]) | (key < first[..., None]))
    scores = (q.reshape(n, kv, -1, D) @ k.transpose(2, 3)).view(n, kv, g, c["max_rows"], -1)
    o = _softmax_pv(scores, seen[:, None, None], v[:, :, None])
    return o.permute(0, 3, 1, 2, 4)[real].to(s["q"].dtype).reshape(len(s["q"]), c["heads"] * D)


def _plain_append(s, c):
    """Blocks by index: the largest value of each touched block, its scale, the kept tokens again, the new ones."""
    kv, page = c["kv_heads"], c["page"]
    per = page // BLOCK
    cu, start, table = s["cu"].long(), s["tokens"].long(), s["table"].long()
    row = torch.arange(len(s["k"]), device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = start[seq] + row - cu[seq]
    head = torch.arange(kv, device="cuda")
    token = (table[seq, pos // page][:, None] * kv + head) * page + (pos % page)[:, None]      # [rows, kv]
    first = (table[torch.arange(len(start), device="cuda"), start // page][:, None] * kv + head) * per + (start % page // BLOCK)[:, None]
    kept = (start % BLOCK)[:, None] + torch.zeros_like(first)                                    # tokens that stay in the first block
    grown = cu[1:] > cu[:-1]
    first, kept = first[grown].view(-1), kept[grown].view(-1)
    for x, codes, scales in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"], s["v_scale"])):
        x = x.float()
        flat_codes, flat_scales = codes.view(-1, BLOCK, D), scales.view(-1)
        top = torch.zeros(flat_scales.shape, device="cuda").index_reduce_(0, (token // BLOCK).view(-1), x.abs().amax(-1).view(-1), "amax")
        m, e = torch.frexp(top)
        e = torch.where(top > 0, e - 9 + (m > 0.875), -64).clamp(min=-64)
        new = torch.ldexp(torch.ones_like(top), e)
        before = flat_scales[first]
        new[first] = torch.where(kept > 0, torch.maximum(new[first], before), new[first])
        old = flat_codes[first].float()
        again = (old * (before / new[first])[:, None, None]).to(torch.float8_e4m3fn).float()
        stays = torch.arange(BLOCK, device="cuda") < kept[:, None]
        flat_codes[first] = torch.where(stays[..., None], again, old).to(torch.float8_e4m3fn)
        touched = (token // BLOCK).view(-1)
        flat_scales[touched] = new[touched]
        codes.view(-1, D)[token.view(-1)] = (x.view(-1, D) / new[touched][:, None]).to(torch.float8_e4m3fn)
    return {"k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---- the definitions in 64 bits, sequence by sequence

def _exact_rows(q, k, v, pos, n, case):
    """q [rows, heads, D], k and v [n, kv, D] in 64 bits -> [rows, heads * D]."""
    g = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i in range(0, len(q), 540):
        p = pos[i:i + 540]
        frame = p // case["block"] * case["block"]
        last = torch.full_like(p, n - 1) if case["right"] < 0 else (frame + case["block"] - 1 + case["right"]).clamp(max=n - 1)
        begin = torch.zeros_like(p) if case["left"] < 0 else frame - case["left"]
        end = max(0, int(last.max()) + 1)
        skip = max(0, int(begin.min()))
        keys = torch.arange(end, device="cuda")
        keys = keys[(keys < case["sinks"]) | (keys >= skip)]
        if not len(keys):
            continue
        mask = (keys <= last[:, None]) & ((keys >= begin[:, None]) | (keys < case["sinks"]))
        for h in range(case["heads"]):
            z = (q[i:i + 540, h] @ k[keys, h // g].T) / math.sqrt(D)
            z = z.masked_fill(~mask, -math.inf)
            z = z - z.amax(1, keepdim=True).nan_to_num(neginf=0.0)
            w = z.exp()
            t = w.sum(1, keepdim=True)
            out[i:i + 540, h] = w @ v[keys, h // g] / torch.where(t > 0, t, 1.0)
    return out.reshape(len(q), -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "window":
        pos = torch.arange(case["lq"], device="cuda") + case["q_pos"]
        return _exact_rows(s["q"].double(), s["k"].double(), s["v"].double(), pos, case["lk"], case)
    rows, tokens = _extents(case)
    cu, page, kv = np.concatenate([[0], np.cumsum(rows)]), case["page"], case["kv_heads"]
    if case["op"] == "cache":
        out = []
        for i, (nq, n) in enumerate(zip(rows.tolist(), tokens.tolist())):
            t = s["table"][i, : -(-n // page)].long()
            k, v = ((codes[t].double() * scale[t].double().repeat_interleave(BLOCK, -1)[..., None]).transpose(1, 2).reshape(-1, kv, D)[:n]
                    for codes, scale in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
            out.append(_exact_rows(s["q"][cu[i]:cu[i + 1]].double(), k, v, torch.arange(n - nq, n, device="cuda"), n, case))
        return torch.cat(out)
    got = {"k": s["k_codes"].double(), "v": s["v_codes"].double(), "k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double()}
    for name in ("k", "v"):
        for i, (nr, at) in enumerate(zip(rows.tolist(), tokens.tolist())):
            x = s[name][cu[i]:cu[i + 1]].double()
            done = 0
            while done < nr:  # one 64-token block of the sequence after the other
                p = at + done
                take = min(BLOCK - p % BLOCK, nr - done)
                pg, b, o = int(s["table"][i, p // page]), p % page // BLOCK, p % BLOCK
                piece = x[done:done + take].transpose(0, 1)  # [kv, take, D]
                part, e = torch.frexp(piece.abs().amax((1, 2)).clamp(min=2.0 ** -100) / 448)
                scale = torch.exp2(torch.where(part == 0.5, e - 1, e).clamp(min=-64).double())
                codes = got[name][pg, :, b * BLOCK:(b + 1) * BLOCK]
                if o:
                    before = got[name + "_scale"][pg, :, b]
                    scale = torch.maximum(scale, before)
                    codes[:, :o] *= (before / scale)[:, None, None]
                codes[:, o:o + take] = piece / scale[:, None, None]
                got[name + "_scale"][pg, :, b] = scale
                done += take
    return got
