"""Windowed attention and the 8-bit cache at the edges of their contracts: pages that no row needs, values that are not
finite, probabilities far below the largest, scales of zero, orders of the cache's operands.  Definitions in 64 bits and
tolerances as in test_gpu_attn_window.py unless a test derives its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_attn_window import BF, HF, check_cache, cuda, filled, gen, i32, mask, normal  # noqa: E402, F401


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
