"""Windowed attention and the 8-bit cache on the CPU: the window arithmetic that kernels and launchers share, walked
through its host entry point against the definition, and the refusals of the entry points (every argument is checked
before the handle is used, so a zeroed block of memory stands in for one)."""
import ctypes as C
import itertools
from pathlib import Path

import numpy as np
import pytest

import h3c_b200
from h3c_b200 import lib as l

ROOT = Path(__file__).resolve().parent.parent


def sees(j, p, n, left, right, sinks, block):
    b = p - p % block
    return (j < n and (right < 0 or j <= b + block - 1 + right)) and (left < 0 or j >= b - left or j < sinks)


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 200])
@pytest.mark.parametrize("unit", [64, 128])
def test_tiles_hold_every_visible_key_once_and_no_idle_tile_beside_gaps(n, unit):
    lib = h3c_b200.load()
    out = [C.c_int() for _ in range(3)]
    for pos0, rows, left, right, sinks, block in itertools.product([0, 1, 100, 190], [1, 2, 70], [-1, 0, 1, 64, 90], [-1, 0, 3, 70],
                                                                   [0, 1, 64, 100, 500], [1, 7, 64, 1000]):
        assert lib.h3b_window_tiles(n, pos0, rows, left, right, sinks, block, unit, *(C.byref(o) for o in out)) == 1
        sink, start, count = (o.value for o in out)
        tiles = [i if i < sink else start + i - sink for i in range(count)]
        assert len(set(tiles)) == count and tiles == sorted(tiles)
        want = {j // unit for j in range(n) for p in range(pos0, pos0 + rows) if sees(j, p, n, left, right, sinks, block)}
        case = (n, pos0, rows, left, right, sinks, block)
        assert want <= set(tiles), case
        assert all(t * unit < max(n, 1) for t in tiles), case
        # a tile without any visible key lies only where the ranges of the first and the last row leave no gap
        idle = set(tiles) - want
        assert all(min(want, default=t) <= t <= max(want, default=t) or left >= 0 or right >= 0 for t in idle), case


def test_tiles_of_extreme_numbers():
    lib = h3c_b200.load()
    a, b, c = C.c_int(), C.c_int(), C.c_int()
    big = (1 << 29) - 1
    assert lib.h3b_window_tiles(big, big - 5, 5, 1 << 62, 1 << 62, 1 << 62, 1 << 62, 64, C.byref(a), C.byref(b), C.byref(c)) == 1
    assert c.value == (big + 63) // 64 and a.value == c.value
    assert lib.h3b_window_tiles(big, big - 5, 5, 100, 0, 0, 1, 64, C.byref(a), C.byref(b), C.byref(c)) == 1
    assert a.value == 0 and b.value == (big - 105) // 64 and b.value + c.value == (big + 63) // 64
    for bad in ((10, -1, 1, 0, 0, 0, 1, 64), (10, 0, 0, 0, 0, 0, 1, 64), (10, 0, 1, 0, 0, -1, 1, 64), (10, 0, 1, 0, 0, 0, 0, 64),
                (1 << 29, 0, 1, 0, 0, 0, 1, 64), (10, 1 << 29, 1, 0, 0, 0, 1, 64), (10, 0, 1, 0, 0, 0, 1, 0)):
        assert lib.h3b_window_tiles(*bad, C.byref(a), C.byref(b), C.byref(c)) == 0


# ------------------------------------------------------------------ refusals

A = 1 << 20   # an aligned address that is never read


def refused(name, *args):
    err = C.create_string_buffer(512)
    assert getattr(h3c_b200.load(), name)(*args, err, 512) == 0
    return err.value.decode()


def block(layout, fields):
    return layout.pack(*(0 if v is None else v for v in fields.values()))


def fake_handle():
    return C.cast(C.create_string_buffer(8192), C.c_void_p)


WINDOW = dict(q=A, k=A, v=A, out=A, qr=1024, qh=128, kr=1024, kh=128, vr=1024, vh=128, orow=1024, oh=128, lq=4, lk=9, heads=8, kv=8,
              hd=128, q_pos=0, left=-1, right=0, sinks=0, block=1, scale=0.1, dtype=l.BF16)


def window(**change):
    return block(l.SDPA_WINDOW_ARGS, WINDOW | change)


@pytest.mark.parametrize("change, says", [
    (dict(dtype=l.F32), "bf16 or f16"), (dict(dtype=9), "bf16 or f16"), (dict(hd=64), "head_dim 64"), (dict(heads=0), "heads over"),
    (dict(kv=3), "8 heads over 3"), (dict(kv=0), "heads over"), (dict(heads=65536), "heads over"),
    (dict(heads=258, kv=2), "more than 128"), (dict(sinks=-1), "sinks"), (dict(block=0), "block"), (dict(block=-4), "block"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "NULL tensor"), (dict(k=None), "NULL tensor"), (dict(v=None), "NULL tensor"), (dict(out=None), "NULL tensor"),
    (dict(q=A + 8), "16-byte"), (dict(k=A + 2), "16-byte"), (dict(v=A + 4), "16-byte"), (dict(out=A + 8), "16-byte"),
    (dict(qr=1028), "multiples of 8"), (dict(kh=129), "multiples of 8"), (dict(vr=4), "multiples of 8"), (dict(oh=2), "multiples of 8"),
    (dict(kr=0), "strides must be given"), (dict(qh=0), "strides must be given"), (dict(vr=1 << 40), "stride too large"),
    (dict(oh=64), "overlap"), (dict(orow=120), "overlap"), (dict(lq=1 << 28, heads=128, kv=8), "too large"),
    (dict(q_pos=-1), "q_pos"), (dict(q_pos=1 << 29), "q_pos"), (dict(lq=1 << 29), "too large"), (dict(lk=1 << 29), "too large")])
def test_window_refusals(change, says):
    assert says in refused("h3b_sdpa_window_dev", fake_handle(), window(**change))


def test_null_handles_are_refused():
    assert "NULL handle" in refused("h3b_sdpa_window_dev", None, window())
    assert "NULL handle" in refused("h3b_kv8_append_dev", None, cache(), append())
    assert "NULL handle" in refused("h3b_kv8_sdpa_dev", None, cache(), attention())
    assert "NULL arguments" in refused("h3b_sdpa_window_dev", fake_handle(), None)
    assert "NULL arguments" in refused("h3b_kv8_append_dev", fake_handle(), cache(), None)
    assert "NULL arguments" in refused("h3b_kv8_sdpa_dev", fake_handle(), cache(), None)
    assert "NULL cache" in refused("h3b_kv8_append_dev", fake_handle(), None, append())
    assert "NULL cache" in refused("h3b_kv8_sdpa_dev", fake_handle(), None, attention())


def cache(**change):
    return block(l.KV8_CACHE, dict(pages=10, page_tokens=128, kv_heads=4, head_dim=128, d_k=A, d_v=A, d_k_scale=A, d_v_scale=A) | change)


APPEND = dict(k=A, v=A, cu=A, start=A, table=A, kr=512, kh=128, vr=512, vh=128, rows=5, stride=3, n_seq=2, max_rows=5, dtype=l.BF16)
CACHE = dict(q=A, out=A, cu=A, len=A, table=A, qr=1024, qh=128, orow=1024, oh=128, rows=6, heads=8, stride=3, n_seq=2, max_rows=5,
             max_len=99, left=-1, right=0, sinks=0, block=1, scale=0.1, dtype=l.F16)


def append(**change):
    return block(l.KV8_APPEND_ARGS, APPEND | change)


def attention(**change):
    return block(l.KV8_SDPA_ARGS, CACHE | change)


BAD_CACHE = [(dict(head_dim=64), "head_dim"), (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=96), "page_tokens"),
             (dict(page_tokens=1 << 17), "page_tokens"), (dict(kv_heads=0), "K/V heads"), (dict(pages=0), "pages"),
             (dict(pages=1 << 24), "pages"), (dict(d_k=None), "NULL cache"), (dict(d_v_scale=None), "NULL cache"),
             (dict(d_v=A + 8), "aligned"), (dict(d_k_scale=A + 2), "aligned")]
BAD_BATCH = [(dict(cu=None), "NULL sequence table"), (dict(table=None), "NULL sequence table"), (dict(table=A + 1), "4-byte"),
             (dict(stride=0), "table_stride"), (dict(stride=1 << 23), "table_stride"), (dict(n_seq=65536), "sequences"),
             (dict(max_rows=7), "max_rows"), (dict(max_rows=-1), "max_rows"), (dict(rows=-1), "large"), (dict(n_seq=-1), "sequences"), (dict(dtype=l.F32), "bf16 or f16")]


@pytest.mark.parametrize("change, says", BAD_CACHE)
def test_cache_layout_refusals(change, says):
    assert says in refused("h3b_kv8_append_dev", fake_handle(), cache(**change), append())
    assert says in refused("h3b_kv8_sdpa_dev", fake_handle(), cache(**change), attention())


@pytest.mark.parametrize("change, says", BAD_BATCH)
def test_batch_refusals(change, says):
    assert says in refused("h3b_kv8_append_dev", fake_handle(), cache(), append(**change))
    assert says in refused("h3b_kv8_sdpa_dev", fake_handle(), cache(), attention(**change))


@pytest.mark.parametrize("change, says", [(dict(k=None), "NULL tensor"), (dict(v=A + 8), "16-byte"), (dict(kr=4), "multiples of 8"),
                                          (dict(vh=0), "strides must be given"), (dict(kr=1 << 40), "stride too large")])
def test_append_refusals(change, says):
    assert says in refused("h3b_kv8_append_dev", fake_handle(), cache(), append(**change))


@pytest.mark.parametrize("change, says", [(dict(heads=6), "6 heads over 4"), (dict(q=None), "NULL tensor"), (dict(out=A + 8), "16-byte"),
                                          (dict(qr=4), "multiples of 8"), (dict(oh=0), "strides must be given"), (dict(sinks=-2), "sinks"),
                                          (dict(block=0), "block"), (dict(scale=-1.0), "scale"), (dict(max_len=1 << 29), "max_len")])
def test_cache_attention_refusals(change, says):
    assert says in refused("h3b_kv8_sdpa_dev", fake_handle(), cache(), attention(**change))


def test_calls_without_work_return_before_the_device():
    lib, err = h3c_b200.load(), C.create_string_buffer(512)
    assert lib.h3b_sdpa_window_dev(fake_handle(), window(lq=0, q=None, out=None), err, 512) == 1
    assert lib.h3b_kv8_append_dev(fake_handle(), cache(), append(n_seq=0, cu=None, start=None, table=None), err, 512) == 1
    assert lib.h3b_kv8_append_dev(fake_handle(), cache(), append(rows=0, max_rows=0, k=None, v=None), err, 512) == 1
    assert lib.h3b_kv8_sdpa_dev(fake_handle(), cache(), attention(rows=0, max_rows=0, q=None, out=None), err, 512) == 1
    assert lib.h3b_kv8_sdpa_dev(fake_handle(), cache(), attention(n_seq=0), err, 512) == 1


def test_argument_blocks_have_the_size_of_the_header_structs(tmp_path):
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "h3_b200.h"\nint main(void) { printf("%zu %zu %zu %zu", sizeof(h3b_sdpa_window_args), '
                   'sizeof(h3b_kv8_cache), sizeof(h3b_kv8_append_args), sizeof(h3b_kv8_sdpa_args)); return 0; }\n')
    subprocess.run(["gcc", "-I" + str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    # a block may leave out the padding behind its last field
    want = [-(-b.size // 8) * 8 for b in (l.SDPA_WINDOW_ARGS, l.KV8_CACHE, l.KV8_APPEND_ARGS, l.KV8_SDPA_ARGS)]
    assert [int(x) for x in got] == want


def test_cache_object_checks_its_tensors():
    import torch
    k = torch.zeros(3, 2, 128, 128, dtype=torch.uint8)
    s = torch.zeros(3, 2, 2)
    h3c_b200.KvCache8(k, k.clone(), s, s.clone())
    c = h3c_b200.KvCache8(k.view(torch.float8_e4m3fn), k, s, s)
    assert c.kv_heads == 2 and l.KV8_CACHE.unpack(c.packed) == (3, 128, 2, 128, k.data_ptr(), k.data_ptr(), s.data_ptr(), s.data_ptr())
    with pytest.raises(AttributeError):
        c.k = k
    for bad in ((k[:2], k, s, s), (k, k, s[..., :1], s), (k.float(), k, s, s), (k, k, s.double(), s),
                (k.transpose(1, 2), k.transpose(1, 2), s, s), (k, k, s.expand(3, 2, 2)[:, :, :1], s)):
        with pytest.raises(h3c_b200.H3Error):
            h3c_b200.KvCache8(*bad)


@pytest.mark.parametrize("rows, heads, orow, oh, overlaps", [
    (4, 8, 128, 128, True),      # row 1 of head 0 is row 0 of head 1
    (4, 8, 1016, 128, True),     # rows a piece shorter than their heads
    (4, 8, 128, 504, True),      # heads a piece shorter than their rows
    (4, 8, 512, 384, True),
    (1 << 28, 8, (1 << 39) - 8, 128, False), (1 << 28, 8, 128, (1 << 35) - 8, True),   # products past 64 bits and past 32
    (4, 8, 1024, 128, False), (4, 8, 2048, 256, False),     # rows of heads, packed and not
    (4, 8, 128, 512, False), (4, 8, 136, 536, False),       # heads of rows
    (1, 8, 8, 128, False), (4, 1, 128, 8, False)])          # a stride that nothing uses
def test_outputs_whose_rows_or_heads_overlap_are_refused(rows, heads, orow, oh, overlaps):
    """Both entry points share the check; another refusal stands behind it, so that nothing is launched (for the largest
    counts another one stands before it: 2^28 rows of 8 heads are 2^31 rows of one K/V head)."""
    large = rows * heads > 0x7fffff00
    says = refused("h3b_sdpa_window_dev", fake_handle(), window(lq=rows, heads=heads, kv=1, orow=orow, oh=oh, q_pos=-1))
    assert ("too large" if large else "overlap" if overlaps else "q_pos") in says
    says = refused("h3b_sdpa_window_dev", fake_handle(), window(lq=rows, heads=heads, kv=heads, orow=orow, oh=oh, q_pos=-1))
    assert ("overlap" if overlaps else "q_pos") in says
    says = refused("h3b_kv8_sdpa_dev", fake_handle(), cache(kv_heads=heads),
                   attention(rows=rows, heads=heads, orow=orow, oh=oh, max_rows=1, max_len=1 << 29))
    assert ("overlap" if overlaps else "max_len") in says


@pytest.mark.parametrize("seed", range(4))
def test_tiles_of_an_item_stay_within_the_bound_that_picks_the_kernel(seed):
    """The host decides by count <= reach // 128 + 4, with reach the sum of left, right, two blocks, rows and sinks, or all
    keys; a side without a bound counts as 2^29."""
    rng, lib, far = np.random.default_rng(seed), h3c_b200.load(), 1 << 29
    s, f, c = C.c_int(), C.c_int(), C.c_int()
    for _ in range(5000):
        n, rows = int(rng.integers(1, [5000, 200000][rng.integers(2)])), int(rng.integers(1, 257))
        pos = int(rng.integers(0, n + 500))
        left, right = (int(rng.choice([-1, 0, rng.integers(0, 3000)])) for _ in range(2))
        block, sinks = int(rng.choice([1, rng.integers(1, 4000)])), int(rng.choice([0, rng.integers(0, 3000)]))
        assert lib.h3b_window_tiles(n, pos, rows, left, right, sinks, block, 128, C.byref(s), C.byref(f), C.byref(c)) == 1
        reach = min(sum(far if x < 0 else x for x in (left, right)) + 2 * block + rows + sinks, n)
        assert c.value <= reach // 128 + 4
