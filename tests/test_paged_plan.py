"""The paged cache's plans of tokens that are still to come, through the C ABI (no GPU)."""

import ctypes

import pytest

from anna_amd import _lib
from test_paged_cache import handle, i32, i64

SIZES = ("sequences", "tokens", "words", "partial_rows", "split_capacity", "unit_capacity", "touch_capacity", "tile_capacity",
         "few_rows", "tile_rows")


def state(h, seqs):
    lengths, live = i64(*[0] * len(seqs)), ctypes.c_int64()
    _lib.call("anna_mi_paged_lengths", h, len(seqs), seqs, lengths, ctypes.byref(live))
    return list(lengths), live.value


@pytest.mark.parametrize("counts", [(1, 1, 1, 1), (0, 7, 64, 1), (70, 200, 1, 0), (0, 0, 0, 0)])
@pytest.mark.parametrize("HQ,H,D", [(4, 2, 64), (64, 8, 128), (2, 2, 256)])
def test_the_plan_of_an_extend_is_that_of_its_tokens(counts, HQ, H, D):
    h = handle(num_pages=64, kv_heads=H, q_heads=HQ, head_dim=D, max_pages=8)
    seqs, starts = i32(0, 0, 0, 0), i64(0, 0, 0, 0)
    _lib.call("anna_mi_paged_add", h, 4, seqs)
    _lib.call("anna_mi_paged_extend", h, 4, seqs, i64(0, 100, 64, 5), None, None)
    before = state(h, seqs)
    ahead, span = _lib.PagedSpan(), _lib.PagedSpan()
    _lib.call("anna_mi_paged_span_plan", h, 4, seqs, None, i64(*counts), ctypes.byref(ahead))
    assert state(h, seqs) == before
    for s, n, have in zip(seqs, counts, before[0]):  # one by one, as no launch may go out here
        starts[list(seqs).index(s)] = have
    _lib.call("anna_mi_paged_destroy", h)

    h = handle(num_pages=64, kv_heads=H, q_heads=HQ, head_dim=D, max_pages=8)
    _lib.call("anna_mi_paged_add", h, 4, seqs)
    _lib.call("anna_mi_paged_extend", h, 4, seqs, i64(*(a + b for a, b in zip(before[0], counts))), None, None)
    _lib.call("anna_mi_paged_span_plan", h, 4, seqs, starts, i64(*counts), ctypes.byref(span))
    assert [getattr(ahead, f) for f in SIZES] == [getattr(span, f) for f in SIZES]
    _lib.call("anna_mi_paged_destroy", h)


def test_refusals():
    h = handle()
    seqs = i32(0, 0)
    _lib.call("anna_mi_paged_add", h, 2, seqs)
    _lib.call("anna_mi_paged_extend", h, 2, seqs, i64(100, 0), None, None)
    span = ctypes.byref(_lib.PagedSpan())
    for args, match in [((2, seqs, None, i64(157, 0), span), "at most 256 fit"), ((2, seqs, None, i64(1, (1 << 63) - 1), span), "at most 256 fit"),
                        ((2, seqs, None, i64(-1, 0), span), "at most 256 fit"), ((2, i32(1, 1), None, i64(1, 1), span), "twice"),
                        ((1, i32(3), None, i64(1), span), "not in use"), ((1, seqs, None, None, span), "null arrays")]:
        with pytest.raises(RuntimeError, match=match):
            _lib.call("anna_mi_paged_span_plan", h, *args)
    with pytest.raises(RuntimeError, match="null starts"):
        _lib.call("anna_mi_paged_span_fill", h, 1, seqs, None, i64(1), ctypes.byref(_lib.PagedSpan(buf=64)), None)
    assert state(h, seqs) == ([100, 0], 2)
    _lib.call("anna_mi_paged_destroy", h)


NO_MEMORY = """
import ctypes, resource, sys
sys.path[:0] = ["tests", "."]
from anna_amd import _lib
_lib.load()
d = _lib.PagedDesc(0, 1, (1 << 30), 1, 1, 64, 1 << 10, 1 << 10, 64, 64)  # 4 GiB of counts for the pages
h = ctypes.c_void_p(7)
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (1 << 30),) * 2)
for _ in range(300):  # 4 MiB of table each, were they kept
    try:
        _lib.call("anna_mi_paged_create", ctypes.byref(d), ctypes.byref(h))
        raise SystemExit("created")
    except RuntimeError as e:
        assert "paged_create" in str(e), e
assert h.value == 7
"""


def test_a_cache_that_finds_no_memory_leaves_nothing():
    import subprocess
    import sys
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", NO_MEMORY], cwd=Path(__file__).parents[1], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
