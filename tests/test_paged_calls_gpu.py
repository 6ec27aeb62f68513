"""PagedInt4Cache's calls where they are refused or fail: what they leave behind."""

import pytest
import torch

from _paged import held
from test_paged_cache_gpu import BF, FP, check_held, fill, make, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host", [True, False])
def test_no_memory_for_the_span_of_forked_sequences(gpu, host):
    """An extend whose span cannot be allocated leaves pages shared as they were; again and again."""
    cache = make(D=256, H=8, HQ=8, pages=16)
    parent, m = fill(cache, [100])
    kids = cache.fork(parent * 3)
    for s in kids:
        m.rows[s] = m.rows[parent[0]]
    seqs = kids if host else torch.tensor(kids)  # the host module takes plain lists alone
    table = cache.page_table(cache.span(kids, [0] * 3, [1] * 3))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.0)  # the span's workspace (32 MiB) is not to be had
    try:
        for _ in range(20):
            with pytest.raises(RuntimeError, match="out of memory"):
                cache.extend(seqs, [130, 130, 130])
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert cache.pages_in_use == 2 and cache.lengths(kids) == [100] * 3
    assert torch.equal(cache.page_table(cache.span(kids, [0] * 3, [1] * 3)), table) and torch.equal(table[0], table[1])
    check_held(cache, m, kids)
    cache.extend(seqs, [130, 130, 130])
    assert cache.pages_in_use == 2 + 3 * 3 and cache.lengths(kids) == [230] * 3


def test_what_requires_grad_is_refused(gpu):
    """There is no backward pass: no call drops a gradient silently."""
    cache = make(D=64, H=2, HQ=4)
    seqs, m = fill(cache, [100])
    span = cache.span(seqs, [90], [10])
    q, kv = rows((10, 4, 64), BF, 5), rows((10, 2, 64), BF, 6)
    want = cache.attend(0, span, q, scaling=0.1, gate=q)
    with_grad, kv_grad = q.clone().requires_grad_(), kv.clone().requires_grad_()
    wide = torch.cat((q, q), -1).requires_grad_()[..., 4:68]  # rows that are copied first
    for name, call in [("query", lambda: cache.attend(0, span, with_grad, scaling=0.1)), ("query", lambda: cache.attend(0, span, wide, scaling=0.1)),
                       ("gate", lambda: cache.attend(0, span, q, scaling=0.1, gate=with_grad)),
                       ("out", lambda: cache.attend(0, span, q, scaling=0.1, out=with_grad)),
                       ("keys", lambda: cache.store(0, span, kv_grad, kv)), ("values", lambda: cache.store(0, span, kv, kv_grad))]:
        with pytest.raises(RuntimeError, match=name + " requires grad"):
            call()
    check_held(cache, m, seqs)
    with torch.no_grad():
        assert torch.equal(cache.attend(0, span, with_grad, scaling=0.1, gate=with_grad), want)
        cache.store(0, span, kv_grad, kv_grad)
    with torch.inference_mode():
        assert cache.attend(0, span, with_grad, scaling=0.1, gate=with_grad).shape == want.shape
    assert torch.equal(with_grad, q)


def test_a_captured_store_is_not_replayed_over_shared_pages(gpu):
    """A replay cannot refuse, so the fill before it does; the span then holds what it held."""
    cache = make(D=64, H=2, HQ=4)
    seqs, m = fill(cache, [100, 90])
    span = cache.span(seqs, [70, 70], [4, 4])
    k = rows((8, 2, 64), BF, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.store(0, span, k, k)
    child, = cache.fork(seqs[:1])
    with pytest.raises(RuntimeError, match="share a page"):
        cache.span([seqs[0], child], [70, 70], [4, 4], span=span)
    assert span.seqs == seqs
    read = cache.span([seqs[0], child], [70, 70], [4, 4])  # another one, not stored: as before
    cache.attend(0, read, rows((8, 4, 64), BF, 6), scaling=0.1)
    cache.span([seqs[0], child], [70, 70], [4, 4], span=read)
    want = held(k.cpu(), k.cpu())[0].to(BF)
    graph.replay()  # what the span was filled with last
    for s, part in zip(seqs, want.split(4)):
        assert torch.equal(cache.read(0, cache.span([s], [70], [4]))[0].cpu(), part)
    cache.span([seqs[1], child], [80, 10], [4, 4], span=span)
    graph.replay()
    for s, at, part in zip([seqs[1], child], [80, 10], want.split(4)):
        assert torch.equal(cache.read(0, cache.span([s], [at], [4]))[0].cpu(), part)


@pytest.mark.parametrize("ours", [True, False])
def test_captures_are_those_of_the_caches_device(gpu, monkeypatch, ours):
    """With another device current, what counts is whether the cache's own records a graph (devices by proxy here)."""
    cache = make(D=64, H=1, HQ=1)
    seqs, _ = fill(cache, [3])
    on_ours = []

    class Device:
        def __init__(self, device):
            assert torch.device(device) == cache.device

        def __enter__(self):
            on_ours.append(1)

        def __exit__(self, *args):
            on_ours.pop()

    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "current_device", lambda: cache.device.index + 1)
        patch.setattr(torch.cuda, "device", Device)
        patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(on_ours) == ours)
        if ours:
            for call in (lambda: cache.extend(seqs), lambda: cache.free(seqs), lambda: cache.compact()):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
        else:
            cache.extend(seqs)
    assert cache.lengths(seqs) == [3 if ours else 4]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("start,count", [(2999, 1), (2992, 8), (2000, 100), (0, 130)])
def test_answers_in_place_of_the_queries_or_gates(gpu, dtype, start, count):
    """out may be the query or the gate itself, in every form, split over the context or not."""
    cache = make(D=128, HQ=8, H=2, dtype=dtype)
    seqs, _ = fill(cache, [3000, 40])
    span = cache.span(seqs, [start, 39], [count, 1])
    q, gate = (rows((count + 1, 8, 128), dtype, i) for i in (5, 6))
    want = cache.attend(0, span, q, scaling=0.1, gate=gate)
    for at in range(2):
        x = [q.clone(), gate.clone()]
        assert torch.equal(cache.attend(0, span, x[0], scaling=0.1, gate=x[1], out=x[at]), want)
