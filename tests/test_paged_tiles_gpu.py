"""PagedInt4Cache's attention in tiles of 256 query rows (eight waves), which the plan takes once such tiles fill the
chip: against the plain 64-bit counterpart, with the plan's choice asserted."""

import pytest
import torch

from _paged import Mirror, attention
from anna_amd.paged_cache import PagedInt4Cache
from test_paged_cache_gpu import BF, FP, check_attend, fill, rows

pytestmark = pytest.mark.gpu


def tiles(D, HQ, H, dtype, lens, counts, length=1024):
    """A cache of sequences of these lengths whose last `counts` tokens are attended for in tiles of 256 rows."""
    cache = PagedInt4Cache(num_layers=1, num_pages=sum(-(-n // 64) for n in lens), kv_heads=H, q_heads=HQ, head_dim=D,
                           max_sequences=len(lens), max_length=length, dtype=dtype)
    seqs, m = fill(cache, lens, seed=D + HQ)
    starts = [n - c for n, c in zip(lens, counts)]
    span = cache.span(seqs, starts, counts)
    assert span._c.tile_rows == 256 and span._c.tile_items * H >= 256
    return cache, seqs, m, starts


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("HQ,H", [(32, 8), (16, 16), (40, 8)])
@pytest.mark.parametrize("gated", [False, True])
def test_prompts(gpu, D, dtype, HQ, H, gated):
    """Ragged prompts whose last tiles hold from a few rows to all 256 of them."""
    G = HQ // H
    n = 1 + 256 // H
    lens = [-(-(65 + 37 * i % 192) // G) for i in range(n - 2)] + [-(-600 // G), 256 // G]
    cache, seqs, m, starts = tiles(D, HQ, H, dtype, lens, lens)
    check_attend(cache, m, seqs, starts, lens, gated=gated)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_chunks_behind_a_context(gpu, D, dtype):
    """Chunks at the end of contexts that end anywhere in a page, beside single tokens and a sequence without any."""
    counts = [17 + 5 * i % 50 for i in range(31)] + [80, 1, 0, 3]
    lens = [c + 23 * i % 150 for i, c in enumerate(counts)]
    cache, seqs, m, starts = tiles(D, 32, 8, dtype, lens, counts)
    check_attend(cache, m, seqs, starts, counts, gated=True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("what", ["key", "value", "query"])
def test_beyond_fp16(gpu, D, dtype, what):
    """What fp16 operands do not hold, from the second page of every other sequence on: bf16's tolerance there."""
    factor = {"key": 2.0 ** 9, "value": 2.0 ** 14 if dtype == BF else 2.0 ** 12, "query": 2.0 ** 12}[what]
    lens = [70 + 11 * i % 90 for i in range(33)]
    cache, seqs, _, _ = tiles(D, 32, 8, dtype, lens, lens)
    total = sum(lens)
    k, v, q = (rows((total, h, D), torch.float32, i) for i, h in ((1, 8), (2, 8), (3, 32)))
    at = [sum(lens[:i]) for i in range(len(lens))]
    for i in range(0, len(lens), 2):
        x = {"key": k, "value": v, "query": q}[what]
        x[at[i] + 66:at[i] + 70] *= factor
    scaling = D ** -0.5 / (1.0 if what == "value" else factor)  # large scores have large errors
    big = torch.finfo(dtype).max
    k, v, q = (x.clamp(-big, big).to(dtype) for x in (k, v, q))
    span = cache.span(seqs, [0] * len(lens), lens)
    cache.store(0, span, k, v)
    got = cache.attend(0, span, q, scaling=scaling).cpu().double()
    for i, n in enumerate(lens):
        here = slice(at[i], at[i] + n)
        m = Mirror()
        m.store(0, 0, k[here].cpu(), v[here].cpu())
        want, tol = attention(q[here].cpu(), *m.rows[0], 0, scaling, dtype)
        if i % 2 == 0:
            tol += attention(q[here].cpu(), *m.rows[0], 0, scaling, BF)[1]
        # the cache holds a value to within half its group's scale, so past the type's largest too: an answer that is past
        # it within its bound may be infinite
        past = torch.isinf(got[here]) & (want.abs() + tol > big) & (got[here] * want > 0)
        assert (((got[here] - want).abs() <= tol) | past).all(), (i, n)


def test_rows_of_other_strides(gpu):
    """Queries and gates out of a wider tensor, and an output given."""
    lens = [60 + i for i in range(33)]
    cache, seqs, m, starts = tiles(64, 32, 8, BF, lens, lens)
    span = cache.span(seqs, starts, lens)
    fused = rows((sum(lens), 32 + 8, 64), BF, 5)
    q, gate = fused[:, :32], fused[:, 8:]
    want = cache.attend(0, span, q.contiguous(), scaling=0.1, gate=gate.contiguous())
    out = torch.empty_like(want)
    assert cache.attend(0, span, q, scaling=0.1, gate=gate, out=out) is out and torch.equal(out, want)


@pytest.mark.parametrize("D,HQ,H,counts,lens,rows_of_a_tile", [
    (64, 8, 2, [1, 3, 40, 100, 0], [2900, 10, 700, 64, 5], 128),
    (256, 4, 2, [33, 1, 70], [1, 1800, 300], 128),
    (128, 32, 8, [17 + i % 40 for i in range(32)] + [1, 2], [50 * (i % 7) for i in range(32)] + [2000, 3], 256),
])
def test_captured_mixed_steps_equal_eager_ones(gpu, D, HQ, H, counts, lens, rows_of_a_tile):
    """store + attend of single tokens, drafts and prompts together, captured once: replays over other sequences, shorter and
    longer ones, whose launches are laid out otherwise than those of the capture."""
    n, total = len(counts), sum(counts)

    def run(captured):
        cache = PagedInt4Cache(num_layers=1, num_pages=sum(-(-(m + 8 * c) // 64) + 1 for m, c in zip(lens, counts)) + 64, kv_heads=H,
                               q_heads=HQ, head_dim=D, max_sequences=n + 1, max_length=4096)
        seqs, _ = fill(cache, lens)
        k, v, q, out = (torch.zeros((total, h, D), dtype=BF, device="cuda") for h in (H, H, HQ, HQ))

        def step(span):
            cache.store(0, span, k, v)
            cache.attend(0, span, q, scaling=0.1, gate=q, out=out)

        seen, span, graph = [], None, None
        for i in range(7):
            if i == 3:  # other sequences, much longer or shorter than those of the capture
                long = max(range(n), key=lambda j: lens[j])
                kid, = cache.fork([seqs[long]])
                cache.truncate(seqs[long], 7)
                other = min(range(n), key=lambda j: lens[j])
                cache.free([seqs[other]])
                seqs[other] = kid
                cache.compact()
            if i == 5:
                seqs.reverse()
            span = cache.extend(seqs, counts, span=span)
            assert span._c.tile_rows == rows_of_a_tile
            for t, seed in ((k, 100), (v, 200), (q, 300)):
                t.copy_(rows(t.shape, BF, seed + i))
            if not captured or i == 0:
                step(span)
            else:
                if graph is None:
                    torch.cuda.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step(span)
                graph.replay()
            seen.append(out.clone())
        return seen

    for i, (a, b) in enumerate(zip(run(False), run(True))):
        assert torch.equal(a, b) and torch.isfinite(a).all(), i
