"""PagedInt4Cache against the plain 64-bit counterpart (tests/_paged.py): what the pages hold, attention over
them in all its forms, and the pages' life (copy on write, truncate, free, compact, resize)."""

import random
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from _paged import Mirror, attention, held
from anna_amd.paged_cache import PagedInt4Cache

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rows(shape, dtype, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x[..., :: 37] *= 8  # channels that stand out, as keys have
    return x.to(dtype).to(device)


def make(D=128, HQ=8, H=2, dtype=BF, pages=64, layers=1, sequences=16, length=4096, **kw):
    return PagedInt4Cache(num_layers=layers, num_pages=pages, kv_heads=H, q_heads=HQ, head_dim=D, max_sequences=sequences,
                          max_length=length, dtype=dtype, **kw)


def fill(cache, lens, seed=0, layer=0):
    """Sequences of these lengths with stored tokens -> (seqs, mirror)."""
    seqs = cache.add(len(lens))
    span = cache.extend(seqs, lens)
    k, v = (rows((sum(lens), cache.kv_heads, cache.head_dim), cache.dtype, seed + i) for i in (0, 1))
    cache.store(layer, span, k, v)
    m, at = Mirror(), 0
    for s, n in zip(seqs, lens):
        m.store(s, 0, k[at:at + n].cpu(), v[at:at + n].cpu())
        at += n
    return seqs, m


def check_held(cache, m, seqs, layer=0):
    for s in seqs:
        n = m.rows[s][0].shape[0]
        k, v = cache.read(layer, cache.span([s], [0], [n]))
        for got, want in ((k, m.rows[s][0]), (v, m.rows[s][1])):
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=123.0), torch.nan_to_num(want.to(cache.dtype), nan=123.0))


def check_attend(cache, m, seqs, starts, counts, scaling=None, gated=False, seed=7, layer=0, out=None):
    D, HQ = cache.head_dim, cache.q_heads
    scaling = D ** -0.5 if scaling is None else scaling
    span = cache.span(seqs, starts, counts)
    q = rows((sum(counts), HQ, D), cache.dtype, seed)
    gate = rows(q.shape, cache.dtype, seed + 1) if gated else None
    got = cache.attend(layer, span, q, scaling=scaling, gate=gate)
    at = 0
    for s, st, n in zip(seqs, starts, counts):
        if n == 0:
            continue
        want, tol = attention(q[at:at + n].cpu(), *(x[:st + n] for x in m.rows[s]), st, scaling, cache.dtype,
                              None if gate is None else gate[at:at + n].cpu())
        err = (got[at:at + n].cpu().double() - want).abs()
        bad = ~((err <= tol) | (torch.isnan(want) & torch.isnan(err)))
        if bad.any():
            i = tuple(bad.nonzero()[0].tolist())
            pytest.fail(f"sequence {s} start {st} count {n}: {int(bad.sum())} of {bad.numel()} values off, the first at {i}: "
                        f"{float(got[at:at + n][i])}, not {float(want[i])} within {float(tol[i])}", pytrace=False)
        at += n
    return got


# ---------------------------------------------------------------- what the pages hold

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_store_and_read_are_exact(gpu, D, dtype):
    cache = make(D=D, H=3, HQ=3, dtype=dtype)
    seqs, m = fill(cache, [1, 63, 64, 65, 0, 200], seed=D)
    check_held(cache, m, seqs)


@pytest.mark.parametrize("pieces", [[1] * 70, [7, 57, 1, 64, 3, 60], [33, 31, 32, 95]])
def test_tokens_enter_in_pieces(gpu, pieces):
    cache = make(D=128)
    seqs, m = fill(cache, [5, 30])
    for i, n in enumerate(pieces):
        span = cache.extend(seqs, [n, max(0, n - 2)])
        assert span.starts == [m.rows[s][0].shape[0] for s in seqs]
        k, v = (rows((span.tokens, 2, 128), BF, 100 + 2 * i + j) for j in (0, 1))
        cache.store(0, span, k, v)
        m.store(seqs[0], span.starts[0], k[:n].cpu(), v[:n].cpu())
        m.store(seqs[1], span.starts[1], k[n:].cpu(), v[n:].cpu())
    check_held(cache, m, seqs)
    check_attend(cache, m, seqs, [0, 0], cache.lengths(seqs))


def special(dtype):
    """Groups where the rounding can go wrong: constant, zero, tiny, huge, one-sided, with ties."""
    big = torch.finfo(dtype).max
    x = torch.zeros(12, 64, dtype=torch.float32)
    x[1] = 3.0
    x[2] = -0.37
    x[3] = torch.linspace(100, 101, 64)
    x[4] = torch.linspace(-big, big, 64, dtype=torch.float64).float()
    x[5] = big
    x[6, 5] = 1.0
    x[7] = torch.arange(64) % 16 - 7.5
    x[8] = torch.arange(64) % 16 * 0.5
    x[9] = torch.linspace(-5, -4, 64)
    x[10] = torch.finfo(dtype).tiny if dtype == FP else 2.0 ** -101
    x[11] = torch.arange(64) % 31 * 2.0 ** -90 if dtype == BF else torch.arange(64) * 2.0 ** -24
    return x.clamp(-big, big).to(dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_store_special_groups(gpu, dtype):
    cache = make(D=64, H=1, HQ=1, dtype=dtype)
    x = special(dtype)[:, None]
    seq = cache.add()
    span = cache.extend(seq, [12])
    cache.store(0, span, x.cuda(), x.flip(0).contiguous().cuda())
    k, v = cache.read(0, span)
    wk, wv, _, _ = held(x, x.flip(0))
    assert torch.equal(k.cpu(), wk.to(dtype)) and torch.equal(v.cpu(), wv.to(dtype))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_a_token_that_is_not_finite_is_its_viewers_alone(gpu, dtype):
    cache = make(D=128, H=2, HQ=4, dtype=dtype)
    seqs = cache.add(2)
    span = cache.extend(seqs, [100, 90])
    k, v = (rows((190, 2, 128), dtype, i) for i in (0, 1))
    k[40, 0, 3] = float("nan")
    v[50, 1, 127] = float("inf")
    v[70, 0, 64] = float("-inf")
    cache.store(0, span, k, v)
    m = Mirror()
    m.store(seqs[0], 0, k[:100].cpu(), v[:100].cpu())
    m.store(seqs[1], 0, k[100:].cpu(), v[100:].cpu())
    check_held(cache, m, seqs)
    got = check_attend(cache, m, seqs, [0, 0], [100, 90])
    assert not torch.isnan(got[:40]).any() and torch.isnan(got[40:100, :2]).all()
    assert not torch.isnan(got[40:50, 2:]).any() and torch.isnan(got[50:100, 2:]).all() and not torch.isnan(got[100:]).any()
    got = check_attend(cache, m, seqs, [39, 0], [3, 1])
    assert not torch.isnan(got[0]).any() and torch.isnan(got[1:3, :2]).all()


# ---------------------------------------------------------------- attention

HEADS = [(16, 2, 256), (32, 8, 128), (28, 4, 128), (8, 8, 64), (8, 1, 64), (24, 2, 256), (5, 5, 128), (40, 2, 64)]


@pytest.mark.parametrize("HQ,H,D", HEADS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attend_single_tokens(gpu, HQ, H, D, dtype):
    lens = [1, 2, 63, 64, 65, 700, 129]
    cache = make(D=D, HQ=HQ, H=H, dtype=dtype)
    seqs, m = fill(cache, lens, seed=HQ)
    check_attend(cache, m, seqs, [n - 1 for n in lens], [1] * len(lens), gated=D == 128)


@pytest.mark.parametrize("HQ,H,D", HEADS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attend_several_tokens(gpu, HQ, H, D, dtype):
    lens = [9, 70, 64, 300, 129, 1, 65]
    counts = [9, 5, 1, 8, 0, 1, 3]
    cache = make(D=D, HQ=HQ, H=H, dtype=dtype)
    seqs, m = fill(cache, lens, seed=H)
    check_attend(cache, m, seqs, [n - c for n, c in zip(lens, counts)], counts, gated=D == 256)


@pytest.mark.parametrize("HQ,H,D", HEADS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attend_prompts_and_chunks(gpu, HQ, H, D, dtype):
    lens = [130, 1, 64, 333, 400, 257, 90]
    counts = [130, 1, 64, 200, 129, 3, 65]
    cache = make(D=D, HQ=HQ, H=H, dtype=dtype)
    seqs, m = fill(cache, lens, seed=D + H)
    check_attend(cache, m, seqs, [n - c for n, c in zip(lens, counts)], counts, gated=HQ == 16)


def test_attend_tokens_before_the_last(gpu):
    lens = [300, 200]
    cache = make(D=128, HQ=8, H=2)
    seqs, m = fill(cache, lens)
    check_attend(cache, m, seqs, [17, 64], [40, 64])
    check_attend(cache, m, seqs[::-1], [0, 299], [1, 1])


@pytest.mark.parametrize("count", [1, 130])
def test_attend_long_context(gpu, count):
    cache = make(D=64, HQ=2, H=1, pages=600, length=40000)
    seqs, m = fill(cache, [33000])
    check_attend(cache, m, seqs, [33000 - count], [count])


@pytest.mark.parametrize("scaling", [1e-6, 4.0])
@pytest.mark.parametrize("count", [1, 90])
def test_attend_flat_and_peaked_scores(gpu, scaling, count):
    cache = make(D=64, HQ=4, H=2, dtype=FP)
    seqs, m = fill(cache, [500])
    check_attend(cache, m, seqs, [500 - count], [count], scaling=scaling)


def test_attend_large_and_small_values(gpu):
    for dtype, big, small in ((BF, 2.0 ** 100, 2.0 ** -90), (FP, 2.0 ** 9, 2.0 ** -14), (FP, 2.0 ** 12, 2.0 ** -14)):
        for factor in (big, small):  # 2^12: infinities among the values
            cache = make(D=64, HQ=2, H=1, dtype=dtype)
            seqs = cache.add(1)
            k = rows((150, 1, 64), dtype, 1)
            v = (rows((150, 1, 64), torch.float32, 2) * factor).to(dtype)
            cache.store(0, cache.extend(seqs, [150]), k, v)
            m = Mirror()
            m.store(seqs[0], 0, k.cpu(), v.cpu())
            for n in (1, 100):
                q = rows((n, 2, 64), dtype, 3)
                got = cache.attend(0, cache.span(seqs, [150 - n], [n]), q, scaling=0.125)
                want, tol = attention(q.cpu(), *m.rows[seqs[0]], 150 - n, 0.125, dtype)
                err = (got.cpu().double() - want).abs()
                assert ((err <= tol) | (torch.isnan(err) & torch.isnan(want))).all(), (dtype, factor, n)


@pytest.mark.parametrize("D,H,HQ", [(64, 2, 4), (128, 1, 4), (256, 1, 2)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("what", ["key", "value", "tiny value", "query"])
def test_tiles_beyond_fp16(gpu, D, H, HQ, dtype, what):
    """Scales of keys or values, or queries, that leave what fp16 operands hold, from some page on: the tiles' form goes
    on in bf16 there, to bf16's tolerance."""
    n, factor = 300, {"key": 2.0 ** 9, "value": 2.0 ** 14 if dtype == BF else 2.0 ** 12, "tiny value": 2.0 ** -22, "query": 2.0 ** 12}[what]
    cache = make(D=D, H=H, HQ=HQ, dtype=dtype)
    seqs = cache.add(1)
    k, v, q = (rows((n, h, D), torch.float32, i) for i, h in ((1, H), (2, H), (3, HQ)))
    if what == "key":
        k[150:170] *= factor
    elif what == "query":
        q[190:, 0] *= factor
    else:
        v[150:170] *= factor
    # large scores have large errors: keep them apart from the ranges that are tested
    scaling = D ** -0.5 / (factor if what in ("key", "query") else 1.0)
    big = torch.finfo(dtype).max
    k, v, q = (x.clamp(-big, big).to(dtype) for x in (k, v, q))
    cache.store(0, cache.extend(seqs, [n]), k, v)
    m = Mirror()
    m.store(seqs[0], 0, k.cpu(), v.cpu())
    got = cache.attend(0, cache.span(seqs, [0], [n]), q, scaling=scaling)
    want, tol = attention(q.cpu(), *m.rows[seqs[0]], 0, scaling, BF)  # bf16's steps
    want16, tol16 = attention(q.cpu(), *m.rows[seqs[0]], 0, scaling, dtype)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol + tol16).all()
    if what != "query":
        assert (err[:128] <= tol16[:128]).all()  # the tiles before that are the type's


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [1, 3, 200])
def test_values_at_the_types_limit(gpu, dtype, n):
    """Values up to the largest number of the type, both signs, in both forms: what is finite stays finite."""
    cache = make(D=64, H=1, HQ=2, dtype=dtype)
    seqs = cache.add(1)
    big = torch.finfo(dtype).max
    k = rows((n, 1, 64), dtype, 1)
    v = torch.where(rows((n, 1, 64), torch.float32, 2) > 0, big, -big).to(dtype)
    v[:, :, 5] = 0.5 * big
    cache.store(0, cache.extend(seqs, [n]), k, v)
    m = Mirror()
    m.store(seqs[0], 0, k.cpu(), v.cpu())
    for count in {1, n}:
        q = rows((count, 2, 64), dtype, 3)
        got = cache.attend(0, cache.span(seqs, [n - count], [count]), q, scaling=0.125)
        want, tol = attention(q.cpu(), *m.rows[seqs[0]], n - count, 0.125, dtype if dtype == FP and count == 1 else BF)
        inside = want.abs() + tol < big
        assert inside.any() and ((got.cpu().double() - want).abs() <= tol)[inside].all()


@pytest.mark.parametrize("count", [1, 40])
def test_what_a_page_held_before(gpu, count):
    """A page taken again holds its last sequence's tokens behind the new one's, here values at the type's limit."""
    cache = make(D=64, H=1, HQ=4, pages=2)
    old, = cache.add()
    big = torch.full((64, 1, 64), torch.finfo(BF).max, dtype=BF, device="cuda")
    big[:, :, ::2] *= -1
    cache.store(0, cache.extend([old], [64]), rows((64, 1, 64), BF, 1), big)
    cache.free([old])
    seqs, m = fill(cache, [40])
    check_attend(cache, m, seqs, [40 - count], [count])


def test_many_empty_sequences_beside_a_long_one(gpu):
    cache = make(D=64, H=2, HQ=4, pages=100, sequences=320, length=6400)
    seqs, m = fill(cache, [4000])
    empty = cache.add(300)
    check_attend(cache, m, seqs + empty, [3999] + [0] * 300, [1] + [0] * 300)
    check_attend(cache, m, empty + seqs, [0] * 300 + [3900], [0] * 300 + [100])


def test_attend_many_query_heads(gpu):
    """More query heads on a key/value head than a tile of the split form has rows."""
    cache = make(D=64, H=1, HQ=80)
    seqs, m = fill(cache, [300, 70])
    check_attend(cache, m, seqs, [299, 69], [1, 1])


def test_attend_many_sequences(gpu):
    lens = [(37 * i) % 150 + 1 for i in range(300)]
    cache = make(D=64, H=2, HQ=4, pages=1000, sequences=300, length=200)
    seqs, m = fill(cache, lens)
    check_attend(cache, m, seqs, [n - 1 for n in lens], [1] * 300)
    kids = cache.fork(seqs[:0])
    assert kids == []


@pytest.mark.parametrize("count", [1, 100])
def test_attend_strided_inputs_and_out(gpu, count):
    cache = make(D=128, HQ=8, H=2)
    seqs, m = fill(cache, [200, 150])
    span = cache.span(seqs, [200 - count, 150 - count], [count] * 2)
    fused = rows((2 * count, 8 + 2 + 2, 128), BF, 5)
    q = fused[:, :8]
    want = cache.attend(0, span, q.contiguous(), scaling=0.1, gate=q.contiguous())
    out = torch.empty_like(want)
    assert cache.attend(0, span, q, scaling=0.1, gate=q, out=out) is out
    assert torch.equal(out, want)
    odd = torch.empty(2 * count * 8 * 128 + 1, dtype=BF, device="cuda")[1:].view(2 * count, 8, 128)  # rows not aligned
    odd.copy_(q)
    assert torch.equal(cache.attend(0, span, odd, scaling=0.1, gate=odd), want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cache.attend(0, span, turned, scaling=0.1, gate=turned), want)
    # keys and values out of the fused tensor
    cache.store(0, span, fused[:, 8:10], fused[:, 10:])
    k, v = cache.read(0, span)
    wk, wv, _, _ = held(fused[:, 8:10].cpu(), fused[:, 10:].cpu())
    assert torch.equal(k.cpu(), wk.to(BF)) and torch.equal(v.cpu(), wv.to(BF))


def test_attend_is_the_same_every_time_and_alone(gpu):
    """No order of workgroups changes a result, and a sequence's result does not depend on its neighbours' values."""
    cache = make(D=128, HQ=8, H=2, pages=200)
    seqs, m = fill(cache, [3000, 40, 900])
    span = cache.span(seqs, [2999, 39, 800], [1, 1, 100])
    q = rows((102, 8, 128), BF, 5)
    first = cache.attend(0, span, q, scaling=0.1)
    for _ in range(3):
        assert torch.equal(cache.attend(0, span, q, scaling=0.1), first)
    q[0] = float("nan")
    assert torch.equal(cache.attend(0, span, q, scaling=0.1)[1:], first[1:])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("row", [0, 1, 40])  # of the split form, and at the front and in the middle of a tile
def test_a_query_that_is_not_finite_is_alone(gpu, row, bad):
    cache = make(D=128, H=2, HQ=8)
    seqs = cache.add(3)
    n = [200, 90, 300]
    cache.store(0, cache.extend(seqs, n), rows((sum(n), 2, 128), BF, 1), rows((sum(n), 2, 128), BF, 2))
    span = cache.span(seqs, [199, 0, 289], [1, 90, 11])
    q = rows((102, 8, 128), BF, 3)
    first = cache.attend(0, span, q, scaling=0.1)
    q[row] = bad
    got = cache.attend(0, span, q, scaling=0.1)
    keep = [i for i in range(102) if i != row]
    assert torch.equal(got[keep], first[keep]) and torch.isnan(got[row]).any()


# ---------------------------------------------------------------- the pages' life

def test_tokens_behind_the_last_stay(gpu):
    """A store writes its tokens alone: what a page holds before and behind them stays."""
    cache = make(D=128)
    seqs, m = fill(cache, [64])
    span = cache.span(seqs, [20], [9])
    k, v = (rows((9, 2, 128), BF, 50 + i) for i in (0, 1))
    cache.store(0, span, k, v)
    new = held(k.cpu(), v.cpu())
    for x, n in zip(m.rows[seqs[0]], new):
        x[20:29] = n
    check_held(cache, m, seqs)


def test_fork_copies_on_write(gpu):
    cache = make(D=128, layers=3, pages=20)
    parent = cache.add()
    data = {}
    span = cache.extend(parent, [100])
    for layer in range(3):
        data[layer] = [rows((100, 2, 128), BF, 10 * layer + i) for i in (0, 1)]
        cache.store(layer, span, *data[layer])
    kids = cache.fork(parent * 3)
    assert cache.pages_in_use == 2 and cache.lengths(kids) == [100] * 3
    span = cache.extend(kids)
    assert cache.pages_in_use == 5
    table = cache.page_table(span)
    assert len(set(table[:, 0].tolist())) == 1 and len(set(table[:, 1].tolist())) == 3 and not table[:, 2:].any()
    new = {}
    for layer in range(3):
        new[layer] = [rows((3, 2, 128), BF, 100 + 10 * layer + i) for i in (0, 1)]
        cache.store(layer, span, *new[layer])
    for layer in range(3):
        m = Mirror()
        m.store(parent[0], 0, *(x.cpu() for x in data[layer]))
        for i, s in enumerate(kids):
            m.store(s, 0, *(torch.cat((x, y[i:i + 1])).cpu() for x, y in zip(data[layer], new[layer])))
        check_held(cache, m, parent + kids, layer)
        check_attend(cache, m, parent + kids, [99, 100, 100, 100], [1] * 4, layer=layer)
    # the parent's page is its own again once it alone holds it: nothing is copied
    cache.extend(parent)
    assert cache.pages_in_use == 5
    cache.free(kids)
    assert cache.pages_in_use == 2
    cache.free(parent)
    assert cache.pages_in_use == 0 and not cache.table.any()


def test_the_last_holder_does_not_copy(gpu):
    cache = make(D=64, H=1, HQ=1, pages=4)
    seqs, m = fill(cache, [30])
    kids = cache.fork(seqs * 2)
    cache.free(seqs)
    cache.extend(kids)  # one copies, the other keeps the page
    assert cache.pages_in_use == 2
    for s in kids:
        k, v = cache.read(0, cache.span([s], [0], [30]))
        assert torch.equal(k.cpu(), m.rows[seqs[0]][0].to(BF)) and torch.equal(v.cpu(), m.rows[seqs[0]][1].to(BF))


def test_random_life(gpu):
    """Every call in any order; after each, all sequences hold and answer what they should."""
    r = random.Random(5)
    cache = make(D=64, H=2, HQ=4, layers=2, pages=40, sequences=8, length=500)
    mirrors, live = [Mirror(), Mirror()], []
    for step in range(60):
        act = r.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact", "resize", "attend"])
        if act == "add" and len(live) < 7:
            s, = cache.add()
            live.append(s)
            for m in mirrors:
                m.store(s, 0, torch.zeros(0, 2, 64), torch.zeros(0, 2, 64))
        elif act == "extend" and live:
            chosen = r.sample(live, r.randint(1, len(live)))
            counts = [r.choice([0, 1, 1, 5, 64, 90]) for _ in chosen]
            lens = cache.lengths(chosen)
            if any(a + b > 500 for a, b in zip(lens, counts)) or cache.free_pages < sum(b // 64 + 2 for b in counts):
                continue
            span = cache.extend(chosen, counts)
            for layer, m in enumerate(mirrors):
                k, v = (rows((span.tokens, 2, 64), BF, 1000 + 4 * step + 2 * layer + i) for i in (0, 1))
                cache.store(layer, span, k, v)
                at = 0
                for s, st, n in zip(chosen, span.starts, counts):
                    m.store(s, st, k[at:at + n].cpu(), v[at:at + n].cpu()) if n else None
                    at += n
        elif act == "fork" and live and len(live) < 7:
            p = r.choice(live)
            s, = cache.fork([p])
            live.append(s)
            for m in mirrors:
                m.rows[s] = [x.clone() for x in m.rows[p]]
        elif act == "truncate" and live:
            s = r.choice(live)
            n = r.randint(0, cache.lengths([s])[0])
            cache.truncate(s, n)
            for m in mirrors:
                m.rows[s] = [x[:n] for x in m.rows[s]]
        elif act == "free" and len(live) > 2:
            s = live.pop(r.randrange(len(live)))
            cache.free([s])
        elif act == "compact":
            n = cache.compact()
            assert n == cache.pages_in_use and int(cache.table.max()) < max(1, n)
        elif act == "resize":
            cache.resize(max(1, cache.pages_in_use) + r.randint(8, 30))
            assert int(cache.table.max()) < max(1, cache.pages_in_use)
        for layer, m in enumerate(mirrors):
            check_held(cache, m, live, layer)
        some = [s for s in live if m.rows[s][0].shape[0] > 0]
        if some:
            lens = cache.lengths(some)
            check_attend(cache, mirrors[1], some, [n - min(n, 3) for n in lens], [min(n, 3) for n in lens], layer=1)


def test_pool_beyond_four_gigabytes(gpu):
    """Page offsets past 32 bits: the pages at the end of a large pool."""
    H, D, layers = 8, 256, 2
    pages = (5 << 30) // (H * 72 * D) // layers * layers + 2  # each layer over 5 GiB
    cache = make(D=D, H=H, HQ=8, layers=layers, pages=pages, length=64 * 40000, sequences=4)
    first, = cache.add()
    cache.extend([first], [64 * (pages - 5)])  # takes all but the last pages: three, one and one copy follow
    seqs, m = fill(cache, [130, 60], layer=1)
    assert int(cache.page_table(cache.span(seqs, [0, 0], [1, 1])).max()) >= pages - 5
    check_held(cache, m, seqs, 1)
    check_attend(cache, m, seqs, [129, 0], [1, 60], layer=1)
    kid = cache.fork([seqs[1]])
    m.rows[kid[0]] = m.rows[seqs[1]]
    cache.extend(kid)
    check_held(cache, m, kid, 1)
    cache.free([first])
    cache.compact()
    check_held(cache, m, seqs + kid, 1)
    cache.resize(8)
    check_held(cache, m, seqs + kid, 1)


# ---------------------------------------------------------------- together: a step, captured

def test_captured_steps_equal_eager_ones(gpu):
    """store + attend of two layers captured once; the span is filled again before every replay."""
    def run(captured):
        cache = make(D=128, HQ=8, H=2, layers=2, pages=100, sequences=8, length=2000)
        seqs = cache.add(3)
        span = cache.extend(seqs, [700, 62, 5])
        for layer in range(2):
            cache.store(layer, span, *(rows((767, 2, 128), BF, 2 * layer + i) for i in (0, 1)))
        k, v, q = (torch.zeros((3, n, 128), dtype=BF, device="cuda") for n in (2, 2, 8))
        out = [torch.zeros((3, 8, 128), dtype=BF, device="cuda") for _ in range(2)]

        def step(span):
            for layer in range(2):
                cache.store(layer, span, k, v)
                cache.attend(layer, span, q, scaling=0.1, out=out[layer])

        seen, span, graph = [], None, None
        for i in range(9):
            if i == 4:  # the batch changes under the captured step
                kid, = cache.fork([seqs[0]])
                cache.free([seqs[0]])
                seqs[0] = kid
                cache.compact()
            span = cache.extend(seqs, span=span)
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
            seen.append(torch.stack(out).clone())
        return seen

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


def test_counting_calls_are_refused_in_a_capture(gpu):
    cache = make(D=64, H=1, HQ=1)
    seqs, _ = fill(cache, [3])
    torch.cuda.synchronize()
    calls = [lambda: cache.extend(seqs), lambda: cache.fork(seqs), lambda: cache.free(seqs), lambda: cache.truncate(seqs[0], 1),
             lambda: cache.compact(), lambda: cache.resize(80), lambda: cache.span(seqs, [0], [1])]
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x += 1
        for call in calls:
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert cache.lengths(seqs) == [3]


def test_another_stream(gpu):
    cache = make(D=128, HQ=8, H=2)
    seqs, m = fill(cache, [150])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_attend(cache, m, seqs, [149], [1])
        check_attend(cache, m, seqs, [0], [150])
        cache.resize(40)
        check_held(cache, m, seqs)
    torch.cuda.current_stream().wait_stream(side)
    check_held(cache, m, seqs)


# ---------------------------------------------------------------- refusals

def test_refusals_leave_the_cache_as_it_was(gpu):
    cache = make(D=64, H=2, HQ=4, pages=4, sequences=3, length=200)
    seqs, m = fill(cache, [100, 30])
    free = cache.free_pages
    other = make(D=64, H=2, HQ=4)
    span = cache.span(seqs, [0, 0], [1, 1])
    q = torch.zeros((2, 4, 64), dtype=BF, device="cuda")
    kv = torch.zeros((2, 2, 64), dtype=BF, device="cuda")
    for call, error, match in [
        (lambda: cache.extend(seqs, [10, 64 * 3]), RuntimeError, "max_length|pages"),
        (lambda: cache.extend(seqs, [64, 100]), RuntimeError, "pages needed"),
        (lambda: cache.extend(seqs, [1]), ValueError, "counts"),
        (lambda: cache.extend(seqs, [1, -1]), ValueError, "negative"),
        (lambda: cache.extend([seqs[0], seqs[0]]), RuntimeError, "twice"),
        (lambda: cache.extend([2]), RuntimeError, "not in use"),
        (lambda: cache.extend([-1]), RuntimeError, "not in use"),
        (lambda: cache.extend([1 << 40]), ValueError, "range"),
        (lambda: cache.extend([0.5]), TypeError, "integer"),
        (lambda: cache.extend(seqs, [1, 1 << 62]), RuntimeError, "max_length"),
        (lambda: cache.extend(seqs, (1, 1 << 70)), ValueError, "range"),
        (lambda: cache.fork([-1]), RuntimeError, "not in use"),
        (lambda: cache.free([1 << 40]), ValueError, "range"),
        (lambda: cache.span(seqs, [0, 30], [101, 1]), RuntimeError, "holds"),
        (lambda: cache.span(seqs, [-1, 0], [1, 1]), RuntimeError, "holds"),
        (lambda: cache.span(seqs, [0], [1]), ValueError, "starts"),
        (lambda: cache.add(2), RuntimeError, "free"),
        (lambda: cache.fork(seqs), RuntimeError, "free"),
        (lambda: cache.fork([2]), RuntimeError, "not in use"),
        (lambda: cache.free([seqs[0], 2]), RuntimeError, "not in use"),
        (lambda: cache.free([seqs[0]] * 2), RuntimeError, "twice"),
        (lambda: cache.truncate(seqs[0], 101), RuntimeError, "length"),
        (lambda: cache.resize(2), RuntimeError, "in use"),
        (lambda: cache.store(1, span, kv, kv), IndexError, "layer"),
        (lambda: cache.store(0, span, kv.half(), kv), ValueError, "keys"),
        (lambda: cache.store(0, span, kv, kv[:1]), ValueError, "values"),
        (lambda: cache.store(0, span, kv.cpu(), kv), RuntimeError, "keys must be on"),
        (lambda: cache.attend(0, span, q[:, :2], scaling=1.0), ValueError, "query"),
        (lambda: cache.attend(0, span, q, scaling=0.0), ValueError, "scaling"),
        (lambda: cache.attend(0, span, q, scaling=float("nan")), ValueError, "scaling"),
        (lambda: cache.attend(0, span, q, scaling=1.0, gate=q[:1]), ValueError, "gate"),
        (lambda: cache.attend(0, span, q, scaling=1.0, out=q.transpose(0, 1)), ValueError, "out"),
        (lambda: other.attend(0, span, q, scaling=1.0), ValueError, "another cache"),
        (lambda: other.extend(other.add(2), span=span), ValueError, "another cache"),
        (lambda: cache.extend(seqs[:1], span=span), ValueError, "same counts"),
    ]:
        with pytest.raises(error, match=match):
            call()
    assert cache.free_pages == free and cache.lengths(seqs) == [100, 30]
    check_held(cache, m, seqs)
    cache.truncate(seqs[0], 0)
    with pytest.raises(RuntimeError, match="holds 0 tokens"):
        cache.attend(0, span, q, scaling=1.0)
    cache.free([seqs[1]])
    with pytest.raises(RuntimeError, match="holds 0 tokens|not in use"):
        cache.read(0, span)


def test_a_span_ends_with_its_sequences(gpu):
    """Another sequence in the same row is none of the span's."""
    cache = make(D=64, H=1, HQ=2)
    seqs = cache.add(2)
    cache.extend(seqs, [60, 30])
    span = cache.span(seqs, [0, 0], [60, 30])
    cache.free([seqs[1]])
    with pytest.raises(RuntimeError, match="not in use"):
        cache.read(0, span)
    again, = cache.add()
    cache.extend([again], [30])
    cache.truncate(seqs[0], 0)
    cache.extend([seqs[0]], [60])
    assert again == seqs[1]
    with pytest.raises(RuntimeError, match="not in use"):
        cache.read(0, span)


def test_sequences_that_share_a_page_are_not_stored_together(gpu):
    cache = make(D=64, H=2, HQ=4)
    seqs, m = fill(cache, [100])
    child, = cache.fork(seqs)
    m.rows[child] = m.rows[seqs[0]]
    k = rows((8, 2, 64), BF, 5)
    both = cache.span([seqs[0], child], [64, 68], [4, 4])
    with pytest.raises(RuntimeError, match="share a page"):
        cache.store(0, both, k, k)
    check_held(cache, m, [seqs[0], child])
    check_attend(cache, m, [seqs[0], child], [64, 68], [4, 4])
    # one of them alone, both in pages of their own, and new tokens of both
    cache.store(0, cache.span([child], [68], [4]), k[:4], k[:4])
    cache.store(0, cache.span([seqs[0], child], [0, 68], [4, 4]), k, k)
    cache.store(0, cache.extend([seqs[0], child], [4, 4]), k, k)


def test_no_memory_for_a_span(gpu, monkeypatch):
    """An extend whose span cannot be allocated leaves the sequences as they were."""
    np = pytest.importorskip("numpy")
    cache = make(D=64, H=2, HQ=4, pages=8)
    seqs, m = fill(cache, [100, 64])
    free = cache.free_pages

    def nothing(*args, **kwargs):
        raise torch.OutOfMemoryError("none left")
    with monkeypatch.context() as patch:
        patch.setattr(torch, "empty", nothing)
        with pytest.raises(torch.OutOfMemoryError):
            cache.extend(np.array(seqs), [30, 1])
    assert cache.lengths(seqs) == [100, 64] and cache.free_pages == free
    check_held(cache, m, seqs)
    check_attend(cache, m, seqs, [99, 0], [1, 64])


def test_sequences_by_other_integers(gpu):
    """Lists, tuples, arrays and numpy integers name sequences alike; the host module takes plain lists alone."""
    np = pytest.importorskip("numpy")
    cache = make(D=64, H=2, HQ=4, length=100)
    seqs, m = fill(cache, [20, 30])
    for names in (seqs, tuple(seqs), np.array(seqs), [np.int64(s) for s in seqs], torch.tensor(seqs)):
        span = cache.extend(names, np.array([1, 2]))
        assert span.seqs == seqs and span.counts == [1, 2] and span.tokens == 3
        kids = cache.fork(names)
        cache.free(np.array(kids))
        assert list(cache.span(names, [0, 0], (1, 1)).rows.cpu()) == seqs
    assert cache.lengths(seqs) == [25, 40]


def test_empty_spans(gpu):
    cache = make(D=64, H=2, HQ=4)
    for span in (cache.extend([], []), cache.extend(cache.add(2), [0, 0])):
        q = torch.zeros((0, 4, 64), dtype=BF, device="cuda")
        assert cache.attend(0, span, q, scaling=1.0).shape == (0, 4, 64)
        cache.store(0, span, q[:, :2], q[:, :2])
        assert cache.read(0, span)[0].shape == (0, 2, 64)
        assert cache.page_table(span).shape[0] == len(span.seqs)


def test_threads_that_share_a_cache(gpu):
    """Sequences that come, grow and go from several host threads, all on one stream."""
    cache = make(D=64, H=2, HQ=4, pages=64, sequences=16)

    def life(seed):
        for turn in range(10):
            n = 30 + 17 * ((seed + turn) % 8)
            seqs = cache.add(2)
            k, v = rows((2 * n, 2, 64), BF, seed), rows((2 * n, 2, 64), BF, seed + 1)
            cache.store(0, cache.extend(seqs, [n, n]), k, v)
            m = Mirror()
            for i, s in enumerate(seqs):
                m.store(s, 0, k[n * i:n * i + n].cpu(), v[n * i:n * i + n].cpu())
            check_held(cache, m, seqs)
            check_attend(cache, m, seqs, [n - 1, 0], [1, n])
            cache.free(seqs)
        return True

    with ThreadPoolExecutor(4) as pool:
        assert all(f.result() for f in [pool.submit(life, 10 * i) for i in range(4)])
    assert cache.pages_in_use == 0
