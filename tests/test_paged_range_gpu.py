"""PagedInt4Cache's attention in tiles at the ends of what 16-bit operands hold: small and large queries, keys and values,
and pages that held other tokens before.  Against the plain 64-bit counterpart."""

import pytest
import torch

from _paged import Mirror, attention
from test_paged_cache_gpu import BF, FP, make, rows

pytestmark = pytest.mark.gpu


def stored(cache, k, v):
    """One sequence of these tokens (values of the cache's type, on the host) -> (sequences, its rows as held)."""
    seqs = cache.add()
    cache.store(0, cache.extend(seqs, [k.shape[0]]), k.cuda(), v.cuda())
    m = Mirror()
    m.store(0, 0, k, v)
    return seqs, m.rows[0]


def check(got, q, held, start, scaling, dtype):
    want, tol = attention(q, *held, start, scaling, dtype)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


# ---------------------------------------------------------------- what no row sees

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("what", ["key", "value", "tiny value"])
def test_tokens_that_a_page_held_before(gpu, D, dtype, what):
    """What stands behind a sequence's end is nothing to its answers, bit by bit: neither tokens of another sequence that
    had the page nor its own that are forgotten or not yet seen."""
    factor = {"key": 2.0 ** 9, "value": 2.0 ** 12, "tiny value": 2.0 ** -22}[what]
    k, v, q = (rows((n, h, D), dtype, i, "cpu") for i, n, h in ((1, 100, 2), (2, 100, 2), (3, 100, 4)))
    k1, v1 = (rows((128, 2, D), torch.float32, i, "cpu") for i in (4, 5))
    k1, v1 = ((k1 * factor).to(dtype), v1.to(dtype)) if what == "key" else (k1.to(dtype), (v1 * factor).to(dtype))

    def answers(before):
        cache = make(D=D, H=2, HQ=4, dtype=dtype, pages=2)
        if before == "another":
            old, _ = stored(cache, k1, v1)
            cache.free(old)
        elif before == "forgotten":
            seqs = cache.add()
            cache.store(0, cache.extend(seqs, [128]), torch.cat((k, k1[100:])).cuda(), torch.cat((v, v1[100:])).cuda())
            cache.truncate(seqs[0], 100)
        elif before == "later":
            seqs = cache.add()
            cache.store(0, cache.extend(seqs, [128]), torch.cat((k, k1[100:])).cuda(), torch.cat((v, v1[100:])).cuda())
        if before in (None, "another"):
            seqs, _ = stored(cache, k, v)
        return cache.attend(0, cache.span(seqs, [0], [100]), q.cuda(), scaling=D ** -0.5)

    first = answers(None)
    for before in ("another", "forgotten", "later"):
        assert torch.equal(answers(before), first), before


@pytest.mark.parametrize("D", [64, 128])
def test_tokens_that_a_page_held_before_in_tiles_of_256(gpu, D):
    lens = [70 + 5 * i % 60 for i in range(32)]
    k, v, q = (rows((sum(lens), h, D), FP, i) for i, h in ((1, 8), (2, 8), (3, 32)))

    def answers(before):
        cache = make(D=D, H=8, HQ=32, dtype=FP, pages=96, sequences=32)
        if before:
            old = cache.add(32)
            big = (rows((32 * 192, 8, D), torch.float32, 4) * 2.0 ** 9).to(FP)
            cache.store(0, cache.extend(old, [192] * 32), big, big)
            cache.free(old)
        span = cache.extend(cache.add(32), lens)
        assert span._c.tile_rows == 256
        cache.store(0, span, k, v)
        return cache.attend(0, span, q, scaling=D ** -0.5)

    assert torch.equal(answers(True), answers(False))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("count", [1, 20, 100])
def test_tokens_that_are_not_finite_and_that_no_row_sees(gpu, D, dtype, count):
    """NaN and infinities of another sequence behind the end, and of its own later tokens: bit by bit as without them."""
    k, v, q = (rows((n, h, D), dtype, i, "cpu") for i, n, h in ((1, 128, 1), (2, 128, 1), (3, count, 4)))

    def answers(before):
        cache = make(D=D, H=1, HQ=4, dtype=dtype, pages=2)
        bad = torch.full((128, 1, D), float("nan"), dtype=dtype)
        if before == "another":
            old, _ = stored(cache, bad, -bad)
            cache.free(old)
        if before == "later":
            bad[:] = float("inf")
            seqs, _ = stored(cache, torch.cat((k[:110], bad[110:])), torch.cat((v[:110], bad[110:])))
        else:
            seqs, _ = stored(cache, k[:110], v[:110])
        return cache.attend(0, cache.span(seqs, [110 - count], [count]), q.cuda(), scaling=D ** -0.5)

    first = answers(None)
    assert torch.isfinite(first).all()
    for before in ("another", "later"):
        assert torch.equal(answers(before), first), before


# ---------------------------------------------------------------- queries

SIZES = [(BF, 2.0 ** -30), (BF, 2.0 ** -100), (BF, 2.0 ** 40), (FP, 2.0 ** -12), (FP, 2.0 ** 11)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,factor", SIZES)
@pytest.mark.parametrize("count", [1, 100])
def test_queries_of_any_size(gpu, D, dtype, factor, count):
    """A query's size is taken back by the scaling, in both forms, to the type's own tolerance."""
    cache = make(D=D, H=1, HQ=2, dtype=dtype)
    seqs, held = stored(cache, *(rows((200, 1, D), dtype, i, "cpu") for i in (1, 2)))
    q = (rows((count, 2, D), torch.float32, 3, "cpu") * factor).to(dtype)
    scaling = D ** -0.5 / factor
    got = cache.attend(0, cache.span(seqs, [200 - count], [count]), q.cuda(), scaling=scaling)
    check(got, q, held, 200 - count, scaling, dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_a_querys_size_is_its_own(gpu, dtype):
    """A row far larger or smaller than the others, or all zeros, changes no other row's bits."""
    cache = make(D=128, H=2, HQ=4, dtype=dtype)
    seqs, held = stored(cache, *(rows((200, 2, 128), dtype, i, "cpu") for i in (1, 2)))
    q = rows((200, 4, 128), dtype, 3, "cpu")
    span = cache.span(seqs, [0], [200])
    first = cache.attend(0, span, q.cuda(), scaling=0.1)
    keep = [i for i in range(200) if i != 70]
    for factor in (0.0, 2.0 ** -14, 2.0 ** 11):
        p = q.clone()
        p[70] *= factor
        got = cache.attend(0, span, p.cuda(), scaling=0.1)
        assert torch.equal(got[keep], first[keep]), factor
        check(got, p, held, 0, 0.1, dtype)


def test_scalings_at_the_ends(gpu):
    """Scalings that leave fp32's normal numbers once the query's size is taken into them: flat or peaked, no NaN."""
    cache = make(D=64, H=1, HQ=2)
    seqs, held = stored(cache, *(rows((150, 1, 64), BF, i, "cpu") for i in (1, 2)))
    for factor, scaling in ((2.0 ** -120, 1e-6), (2.0 ** -126, 1e-30), (2.0 ** 100, 2.0 ** -103), (2.0 ** -97, 2.0 ** 94), (0.0, 1e29)):
        q = (rows((150, 2, 64), torch.float32, 3, "cpu") * factor).to(BF)
        got = cache.attend(0, cache.span(seqs, [0], [150]), q.cuda(), scaling=scaling)
        check(got, q, held, 0, scaling, BF)


# ---------------------------------------------------------------- keys

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,factor,as_type", [(BF, 2.0 ** -16, BF), (BF, 2.0 ** -24, BF), (BF, 2.0 ** -60, BF), (FP, 2.0 ** -12, FP),
                                                  (FP, 2.0 ** -20, BF)])
@pytest.mark.parametrize("count", [1, 100])
def test_keys_of_any_size(gpu, D, dtype, factor, as_type, count):
    """Small keys under a large scaling.  Where fp16 does not hold them, the tiles go on in bf16, to its tolerance."""
    cache = make(D=D, H=1, HQ=2, dtype=dtype)
    k = (rows((200, 1, D), torch.float32, 1, "cpu") * factor).to(dtype)
    seqs, held = stored(cache, k, rows((200, 1, D), dtype, 2, "cpu"))
    q = rows((count, 2, D), dtype, 3, "cpu")
    scaling = D ** -0.5 / factor
    got = cache.attend(0, cache.span(seqs, [200 - count], [count]), q.cuda(), scaling=scaling)
    check(got, q, held, 200 - count, scaling, as_type)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_keys_with_large_channels(gpu, D, dtype):
    """Channels of keys in the hundreds, as biased projections make them: the type's own tolerance."""
    cache = make(D=D, H=2, HQ=4, dtype=dtype)
    k = (rows((200, 2, D), torch.float32, 1, "cpu") * 8).to(dtype)
    seqs, held = stored(cache, k, rows((200, 2, D), dtype, 2, "cpu"))
    assert 16 < held[2].max() < 64
    q = rows((200, 4, D), dtype, 3, "cpu")
    for scaling in (D ** -0.5 / 8, 1e-5):  # and with scores near 0, whose errors do not hide those of the values
        got = cache.attend(0, cache.span(seqs, [0], [200]), q.cuda(), scaling=scaling)
        check(got, q, held, 0, scaling, dtype)


@pytest.mark.parametrize("dtype,factor", [(BF, 2.0 ** -26), (BF, 2.0 ** -20), (FP, 2.0 ** -20)])
def test_a_small_group_that_alone_counts(gpu, dtype, factor):
    """Queries that are zero where the keys are large: the scores come from a group of small keys alone."""
    cache = make(D=128, H=1, HQ=2, dtype=dtype)
    k = rows((200, 1, 128), torch.float32, 1, "cpu")
    k[..., 64:] *= factor
    k = k.to(dtype)
    seqs, held = stored(cache, k, rows((200, 1, 128), dtype, 2, "cpu"))
    q = rows((200, 2, 128), dtype, 3, "cpu")
    q[..., :64] = 0
    got = cache.attend(0, cache.span(seqs, [0], [200]), q.cuda(), scaling=0.125 / factor)
    check(got, q, held, 0, 0.125 / factor, BF)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [128, 256])
def test_a_small_group_beside_ordinary_ones(gpu, D, dtype):
    """Channels that are nearly dead cost no precision under an ordinary scaling: the type's own tolerance."""
    cache = make(D=D, H=1, HQ=2, dtype=dtype)
    k = rows((200, 1, D), torch.float32, 1, "cpu")
    k[..., 64:128] *= 2.0 ** -21
    k = k.to(dtype)
    seqs, held = stored(cache, k, rows((200, 1, D), dtype, 2, "cpu"))
    q = rows((200, 2, D), dtype, 3, "cpu")
    got = cache.attend(0, cache.span(seqs, [0], [200]), q.cuda(), scaling=D ** -0.5)
    check(got, q, held, 0, D ** -0.5, dtype)


# ---------------------------------------------------------------- values

@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_whose_scale_fp16_rounds(gpu, D):
    """Values whose scale, 65.5 * 2^-24, lies between two of fp16's subnormal numbers: the first token's answer is its
    value, to half a step of bf16 at most."""
    cache = make(D=D, H=1, HQ=4, dtype=FP)
    g = torch.Generator().manual_seed(1)
    units = 1572 + 2 * (32.74 * torch.randint(0, 16, (100, 1, D), generator=g)).round()
    units[..., ::64], units[..., 1::64] = 1572, 2554
    v = (units * 2.0 ** -24).to(FP)
    seqs, held = stored(cache, rows((100, 1, D), FP, 2, "cpu"), v)
    assert (held[3] == 65.5 * 2.0 ** -24).all()
    got = cache.attend(0, cache.span(seqs, [0], [100]), rows((100, 4, D), FP, 3).cuda(), scaling=D ** -0.5)
    want = held[1][0].expand(4, D)
    assert ((got[0].cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * want.abs() + 2.0 ** -25).all()
