"""The linear-attention operators on the GPU against plain 64-bit counterparts on the CPU (tests/_linear.py)."""

import pytest
import torch

import _linear as plain
from anna_amd import linear_attention as la

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def nothing_cached():
    """The large tensors' segments go back to the device, so that nobody's lasting tensors come to lie in them."""
    yield
    torch.cuda.empty_cache()


BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
STEPS = 12  # sequences of more tokens go in chunks


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def delta_case(seed, counts, HK, HV, DK, DV, dtype, raw, slots=None, pool=None):
    n, tokens = len(counts), sum(counts)
    pool = pool or n + 2
    q, k = randn(seed, tokens, HK, DK).to(dtype), randn(seed + 1, tokens, HK, DK).to(dtype)
    v, state = randn(seed + 2, tokens, HV, DV).to(dtype), 0.5 * randn(seed + 3, pool, HV, DK, DV)
    a, b = randn(seed + 4, tokens, HV), randn(seed + 5, tokens, HV)
    a_log, dt_bias = randn(seed + 6, HV), randn(seed + 7, HV) - 3
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    slots = slots or order[:n]
    if raw:
        return dict(q=q, k=k, v=v, decay=a.to(dtype), beta=b.to(dtype), a_log=a_log, dt_bias=dt_bias, state=state, slots=slots)
    g, beta = plain.gates(a, b, a_log, dt_bias)
    return dict(q=q, k=k, v=v, decay=g.float(), beta=beta.float(), a_log=None, dt_bias=None, state=state, slots=slots)


def run_delta(gpu, c, counts, fresh, scaling, normalize=True, **kw):
    def put(t):
        return None if t is None else t.to(gpu)

    state = put(c["state"])
    span = la.StateSpan(c["slots"], counts, fresh=fresh, device=gpu)
    out = la.gated_delta_rule(put(c["q"]), put(c["k"]), put(c["v"]), put(c["decay"]), put(c["beta"]), state, span, scaling=scaling,
                              normalize=normalize, a_log=put(c["a_log"]), dt_bias=put(c["dt_bias"]), **kw)
    return out.cpu(), state.cpu()


def check_delta(c, counts, fresh, scaling, out, state, normalize=True):
    g, beta = plain.gates(c["decay"], c["beta"], c["a_log"], c["dt_bias"])
    at, named = 0, set()
    for i, (slot, n) in enumerate(zip(c["slots"], counts)):
        rows = slice(at, at + n)
        at += n
        if slot < 0:
            assert (out[rows] == 0).all()
            continue
        if n == 0:
            continue
        named.add(slot)
        S0 = torch.zeros_like(c["state"][slot]) if fresh[i] else c["state"][slot]
        want, S, sums, errors, E, eps = plain.delta_rule(c["q"][rows], c["k"][rows], c["v"][rows], g[rows], beta[rows], S0, scaling,
                                                         normalize, chunked=n > STEPS)
        tol = plain.delta_tolerance(want, sums, errors, eps, out.dtype, scaling, n > STEPS)
        off = (out[rows].double() - want).abs()
        assert (off <= tol).all(), (i, n, float((off / tol).max()))
        err = (state[slot].double() - S).norm(dim=1)
        assert (err <= E).all(), (i, n, float((err / E).max()))
    for slot in range(state.shape[0]):
        if slot not in named:
            assert torch.equal(state[slot], c["state"][slot])


DELTA = [
    # counts, fresh, key heads, value heads, key dim, value dim, dtype, raw gates
    ([1], [False], 2, 4, 128, 128, BF, True),
    ([1, 1, 1], [False, True, False], 1, 3, 64, 32, HF, False),
    ([1, 0, 12, 2, 5], [False, False, True, True, False], 2, 2, 128, 96, BF, False),
    ([3, 7, 1], [False, False, True], 2, 6, 64, 256, HF, True),
    ([13], [False], 1, 1, 64, 32, BF, True),
    ([63, 64, 65], [False, True, False], 2, 4, 64, 64, BF, True),
    ([200, 1, 0, 12, 128, 13], [True, False, True, False, False, True], 2, 4, 128, 128, BF, True),
    ([129, 30], [False, False], 1, 2, 128, 256, HF, False),
    ([300], [True], 1, 1, 128, 96, HF, True),
    ([70, 64], [False, True], 3, 3, 128, 32, BF, False),
]


@pytest.mark.parametrize("case", DELTA, ids=[f"{c[0]}x{c[2]}-{c[3]}x{c[4]}-{c[5]}" for c in DELTA])
def test_delta_rule(gpu, case):
    counts, fresh, HK, HV, DK, DV, dtype, raw = case
    c = delta_case(len(counts) * 7 + sum(counts), counts, HK, HV, DK, DV, dtype, raw)
    for i, f in enumerate(fresh):
        if f and counts[i]:
            c["state"][c["slots"][i]] = float("nan")  # what was there has no say
    out, state = run_delta(gpu, c, counts, fresh, DK ** -0.5)
    assert torch.isfinite(out).all()
    check_delta(c, counts, fresh, DK ** -0.5, out, state)


# Workgroups of the chunks' form take 1, 2 or 4 groups of 16 columns, by the work beside the longest sequence: chunks *
# value heads * columns / 16 against 256 of its chunks.  The cases above take 1, these 4, or 2 where 64 does not divide value_dim.
MANY = [
    (20, 2, 4, 128, 128, BF), (20, 4, 4, 64, 128, HF), (40, 2, 4, 128, 128, BF), (40, 1, 4, 128, 128, HF), (70, 2, 4, 64, 64, BF),
    (70, 1, 4, 64, 64, HF), (60, 2, 3 * 2, 128, 96, BF), (45, 2, 2, 128, 256, HF),
]


@pytest.mark.parametrize("case", MANY, ids=["x".join(map(str, c[:5])) + str(c[5])[6:] for c in MANY])
def test_delta_rule_of_many_sequences(gpu, case):
    n, HK, HV, DK, DV, dtype = case
    counts = [13 + (7 * i) % 90 if i % 9 else 1 for i in range(n)]
    fresh = [i % 3 == 0 for i in range(n)]
    c = delta_case(n, counts, HK, HV, DK, DV, dtype, True)
    c["slots"][5] = -1
    out, state = run_delta(gpu, c, counts, fresh, DK ** -0.5)
    check_delta(c, counts, fresh, DK ** -0.5, out, state)


@pytest.mark.parametrize("case", [(6, 16, 128, 128, BF), (6, 16, 128, 128, HF), (7, 24, 128, 96, BF), (6, 16, 64, 256, HF)],
                         ids=lambda c: "x".join(map(str, c[:4])))
def test_delta_rule_of_several_long_sequences(gpu, case):
    n, HV, DK, DV, dtype = case
    counts = [250 + 17 * i for i in range(n)]
    fresh = [i % 2 == 0 for i in range(n)]
    c = delta_case(n, counts, 2, HV, DK, DV, dtype, True)
    out, state = run_delta(gpu, c, counts, fresh, DK ** -0.5)
    check_delta(c, counts, fresh, DK ** -0.5, out, state)


@pytest.mark.parametrize("n,DV", [(6, 128), (20, 128), (40, 96)])
def test_delta_rule_of_many_sequences_with_some_not_finite(gpu, n, DV):
    counts = [70] * n
    c = delta_case(n, counts, 2, 4, 128, DV, BF, False)
    c["v"][70 * 3 + 40, 2, 17] = float("nan")
    c["k"][70 * 5 + 66, 0, 3] = float("inf")
    out, state = run_delta(gpu, c, counts, [False] * n, 0.1)
    bad = {3: (40, [2]), 5: (66, [0, 1])}
    for i in bad:
        at, heads = bad[i]
        part = out[70 * i:70 * i + 70].float()
        assert torch.isfinite(part[:at]).all() and not torch.isfinite(part[at:, heads]).all(-1).any()
        rest = [h for h in range(4) if h not in heads]
        assert torch.isfinite(part[:, rest]).all() and torch.isfinite(state[c["slots"][i]][rest]).all()
    assert torch.isfinite(state[c["slots"][3]][2][:, [j for j in range(DV) if j != 17]]).all()
    # the tokens in front, and all other sequences
    c["v"][70 * 3 + 40:70 * 4] = 0
    c["k"][70 * 5 + 66:70 * 6] = 0
    c["k"][70 * 3 + 40:70 * 4] = 0
    clean, _ = run_delta(gpu, c, counts, [False] * n, 0.1)
    g, beta = c["decay"].double(), c["beta"].double()
    for i in range(n):
        m = bad[i][0] if i in bad else 70
        rows = slice(70 * i, 70 * i + m)
        want, S, sums, errors, E, eps = plain.delta_rule(c["q"][rows], c["k"][rows], c["v"][rows], g[rows], beta[rows], c["state"][c["slots"][i]], 0.1,
                                                         chunked=True)
        tol = plain.delta_tolerance(want, sums, errors, eps, BF, 0.1, True)
        for got in (out, clean):
            assert ((got[rows].double() - want).abs() <= tol).all(), i
        if i not in bad:
            assert ((state[c["slots"][i]].double() - S).norm(dim=1) <= E).all()


@pytest.mark.parametrize("counts", [[4, 1], [100, 20]])
def test_delta_rule_precision(gpu, counts):
    """The state is as exact as fp32 sums make it.  An operand split in two fp16 values is off by 2^-24 to 2^-23 of
    itself and a sum of 64 to 192 products by at most some 8 roundings of 2^-24 in the mean of their squares; with eight
    such steps in a row, independent of each other, the state's 2-norm is off by less than 2^-20."""
    c = delta_case(5, counts, 2, 4, 128, 128, HF, False)
    _, state = run_delta(gpu, c, counts, [False, False], 0.1)
    at = 0
    for slot, n in zip(c["slots"], counts):
        rows = slice(at, at + n)
        at += n
        _, S, *_ = plain.delta_rule(c["q"][rows], c["k"][rows], c["v"][rows], c["decay"][rows].double(), c["beta"][rows].double(),
                                    c["state"][slot], 0.1)
        assert float((state[slot].double() - S).norm() / S.norm()) < 2.0 ** -20


@pytest.mark.parametrize("counts", [[9], [90]])
def test_delta_rule_without_normalizing(gpu, counts):
    c = delta_case(11, counts, 2, 2, 64, 64, BF, False)
    c["k"] = (c["k"].float() / (1.01 * c["k"].float().norm(dim=-1, keepdim=True))).to(BF)  # shorter than 1
    out, state = run_delta(gpu, c, counts, [False], -0.7, normalize=False)
    g, beta = plain.gates(c["decay"], c["beta"])
    want, S, sums, errors, E, eps = plain.delta_rule(c["q"], c["k"], c["v"], g, beta, c["state"][c["slots"][0]], -0.7, False, counts[0] > STEPS)
    q_norm = float(c["q"].float().norm(dim=-1).max())
    tol = plain.delta_tolerance(want, sums, errors, eps, BF, 0.7 * q_norm, counts[0] > STEPS)
    assert ((out.double() - want).abs() <= tol).all()
    assert ((state[c["slots"][0]].double() - S).norm(dim=1) <= E).all()


@pytest.mark.parametrize("counts", [[10], [140]])
@pytest.mark.parametrize("what", ["reset", "never", "repeated keys", "zero keys", "no beta", "tiny", "large", "deep"])
def test_delta_rule_at_its_limits(gpu, what, counts):
    c = delta_case(21, counts, 1, 2, 64, 64, BF, False)
    n = counts[0]
    c["decay"], c["beta"] = c["decay"].clone(), c["beta"].clone()
    if what == "reset":  # some tokens forget all before them
        c["decay"][3::7] = -float("inf")
        c["decay"][5::11] = -1e30
    elif what == "never":
        c["decay"][:] = 0
        c["beta"][:] = 1
    elif what == "repeated keys":
        c["k"][:] = c["k"][:1]
        c["beta"][:] = 1
        c["decay"][:] = -1e-4
    elif what == "zero keys":
        c["k"][::3] = 0
        c["q"][::4] = 0
        c["v"][::5] = 0
    elif what == "no beta":
        c["beta"][::2] = 0
    elif what == "tiny":
        c["k"] = (c["k"].float() * 2.0 ** -100).to(BF)
        c["q"] = (c["q"].float() * 2.0 ** -120).to(BF)
        c["v"] = (c["v"].float() * 2.0 ** -60).to(BF)
    elif what == "large":
        c["k"] = (c["k"].float() * 2.0 ** 50).to(BF)
        c["q"] = (c["q"].float() * 2.0 ** 50).to(BF)
        c["v"] = (c["v"].float() * 2.0 ** 80).to(BF)
    elif what == "deep":
        c["decay"][:] = c["decay"] * 1000
    out, state = run_delta(gpu, c, counts, [False], 0.125)
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    check_delta(c, counts, [False], 0.125, out, state)


@pytest.mark.parametrize("counts", [[2, 8, 3], [20, 150, 14]])
@pytest.mark.parametrize("what", ["k", "v", "q", "beta", "decay", "v inf"])
def test_delta_rule_what_is_not_finite_reaches_nothing_before_it(gpu, what, counts):
    c = delta_case(31, counts, 2, 4, 64, 32, BF, False)
    at = counts[0] + counts[1] * 2 // 3
    bad = float("inf") if what == "v inf" else float("nan")
    name = {"beta": "beta", "decay": "decay"}.get(what, what[0])
    clean = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in c.items()}
    c[name] = c[name].clone()
    if c[name].dim() == 3:
        c[name][at, 1, 7] = bad  # of one head: key heads 1 of 2, value head 1 of 4
    else:
        c[name][at, 1] = bad
    out, state = run_delta(gpu, c, counts, [False] * 3, 0.125)
    heads = {"k": [2, 3], "q": [2, 3]}.get(name, [1])  # value heads that see it
    rest = [h for h in range(4) if h not in heads]
    # all that it does not reach is as the clean inputs make it, within the tolerance
    g, beta = plain.gates(clean["decay"], clean["beta"])
    first = 0
    for i, (slot, n) in enumerate(zip(c["slots"], counts)):
        want, S, sums, errors, E, eps = plain.delta_rule(*(clean[x][first:first + n] for x in "qkv"), g[first:first + n], beta[first:first + n],
                                                         clean["state"][slot], 0.125, chunked=n > STEPS)
        tol = plain.delta_tolerance(want, sums, errors, eps, BF, 0.125, n > STEPS)
        ok = torch.ones_like(want, dtype=torch.bool)
        if i == 1:
            ok[at - first:, heads] = False
        assert ((out[first:first + n].double() - want).abs() <= tol)[ok].all()
        whole = list(range(4)) if i != 1 or what == "q" else rest
        assert ((state[slot].double() - S).norm(dim=1) <= E)[whole].all()
        if i == 1:
            assert not torch.isfinite(out[at, heads].float()).all()
            if what != "q":
                assert not torch.isfinite(state[slot][heads]).all()
            if what.startswith("v"):  # one column of the state
                assert torch.isfinite(state[slot][1][:, [n for n in range(32) if n != 7]]).all()
        first += n


@pytest.mark.parametrize("normalize", [True, False])
def test_delta_rule_a_query_has_a_say_in_its_own_row_only(gpu, normalize):
    """Queries of very different size, one of them not finite, in one chunk: each row is as exact as alone."""
    counts = [100]
    c = delta_case(71, counts, 2, 4, 64, 64, HF, False)
    c["k"] = (c["k"].float() / (1.01 * c["k"].float().norm(dim=-1, keepdim=True))).to(HF)
    c["q"] = c["q"].to(BF)
    c["k"], c["v"] = c["k"].to(BF), c["v"].to(BF)
    c["k"] = (c["k"].float() * 0.99).to(BF)
    c["q"][::3] = (c["q"][::3].float() * 2.0 ** 60).to(BF)
    c["q"][1::3] = (c["q"][1::3].float() * 2.0 ** -40).to(BF)
    if not normalize:
        c["q"][31, 0, 5] = float("inf")
    else:
        c["q"][31, 0, 5] = float("nan")
    out, state = run_delta(gpu, c, counts, [False], 0.1, normalize=normalize)
    g, beta = plain.gates(c["decay"], c["beta"])
    clean = c["q"].clone()
    clean[31, 0] = 0
    want, S, sums, errors, E, eps = plain.delta_rule(clean, c["k"], c["v"], g, beta, c["state"][c["slots"][0]], 0.1, normalize, chunked=True)
    q_norm = clean.double().norm(dim=-1, keepdim=True).repeat_interleave(2, 1) if not normalize else 1.0
    tol = plain.delta_tolerance(want, sums, errors * q_norm, eps, BF, 0.1, True)
    ok = torch.ones_like(want, dtype=torch.bool)
    ok[31, :2] = False
    assert ((out.double() - want).abs() <= tol)[ok].all()
    assert not torch.isfinite(out[31, :2].float()).any()
    assert ((state[c["slots"][0]].double() - S).norm(dim=1) <= E).all()


# A key head's value heads go in one workgroup from 1024 chunks and key heads on
GROUPED = [(128, 8, 48, 64, 32, BF), (64, 16, 32, 64, 32, HF)]


@pytest.mark.parametrize("case", GROUPED, ids=["x".join(map(str, c[:3])) for c in GROUPED])
def test_delta_rule_of_many_chunks(gpu, case):
    n, HK, HV, DK, DV, dtype = case
    counts = [13 + i % 3 for i in range(n)]
    c = delta_case(n, counts, HK, HV, DK, DV, dtype, True)
    out, state = run_delta(gpu, c, counts, [False] * n, DK ** -0.5)
    check_delta(c, counts, [False] * n, DK ** -0.5, out, state)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("DK,DV", [(64, 96), (128, 128), (64, 256), (128, 32)])
def test_delta_rule_of_short_and_long_sequences(gpu, DK, DV, dtype):
    """Sequences that are taken token by token beside those taken in chunks, of one call."""
    counts = [1, 20, 12, 0, 13, 5, 130, 1, 7]
    fresh = [False, True, True, False, False, False, False, True, False]
    c = delta_case(DK + DV, counts, 2, 6, DK, DV, dtype, True)
    out, state = run_delta(gpu, c, counts, fresh, DK ** -0.5)
    check_delta(c, counts, fresh, DK ** -0.5, out, state)
    for nobody in (0, 1):  # a short one, a long one
        slots = list(c["slots"])
        slots[nobody] = -1
        part, after = run_delta(gpu, dict(c, slots=slots), counts, fresh, DK ** -0.5)
        own = slice(0, 1) if nobody == 0 else slice(1, 21)
        assert (part[own] == 0).all()
        rest = torch.ones(len(part), dtype=torch.bool)
        rest[own] = False
        assert torch.equal(part[rest], out[rest])
        assert torch.equal(after[c["slots"][nobody]], c["state"][c["slots"][nobody]].to(after))


def test_delta_rule_in_pieces(gpu):
    """A sequence in one call, and in calls that continue each other through both forms."""
    counts = [150]
    c = delta_case(41, counts, 2, 4, 128, 64, HF, True)
    whole, state = run_delta(gpu, c, counts, [True], 0.09)
    parts, pool = [], c["state"].to(gpu)
    put = {n: (t.to(gpu) if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    at = 0
    for n in (1, 12, 64, 13, 0, 60):
        span = la.StateSpan(c["slots"], [n], fresh=[at == 0], device=gpu)
        row = slice(at, at + n)
        parts.append(la.gated_delta_rule(put["q"][row], put["k"][row], put["v"][row], put["decay"][row], put["beta"][row], pool, span,
                                         scaling=0.09, a_log=put["a_log"], dt_bias=put["dt_bias"]))
        at += n
    check_delta(c, counts, [True], 0.09, whole, state)
    check_delta(c, counts, [True], 0.09, torch.cat(parts).cpu(), pool.cpu())


@pytest.mark.parametrize("counts", [[1, 3], [40, 1, 80]])
def test_delta_rule_reads_slices_and_padding(gpu, counts):
    """q, k and v in one projection's rows, gates in another's, a slice of a larger pool, a sequence of nobody."""
    HK, HV, DK, DV, n = 2, 4, 64, 96, sum(counts) + 5 + 33
    full = counts + [5, 33]
    c = delta_case(51, full, HK, HV, DK, DV, BF, True, slots=list(range(1, len(counts) + 1)) + [-1, -1])
    fresh = [False] * len(full)
    mixed = torch.cat([c[x].flatten(1) for x in "qkv"] + [torch.zeros(n, 8, dtype=BF)], 1).to(gpu)
    q, k, v, _ = mixed.split((HK * DK, HK * DK, HV * DV, 8), 1)
    ba = torch.cat((c["beta"], c["decay"]), 1).to(gpu)
    pools = torch.full((c["state"].shape[0], 3, HV, DK, DV), 7.0, device=gpu)
    pools[:, 1] = c["state"].to(gpu)
    span = la.StateSpan(c["slots"], full, device=gpu)
    out = torch.full((n, HV, DV), 9.0, dtype=BF, device=gpu)
    got = la.gated_delta_rule(q.unflatten(1, (HK, DK)), k.unflatten(1, (HK, DK)), v.unflatten(1, (HV, DV)), ba[:, HV:], ba[:, :HV], pools[:, 1],
                              span, scaling=0.1, a_log=c["a_log"].to(gpu), dt_bias=c["dt_bias"].to(gpu), out=out)
    assert got is out
    check_delta(c, full, fresh, 0.1, out.cpu(), pools[:, 1].cpu())
    assert (pools[:, 0] == 7).all() and (pools[:, 2] == 7).all()
    # rows that are not 16-byte aligned are copied
    odd = torch.zeros(n, HK, DK + 1, dtype=BF, device=gpu)
    odd[..., 1:] = q.unflatten(1, (HK, DK))
    again = torch.empty_like(pools[:, 1].contiguous()).copy_(c["state"].to(gpu))
    got = la.gated_delta_rule(odd[..., 1:], k.unflatten(1, (HK, DK)), v.unflatten(1, (HV, DV)), ba[:, HV:], ba[:, :HV], again, span,
                              scaling=0.1, a_log=c["a_log"].to(gpu), dt_bias=c["dt_bias"].to(gpu))
    assert torch.equal(got, out) and torch.equal(again, pools[:, 1])


def test_delta_rule_gives_the_same_bits_again(gpu):
    counts = [1, 100, 7, 64, 1000]
    c = delta_case(61, counts, 2, 4, 128, 128, BF, True)
    first = run_delta(gpu, c, counts, [False] * 5, 0.1)
    for _ in range(3):
        out, state = run_delta(gpu, c, counts, [False] * 5, 0.1)
        assert torch.equal(out, first[0]) and torch.equal(state, first[1])


def test_no_tokens(gpu):
    span = la.StateSpan([1, 0], [0, 0], fresh=[True, True], device=gpu)
    state, conv_state = torch.ones(2, 2, 64, 32, device=gpu), torch.ones(2, 3, 16, device=gpu)
    e = torch.empty
    out = la.gated_delta_rule(e(0, 1, 64, dtype=BF, device=gpu), e(0, 1, 64, dtype=BF, device=gpu), e(0, 2, 32, dtype=BF, device=gpu),
                              e(0, 2, device=gpu), e(0, 2, device=gpu), state, span, scaling=1.0)
    assert out.shape == (0, 2, 32)
    assert la.causal_conv1d(e(0, 16, device=gpu), e(16, 4, device=gpu), None, conv_state, span).shape == (0, 16)
    assert (state == 1).all() and (conv_state == 1).all()
    assert la.rms_norm(e(0, 5, 8, device=gpu), e(8, device=gpu)).shape == (0, 5, 8)
    codes, scales = la.rms_norm_e4m3(e(0, 64, device=gpu), e(64, device=gpu), group_size=32)
    assert codes.shape == (0, 64) and scales.shape == (0, 2)


# ---------------------------------------------------------------- convolution

CONV = [
    # counts, fresh, channels, width, dtype, bias, silu
    ([1, 1, 1], [False, True, False], 64, 4, BF, False, True),
    ([1, 0, 2, 3, 4, 5], [False, True, True, False, True, False], 24, 4, HF, True, True),
    ([40, 1, 17], [False, False, True], 13, 3, BF, True, False),
    ([2, 1, 9, 33], [False] * 4, 1000, 8, BF, False, True),
    ([5, 16, 100], [True, False, False], 8, 2, F32, True, True),
    ([700, 3, 1], [False, True, False], 2056, 4, BF, True, True),
    ([6, 6, 6], [False, False, False], 7, 7, HF, False, False),
    ([3000], [False], 3, 5, F32, False, True),
]


@pytest.mark.parametrize("case", CONV, ids=[f"{c[0]}x{c[2]}w{c[3]}" for c in CONV])
@pytest.mark.parametrize("strided", [False, True])
def test_conv(gpu, case, strided):
    counts, fresh, ch, W, dtype, biased, silu = case
    n, pool = sum(counts), len(counts) + 3
    x, w = randn(1, n, ch).to(dtype), randn(2, ch, W).to(dtype)
    bias = randn(3, ch).to(dtype) if biased else None
    state = randn(4, pool, W - 1, ch).to(dtype)
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(9)).tolist()[:len(counts)]
    slots[-1] = -1 if strided and len(counts) > 1 else slots[-1]
    for s, f, m in zip(slots, fresh, counts):
        if f and m and s >= 0:
            state[s] = float("nan")
    rows, pools = x.to(gpu), state.to(gpu)
    if strided:
        wide, deep = torch.full((n, ch + 24), 3.0, dtype=dtype, device=gpu), torch.full((pool, 2, W - 1, ch), 3.0, dtype=dtype, device=gpu)
        wide[:, 8:8 + ch], deep[:, 1] = rows, pools
        rows, pools = wide[:, 8:8 + ch], deep[:, 1]
    got = la.causal_conv1d(rows, w.to(gpu), None if bias is None else bias.to(gpu), pools, la.StateSpan(slots, counts, fresh=fresh, device=gpu),
                           activation="silu" if silu else None)
    got, after, at = got.cpu(), pools.cpu(), 0
    u = torch.finfo(dtype).eps / 2
    step = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    for slot, f, m in zip(slots, fresh, counts):
        part = got[at:at + m]
        if slot < 0:
            assert (part == 0).all()
        elif m:
            old = torch.zeros_like(state[slot]) if f else state[slot]
            want, new, size = plain.conv(x[at:at + m], w, bias, old, silu)
            # the type's rounding; W + 1 roundings of the sum (SiLU's slope is at most 1.1) and its own function's
            tol = u * want.abs() + (1 + u) * 2.0 ** -24 * (1.1 * (W + 1) * size + 8 * want.abs()) + step
            assert ((part.double() - want).abs() <= tol).all()
            assert torch.equal(after[slot], new)
        else:
            assert torch.equal(after[slot], state[slot])
        at += m
    for s in range(pool):
        if s not in slots:
            assert torch.equal(after[s], state[s])
    if strided:
        assert (deep[:, 0] == 3).all() and (wide[:, :8] == 3).all() and (wide[:, 8 + ch:] == 3).all()


def test_conv_refuses_an_output_over_its_input(gpu):
    x = torch.zeros(4, 16, device=gpu)
    span = la.StateSpan([0], [4], device=gpu)
    with pytest.raises(ValueError, match="must not overlap x"):
        la.causal_conv1d(x, torch.zeros(16, 4, device=gpu), None, torch.zeros(1, 3, 16, device=gpu), span, out=x)


# ---------------------------------------------------------------- norms

COLS = [1, 7, 8, 40, 64, 100, 128, 256, 520, 2048, 2050, 4096, 8192, 8200, 20000, 20001]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("cols", COLS)
def test_norm(gpu, cols, dtype):
    for i, (rows, residual, gate, offset) in enumerate([(1, False, False, 0.0), (5, True, False, 1.0), (37, False, True, 0.0), (3, True, True, 0.5)]):
        x, w = (2 * randn(i, rows, cols)).to(dtype), randn(i + 50, cols).to(dtype)
        r = (5 * randn(i + 60, rows, cols)).to(dtype) if residual else None
        z = randn(i + 70, rows, cols).to(dtype) if gate else None
        stream = None if r is None else r.to(gpu)
        got = la.rms_norm(x.to(gpu), w.to(gpu), eps=1e-5, weight_offset=offset, residual=stream, gate=None if z is None else z.to(gpu))
        want, kept = plain.norm(x, w, 1e-5, offset, r, z)
        # the type's rounding; a sum of squares in chains of at most 48 + 10 roundings (half of its error), 8 products and functions
        tol = (torch.finfo(dtype).eps / 2 + 40 * 2.0 ** -24) * want.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert ((got.cpu().double() - want).abs() <= tol).all(), (rows, float(((got.cpu().double() - want).abs() / tol).max()))
        if r is not None:
            assert torch.equal(stream.cpu(), kept)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols,group", [(32, 32), (64, 64), (128, 128), (128, None), (384, 64), (100, None), (2048, 128), (4096, None), (4096, 32),
                                        (8320, 128), (20480, 64), (20001, None)])
def test_norm_e4m3(gpu, cols, group, dtype):
    for i, (rows, residual, gate) in enumerate([(1, False, False), (9, True, False), (4, False, True)]):
        x, w = randn(i, rows, cols).to(dtype), randn(i + 50, cols).to(dtype)
        r = (5 * randn(i + 60, rows, cols)).to(dtype) if residual else None
        z = randn(i + 70, rows, cols).to(dtype) if gate else None
        stream = None if r is None else r.to(gpu)
        codes, scales = la.rms_norm_e4m3(x.to(gpu), w.to(gpu), weight_offset=1.0, residual=stream, gate=None if z is None else z.to(gpu), group_size=group)
        want, kept = plain.norm(x, w, 1e-6, 1.0, r, z)
        n = group or cols
        parts = want.view(rows, cols // n, n)
        assert codes.dtype == torch.float8_e4m3fn and scales.shape == (rows, cols // n)
        top = parts.abs().amax(-1)
        assert ((scales.cpu().double() - top / 448).abs() <= 42 * 2.0 ** -24 * top / 448).all()
        got = codes.cpu().to(torch.float32).double().view_as(parts) * scales.cpu().double()[..., None]
        # half a step: 2^-4 of the value, 2^-10 scales below e4m3's normal values; fp32's part as above
        tol = (2.0 ** -4 + 80 * 2.0 ** -24) * parts.abs() + 2.0 ** -10 * scales.cpu().double()[..., None]
        assert ((got - parts).abs() <= tol).all()
        if r is not None:
            assert torch.equal(stream.cpu(), kept)


def test_norm_values_that_are_not_finite_or_tiny(gpu):
    x = randn(3, 6, 256)
    x[1, 7], x[2, 9], x[3] = float("nan"), float("inf"), 0.0
    x[4] *= 2.0 ** -40
    w = torch.ones(256)
    for dtype in (BF, F32):
        got = la.rms_norm(x.to(dtype).to(gpu), w.to(dtype).to(gpu)).cpu()
        want, _ = plain.norm(x.to(dtype), w, 1e-6, 0.0)
        assert torch.isnan(got[1]).all() and torch.isnan(got[2, 9]) and (got[2, :9] == 0).all()
        assert (got[3] == 0).all()
        ok = [0, 4, 5]
        assert ((got[ok].double() - want[ok]).abs() <= (torch.finfo(dtype).eps / 2 + 40 * 2.0 ** -24) * want[ok].abs()).all()
        codes, scales = la.rms_norm_e4m3(x.to(dtype).to(gpu), w.to(dtype).to(gpu), group_size=128)
        codes, scales = codes.cpu().float(), scales.cpu()
        assert torch.isnan(codes[1]).all() and torch.isnan(scales[1]).all()
        assert (codes[3] == 0).all() and (scales[3] == 0).all()
        assert torch.isfinite(codes[ok]).all() and (codes[ok].abs().amax(-1) == 448).all()
    # a weight that is not finite reaches its group alone
    w[130] = float("nan")
    codes, scales = la.rms_norm_e4m3(randn(4, 3, 256).to(gpu), w.to(gpu), group_size=128)
    assert torch.isfinite(codes.cpu().float()[:, :128]).all() and torch.isfinite(scales[:, 0]).all()
    assert torch.isnan(codes.cpu().float()[:, 130]).all() and torch.isnan(scales[:, 1]).all()


def test_norm_of_many_short_rows(gpu):
    rows = (1 << 23) + 5  # more than a launch has workgroups of one row
    x, w = randn(1, 64, 8).to(BF), randn(2, 8).to(BF)
    wide = x.to(gpu).repeat(rows // 64 + 1, 1)[:rows]
    got = la.rms_norm(wide, w.to(gpu))
    want, _ = plain.norm(x, w, 1e-6, 0.0)
    tol = (2.0 ** -8 + 40 * 2.0 ** -24) * want.abs() + 2.0 ** -140
    assert ((got[:64].cpu().double() - want).abs() <= tol).all()
    assert torch.equal(got[64:rows // 64 * 64].view(-1, 64, 8), got[:64].expand(rows // 64 - 1, 64, 8))
    assert torch.equal(got[rows // 64 * 64:], got[:rows % 64])


@pytest.mark.parametrize("cols", [64, 20000])
def test_norm_of_slices_of_one_matrix(gpu, cols):
    """x, residual and gate as columns of one matrix, and a residual that is x itself."""
    wide, w = randn(1, 9, 3 * cols).to(BF).to(gpu), randn(2, cols).to(BF).to(gpu)
    x, residual, gate = wide.split(cols, 1)
    apart = [t.clone() for t in (x, residual, gate)]
    want = la.rms_norm(apart[0], w, residual=apart[1], gate=apart[2])
    assert torch.equal(la.rms_norm(x, w, residual=residual, gate=gate), want)
    assert all(torch.equal(a, b) for a, b in zip((x, residual, gate), apart))
    twice = 2 * x
    want = la.rms_norm(twice, w)
    assert torch.equal(la.rms_norm(x, w, residual=x), want) and torch.equal(x, twice)
    with pytest.raises(ValueError, match="residual must not overlap x"):
        la.rms_norm(wide[:-1, :cols], w, residual=wide[1:, :cols])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols,group", [(96, 32), (128, None), (2048, 128), (20480, 64), (20480, None)])
def test_norm_of_unaligned_rows(gpu, cols, group, dtype):
    """Columns 3 and on of a wider matrix, to the bit as aligned ones."""
    wide, w = randn(cols, 5, cols + 8).to(dtype).to(gpu), randn(2, cols).to(dtype).to(gpu)
    x, residual = wide[:, 3:3 + cols], wide.flip(0)[:, 3:3 + cols]
    kept = residual.contiguous()
    for a, b in zip(la.rms_norm_e4m3(x, w, residual=residual, group_size=group),
                    la.rms_norm_e4m3(x.contiguous(), w, residual=kept, group_size=group)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(residual, kept)
    assert torch.equal(la.rms_norm(x, w), la.rms_norm(x.contiguous(), w))


def test_norm_layouts(gpu):
    """Rows of a wider tensor, an output in place, heads as leading dimensions."""
    x, w, z = randn(1, 6, 4, 64).to(BF), randn(2, 64).to(BF), randn(3, 6, 4, 64).to(BF)
    want, _ = plain.norm(x, w, 1e-6, 0.0, None, z)
    tol = (2.0 ** -8 + 40 * 2.0 ** -24) * want.abs() + 2.0 ** -140
    wide = torch.zeros(6, 4, 96, dtype=BF, device=gpu)
    wide[..., 8:72] = z.to(gpu)
    assert ((la.rms_norm(x.to(gpu), w.to(gpu), gate=wide[..., 8:72]).cpu().double() - want).abs() <= tol).all()
    assert ((la.rms_norm(x.to(gpu).transpose(0, 1), w.to(gpu), gate=z.to(gpu).transpose(0, 1)).cpu().double() - want.transpose(0, 1)).abs()
            <= tol.transpose(0, 1)).all()
    for place in ("x", "gate"):
        t = dict(x=x.to(gpu), gate=z.to(gpu))
        got = la.rms_norm(t["x"], w.to(gpu), gate=t["gate"], out=t[place])
        assert got is t[place] and ((got.cpu().double() - want).abs() <= tol).all()
    stream = torch.zeros(6, 4, 96, dtype=BF, device=gpu)
    rows = stream.view(24, 96)[:, 16:80]
    got = la.rms_norm(x.to(gpu).view(24, 64), w.to(gpu), residual=rows)
    assert torch.equal(rows.cpu(), x.view(24, 64)) and (stream.view(24, 96)[:, :16] == 0).all() and (stream.view(24, 96)[:, 80:] == 0).all()
    with pytest.raises(ValueError, match="written in place"):
        la.rms_norm(x.to(gpu), w.to(gpu), residual=torch.zeros(64, 4, 6, dtype=BF, device=gpu).permute(2, 1, 0))
