"""How the linear-attention calls are made: captured in graphs, on other streams, from threads, one after the other as a
layer runs them, and what they refuse on the device."""

import threading

import pytest
import torch

import _linear as plain
from _util import int4_payload
from anna_amd import _lib
from anna_amd import linear_attention as la
from anna_amd.quantization import XPUInt4Linear

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def nothing_cached():
    """The large tensors' segments go back to the device, so that nobody's lasting tensors come to lie in them."""
    yield
    torch.cuda.empty_cache()


BF = torch.bfloat16


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


class Layer:
    """The inner part of a linear-attention layer, with its states' pools."""

    def __init__(self, gpu, pool, HK=2, HV=4, D=128, width=4, seed=0):
        self.HK, self.HV, self.D, ch = HK, HV, D, (2 * HK + HV) * D
        self.conv_weight = (0.5 * randn(seed, ch, width)).to(BF).to(gpu)
        self.conv_state = randn(seed + 1, pool, width - 1, ch).to(BF).to(gpu)
        self.state = (0.3 * randn(seed + 2, pool, HV, D, D)).to(gpu)
        self.a_log, self.dt_bias = randn(seed + 3, HV).to(gpu), (randn(seed + 4, HV) - 3).to(gpu)
        self.norm = (1 + 0.1 * randn(seed + 5, D)).to(BF).to(gpu)

    def states(self):
        return self.conv_state.clone(), self.state.clone()

    def set(self, states):
        self.conv_state.copy_(states[0])
        self.state.copy_(states[1])

    def __call__(self, x, a, b, z, span):
        HK, HV, D = self.HK, self.HV, self.D
        mixed = la.causal_conv1d(x, self.conv_weight, None, self.conv_state, span)
        q, k, v = mixed.split((HK * D, HK * D, HV * D), 1)
        out = la.gated_delta_rule(q.unflatten(1, (HK, D)), k.unflatten(1, (HK, D)), v.unflatten(1, (HV, D)), a, b, self.state, span,
                                  scaling=D ** -0.5, a_log=self.a_log, dt_bias=self.dt_bias)
        return la.rms_norm(out, self.norm, gate=z)

    def inputs(self, seed, n, gpu):
        ch = (2 * self.HK + self.HV) * self.D
        return (randn(seed, n, ch).to(BF).to(gpu), randn(seed + 1, n, self.HV).to(BF).to(gpu), randn(seed + 2, n, self.HV).to(BF).to(gpu),
                randn(seed + 3, n, self.HV, self.D).to(BF).to(gpu))


@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 1, 5], [70, 1, 20], [13] * 40])
def test_captured_steps_equal_eager_ones(gpu, counts):
    n = sum(counts)
    layer = Layer(gpu, len(counts) + 4)
    slots = list(range(len(counts)))
    span = la.StateSpan(slots, counts, device=gpu)
    given = layer.inputs(7, n, gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(*given, span)
    torch.cuda.current_stream().wait_stream(side)
    start = layer.states()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(*given, span)
    for step in range(4):  # other inputs, other slots, with the program's own work in between
        new = layer.inputs(100 + 10 * step, n, gpu)
        turned = [(s + step) % (len(counts) + 4) for s in slots]
        if step == 3:
            turned[0] = -1
        fresh = [(i + step) % 3 == 0 for i in range(len(counts))]
        before = layer.states()
        want = layer(*new, la.StateSpan(turned, counts, fresh=fresh, device=gpu))
        after = layer.states()
        layer.set(before)
        for t, x in zip(given, new):
            t.copy_(x)
        span.refill(turned, fresh=fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for got, kept in zip(layer.states(), after):
            assert torch.equal(got, kept)
    assert not torch.equal(start[1], layer.state)


def test_two_captured_graphs_share_nothing(gpu):
    """Each keeps a workspace of its own: replays of the two, one after the other and again, answer as alone."""
    layers = [Layer(gpu, 3, seed=s) for s in (0, 50)]
    counts = [100, 1, 30]
    graphs, outs, given = [], [], []
    for i, layer in enumerate(layers):
        span = la.StateSpan([0, 1, 2], counts, device=gpu)
        x = layer.inputs(20 + i, sum(counts), gpu)
        first = layer.states()
        want = layer(*x, span)
        layer.set(first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(*x, span)
        graphs.append((graph, span, layer, first))
        outs.append((out, want))
        given.append(x)
    for _ in range(3):
        for graph, _, layer, first in graphs:
            layer.set(first)
            graph.replay()
        torch.cuda.synchronize()
        for out, want in outs:
            assert torch.equal(out, want)


def test_spans_are_not_made_while_capturing(gpu):
    span = la.StateSpan([0], [1], device=gpu)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(8, device=gpu)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            la.StateSpan([0], [1], device=gpu)
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            span.refill([0])


def test_on_another_stream(gpu):
    layer = Layer(gpu, 4)
    counts = [90, 1, 3]
    x = layer.inputs(3, sum(counts), gpu)
    first = layer.states()
    want = layer(*x, la.StateSpan([2, 0, 3], counts, device=gpu))
    layer.set(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        span = la.StateSpan([2, 0, 3], counts, device=gpu)
        got = layer(*x, span)
        del span  # its memory stays until the stream has passed
    junk = [torch.full((4096,), -1, dtype=torch.int32, device=gpu) for _ in range(20)]
    side.synchronize()
    assert torch.equal(got, want) and len(junk) == 20


def test_from_threads(gpu):
    """Every thread with a layer and a stream of its own."""
    counts, answers, errors = [40, 2, 1, 13], {}, []
    layers = [Layer(gpu, 5, seed=20 * i) for i in range(4)]
    firsts = [layer.states() for layer in layers]
    wants = []
    for i, layer in enumerate(layers):
        wants.append(layer(*layer.inputs(i, sum(counts), gpu), la.StateSpan([4, 1, 0, 2], counts, device=gpu)))
        layer.set(firsts[i])
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    layers[i].set(firsts[i])
                    answers[i] = layers[i](*layers[i].inputs(i, sum(counts), gpu), la.StateSpan([4, 1, 0, 2], counts, device=gpu))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(4):
        assert torch.equal(answers[i], wants[i])


def test_the_host_module_and_the_general_way_agree(gpu, monkeypatch):
    layer = Layer(gpu, 4)
    counts = [20, 1, 0, 2]
    x = layer.inputs(9, sum(counts), gpu)
    span = la.StateSpan([3, 1, 0, 2], counts, fresh=[True, False, True, False], device=gpu)
    first = layer.states()
    hidden, stream, weight = randn(1, 5, 256).to(BF).to(gpu), randn(2, 5, 256).to(BF).to(gpu), randn(3, 256).to(BF).to(gpu)

    def all_calls():
        layer.set(first)
        kept = stream.clone()
        return [layer(*x, span), *layer.states(), la.rms_norm(hidden, weight, residual=kept, weight_offset=1.0), kept,
                *la.rms_norm_e4m3(hidden, weight, group_size=64), *la.rms_norm_e4m3(hidden, weight, gate=stream)]

    want = all_calls()

    class Nothing:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(la, "_host", Nothing)
    for got, w in zip(all_calls(), want):
        assert got.dtype == w.dtype and torch.equal(got.float(), w.float())


def test_device_refusals(gpu):
    layer = Layer(gpu, 2)
    x, a, b, z = layer.inputs(1, 3, gpu)
    span = la.StateSpan([0, 1], [1, 2], device=gpu)
    with pytest.raises(RuntimeError, match="slot 2 of a state of 2"):
        layer(x, a, b, z, la.StateSpan([0, 2], [1, 2], device=gpu))
    with pytest.raises(ValueError, match="span holds 3 tokens, got 2"):
        la.causal_conv1d(x[:2], layer.conv_weight, None, layer.conv_state, span)
    with pytest.raises(RuntimeError, match="weight must be on cuda"):
        la.causal_conv1d(x, layer.conv_weight.cpu(), None, layer.conv_state, span)
    with pytest.raises(RuntimeError, match="x requires grad"):
        la.causal_conv1d(x.clone().requires_grad_(), layer.conv_weight, None, layer.conv_state, span)
    with pytest.raises(RuntimeError, match="weight requires grad"):
        la.rms_norm(z, layer.norm.clone().requires_grad_())
    with torch.no_grad():
        la.rms_norm(z, layer.norm.clone().requires_grad_())
    q = torch.zeros(3, 2, 128, dtype=BF, device=gpu)
    v = torch.zeros(3, 4, 128, dtype=BF, device=gpu)
    with pytest.raises(RuntimeError, match="value requires grad"):
        la.gated_delta_rule(q, q, v.clone().requires_grad_(), a, b, layer.state, span, scaling=1.0)
    with pytest.raises(ValueError, match="must not overlap value"):
        la.gated_delta_rule(q, q, v, a, b, layer.state, span, scaling=1.0, out=v)
    with pytest.raises(ValueError, match="span holds 3 tokens, got 0"):
        la.gated_delta_rule(q[:0], q[:0], v[:0], a[:0], b[:0], layer.state, span, scaling=1.0)
    with pytest.raises(RuntimeError, match="named twice"):
        la.StateSpan([0, 0], [1, 1], device=gpu)
    with pytest.raises(ValueError, match="2 slots, 1 counts"):
        la.StateSpan([0, 1], [1], device=gpu)
    with pytest.raises(ValueError, match="same counts"):
        span._lay_out([0, 1], [2, 1], None)
    with pytest.raises(RuntimeError, match="slot 5 is named twice"):
        span.refill([5, 5])
    la.causal_conv1d(x, layer.conv_weight, None, layer.conv_state, span)
    with pytest.raises(RuntimeError, match="slot 2: the span was used with states of 2 slots"):
        span.refill([2, 0])  # a graph captured with it would write behind the pool
    assert span.slots == [0, 1] and span.counts == [1, 2] and span.tokens == 3
    la.causal_conv1d(x, layer.conv_weight, None, layer.conv_state, span)  # as it was


def test_a_layer_between_int4_projections(gpu):
    """residual norm -> int4 projection -> convolution -> delta rule -> gated norm -> int4 projection, over a prompt of each
    sequence and then drafted and single tokens, against the same steps in 64 bits rounded to the type where the calls
    round.  Each of the nine roundings on the way is off by at most 2^-8 of its value, most by far less, and none grows: the
    2-norm of the difference stays below 9 * 2^-8 / sqrt(3) of the answer's, a uniform error's mean square a rounding."""
    H, HK, HV, D, W, pool = 256, 2, 4, 64, 4, 4
    ch = (2 * HK + HV) * D
    import numpy as np

    rng = np.random.default_rng(3)

    def linear(out_features, in_features):
        qweight, scales, zeros = int4_payload(rng, out_features, in_features, 128)
        codes = (torch.from_numpy(qweight).long()[..., None] >> (4 * torch.arange(8))) & 15
        s, z = (torch.from_numpy(t).double().repeat_interleave(128, 0).T for t in (scales / 4, zeros))
        layer = XPUInt4Linear(in_features, out_features, bias=False, group_size=128, compute_dtype=BF, device=gpu)
        layer.qweight.copy_(torch.from_numpy(qweight))
        layer.qscale.copy_(torch.from_numpy(scales / 4))
        layer.qzeros.copy_(torch.from_numpy(zeros))
        return layer, ((codes.flatten(1).double() - z) * s).to(BF).double()

    proj, w_in = linear(ch + HV * D + 64, H)  # q, k, v | z | a, b, padding
    back, w_out = linear(H, HV * D)
    conv_w, norm_w, pre_w = (0.5 * randn(1, ch, W)).to(BF), (1 + 0.1 * randn(2, D)).to(BF), (0.1 * randn(3, H)).to(BF)
    a_log, dt_bias = randn(4, HV), randn(5, HV) - 2
    conv_state, state = torch.zeros(pool, W - 1, ch, dtype=BF), torch.zeros(pool, HV, D, D)
    dev = {n: t.to(gpu) for n, t in dict(conv_w=conv_w, norm_w=norm_w, pre_w=pre_w, a_log=a_log, dt_bias=dt_bias, conv=conv_state, state=state).items()}
    ref_conv, ref_state = conv_state.clone(), state.double()
    slots = [2, 0, 3]
    for step, counts in enumerate(([90, 5, 14], [1, 3, 1], [1, 1, 1])):
        n = sum(counts)
        x, stream = randn(50 + step, n, H).to(BF), randn(60 + step, n, H).to(BF)
        span = la.StateSpan(slots, counts, fresh=[step == 0] * 3, device=gpu)
        kept = stream.to(gpu)
        h = la.rms_norm(x.to(gpu), dev["pre_w"], weight_offset=1.0, residual=kept)
        p = proj(h)
        mixed = la.causal_conv1d(p[:, :ch], dev["conv_w"], None, dev["conv"], span)
        q, k, v = mixed.split((HK * D, HK * D, HV * D), 1)
        z, b, a = p[:, ch:ch + HV * D], p[:, ch + HV * D:ch + HV * D + HV], p[:, ch + HV * D + HV:ch + HV * D + 2 * HV]
        o = la.gated_delta_rule(q.unflatten(1, (HK, D)), k.unflatten(1, (HK, D)), v.unflatten(1, (HV, D)), a, b, dev["state"], span,
                                scaling=D ** -0.5, a_log=dev["a_log"], dt_bias=dev["dt_bias"])
        got = back(la.rms_norm(o, dev["norm_w"], gate=z.unflatten(1, (HV, D))).flatten(1)).cpu()

        hr, kr = plain.norm(x, pre_w, 1e-6, 1.0, stream)
        assert torch.equal(kept.cpu(), kr)
        pr = (hr.to(BF).double() @ w_in.T).to(BF)
        want, at = torch.empty(n, H, dtype=torch.float64), 0
        for slot, m in zip(slots, counts):
            rows = slice(at, at + m)
            at += m
            y, ref_conv[slot], _ = plain.conv(pr[rows, :ch], conv_w, None, ref_conv[slot], True)
            qr, kr2, vr = y.to(BF).split((HK * D, HK * D, HV * D), 1)
            zr, br, ar = pr[rows, ch:ch + HV * D], pr[rows, ch + HV * D:ch + HV * D + HV], pr[rows, ch + HV * D + HV:ch + HV * D + 2 * HV]
            g, beta = plain.gates(ar, br, a_log, dt_bias)
            o_ref, ref_state[slot], *_ = plain.delta_rule(qr.unflatten(1, (HK, D)), kr2.unflatten(1, (HK, D)), vr.unflatten(1, (HV, D)), g, beta,
                                                          ref_state[slot], D ** -0.5)
            y, _ = plain.norm(o_ref.to(BF), norm_w, 1e-6, 0.0, None, zr.unflatten(1, (HV, D)))
            want[rows] = y.to(BF).flatten(1).double() @ w_out.T
        assert float((got.double() - want).norm() / want.norm()) < 9 * 2.0 ** -8 / 3 ** 0.5
        assert float((dev["state"].cpu().double() - ref_state).norm() / ref_state.norm()) < 9 * 2.0 ** -8 / 3 ** 0.5


def test_many_tokens_cross_32_bits_of_elements(gpu):
    """A packed batch whose rows lie further apart than 2^31 bytes, and a pool whose slots do."""
    HK, HV, D = 1, 1, 64
    tokens, stride = 3, (1 << 30) + 64  # elements of 2 bytes
    store = torch.empty((tokens - 1) * stride + 256, dtype=BF, device=gpu)
    rows = [randn(i, 3 * D).to(BF) for i in range(tokens)]
    for i, r in enumerate(rows):
        store[i * stride:i * stride + 3 * D] = r.to(gpu)
    mixed = store.as_strided((tokens, 3 * D), (stride, 1))
    pool = torch.empty(2 * ((1 << 30) + 64), device=gpu).as_strided((2, HV, D, D), ((1 << 30) + 64, D * D, D, 1))
    pool.zero_()
    g, beta = torch.full((tokens, 1), -0.5, device=gpu), torch.full((tokens, 1), 0.5, device=gpu)
    out = la.gated_delta_rule(*(mixed[:, i * D:(i + 1) * D].unflatten(1, (1, D)) for i in range(3)), g, beta, pool,
                              la.StateSpan([1], [tokens], device=gpu), scaling=1.0)
    x = torch.stack(rows).view(tokens, 3, 1, D)
    want, S, sums, errors, E, c = plain.delta_rule(x[:, 0], x[:, 1], x[:, 2], g.cpu().double(), beta.cpu().double(), torch.zeros(1, D, D), 1.0)
    assert ((out.cpu().double() - want).abs() <= plain.delta_tolerance(want, sums, errors, c, BF, 1.0, False)).all()
    assert ((pool[1].cpu().double() - S).norm(dim=1) <= E).all() and (pool[0] == 0).all()
    w = randn(9, 3 * D, 4).to(BF)
    conv_state = torch.zeros(1, 3, 3 * D, dtype=BF, device=gpu)
    y = la.causal_conv1d(mixed, w.to(gpu), None, conv_state, la.StateSpan([0], [tokens], device=gpu))
    ref, _, size = plain.conv(torch.stack(rows), w, None, torch.zeros(3, 3 * D, dtype=BF), True)
    assert ((y.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -24 * (7 * size + 8 * ref.abs()) * 1.01).all()
    n = la.rms_norm(mixed, torch.ones(3 * D, dtype=BF, device=gpu))
    ref, _ = plain.norm(torch.stack(rows), torch.ones(3 * D), 1e-6, 0.0)
    assert ((n.cpu().double() - ref).abs() <= (2.0 ** -8 + 40 * 2.0 ** -24) * ref.abs()).all()


def test_c_abi_without_a_stream(gpu):
    """A C caller's default stream, and a span of its own."""
    import ctypes

    x, w = randn(1, 4, 96).to(BF).to(gpu), randn(2, 96).to(BF).to(gpu)
    out = torch.empty_like(x)
    args = _lib.RmsNormArgs(dtype=_lib.BF16, rows=4, cols=96, x=x.data_ptr(), x_stride=96, weight=w.data_ptr(), eps=1e-6, out=out.data_ptr(), out_stride=96)
    torch.cuda.synchronize()
    _lib.call("anna_mi_rms_norm", ctypes.byref(args), None)
    torch.cuda.synchronize()
    assert torch.equal(out, la.rms_norm(x, w))
