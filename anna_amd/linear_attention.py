"""Linear attention: the operators between the projections of a gated-delta-rule layer.

Hybrid models alternate attention layers, whose caches this package quantizes, with layers that keep a state of fixed
size per sequence.  Between its (int4) projections such a layer runs a short causal convolution, the
gated delta rule and a gated root-mean-square norm; around the layer the residual stream is added and
normalised.  The reference runs them as SYCL kernels on batches of equal lengths (sycl:5618-7600, 3345-3714,
1764-1986).  Here the tokens of a step are packed, one sequence after the other, and the states of all sequences are
rows ("slots") of pools; prompts, chunks of them, drafted and single tokens mix as they come:

    span = StateSpan(slots=[3, 0, 7], counts=[1000, 37, 1], fresh=[True, True, False])   # once for all layers
    mixed = causal_conv1d(mixed, conv_weight, None, conv_state[layer], span)             # [1038, channels]
    out = gated_delta_rule(query, key, value, a, b, state[layer], span, scaling=128 ** -0.5,
                           a_log=a_log, dt_bias=dt_bias)                                 # [1038, heads, 128]
    out = rms_norm(out, norm_weight, gate=z)
    hidden = rms_norm(out_proj, next_weight, weight_offset=1.0, residual=stream)         # stream += out_proj

The operators are for inference: tensors that require grad are refused outside ``torch.no_grad()``, dual tensors everywhere.  They run on
the current stream of their tensors' device and can be captured in a graph, with a span made before; between replays
``StateSpan.refill`` names other slots.  Calls that share states must not overlap on the GPU.
"""

from __future__ import annotations

import ctypes
import operator

import torch
from torch.autograd import forward_ad

from . import _lib

KEY_DIMS = (64, 128)
E4M3_GROUPS = (32, 64, 128)


def _ints(what: str, values, low: int, high: int, ctype):
    values = [operator.index(v) for v in values]
    for v in values:
        if not low <= v <= high:
            raise ValueError(f"{what} {v} is out of range")
    return (ctype * len(values))(*values)


class StateSpan:
    """The packed tokens of a step: ``counts[i]`` tokens (one each by default, 0 allowed) that continue the states in
    row ``slots[i]`` of the pools, one sequence after the other.

    A slot is named at most once.  Slot -1 stands for a sequence of nobody, as the padding of a captured batch
    holds: its outputs are zeros and it touches no state.  ``fresh[i]``: the sequence is new, its states' content is taken as
    zeros.  A sequence without tokens leaves its states as they are, whatever ``fresh`` says."""

    def __init__(self, slots, counts=None, *, fresh=None, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"StateSpan needs a ROCm device, got {device}")
        self._index = torch.cuda.current_device() if device.index is None else device.index
        self.device = torch.device("cuda", self._index)
        self._counts = None
        self._c = _lib.StateSpan()
        self._ref = ctypes.byref(self._c)
        words = self._lay_out(slots, counts, fresh)
        self._buf = words.to(self.device)
        self._c.buf = self._buf.data_ptr()
        self._address = ctypes.addressof(self._c)
        self._streams = {self._stream()}

    def _lay_out(self, slots, counts, fresh) -> torch.Tensor:
        slots = _ints("slot", slots, -1, (1 << 31) - 1, ctypes.c_int32)
        n = len(slots)
        counts = _ints("count", [1] * n if counts is None else counts, 0, (1 << 31) - 1, ctypes.c_int64)
        fresh = (ctypes.c_int32 * n)(*[bool(f) for f in ([False] * n if fresh is None else fresh)])
        if len(counts) != n or len(fresh) != n:
            raise ValueError(f"{n} slots, {len(counts)} counts and {len(fresh)} values of fresh")
        if self._counts is not None and list(counts) != self._counts:
            raise ValueError("a span is filled again with the same counts")
        if torch.cuda.is_available() and self._capturing():
            # the layout is made on the host: a replay would not make it again
            raise RuntimeError("a StateSpan cannot be made or filled while a graph is captured")
        plan = _lib.StateSpan()
        _lib.call("anna_mi_state_span_plan", n, slots, counts, fresh, ctypes.byref(plan))
        words = torch.empty((plan.words,), dtype=torch.int32)
        _lib.call("anna_mi_state_span_fill", n, slots, counts, fresh, ctypes.byref(plan), words.data_ptr())
        if self._counts is None:
            ctypes.memmove(ctypes.addressof(self._c), ctypes.addressof(plan), ctypes.sizeof(plan))
        else:  # refuses what a graph captured with this span would write to; nothing else of the span changes
            _lib.call("anna_mi_state_span_refill", self._ref, ctypes.byref(plan))
        self.slots, self._counts, self.fresh = list(slots), list(counts), [bool(f) for f in fresh]
        return words

    def refill(self, slots, *, fresh=None) -> None:
        """Other slots for the same counts, in place: what a graph that was captured with this span replays next.
        Ordered on the current stream, behind the work that reads the old ones."""
        self._used()
        self._buf.copy_(self._lay_out(slots, self._counts, fresh))

    def _capturing(self) -> bool:
        with torch.cuda.device(self.device):
            return torch.cuda.is_current_stream_capturing()

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self._index)

    def _used(self) -> int:
        """The current stream, on which the span's buffer is used from now on."""
        stream = _raw_stream(self._index)
        if stream not in self._streams:
            self._streams.add(stream)
            self._buf.record_stream(torch.cuda.current_stream(self.device))
        return stream

    @property
    def counts(self) -> list[int]:
        return list(self._counts)

    @property
    def tokens(self) -> int:
        """Tokens of all sequences."""
        return self._c.tokens


# ---------------------------------------------------------------- checks


def _on(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device}, got a tensor on {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            # an answer without a graph would lose its gradient without a word
            raise RuntimeError(f"{name} requires grad, but there is no backward pass: call it under torch.no_grad()")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has a tangent, but there is no forward derivative")


def _call(device: torch.device, name: str, *args) -> None:
    if torch.cuda.current_device() == device.index:
        _lib.call(name, *args)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args)


def _written(*tensors: torch.Tensor | None) -> None:
    """Lets autograd see what a call has written, where it keeps the tensor; inference tensors have no version."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _memory(t: torch.Tensor) -> tuple[int, int]:
    """First byte and the one behind the last that a tensor's elements lie in."""
    start = t.data_ptr()
    if t.numel() == 0:
        return start, start
    return start, start + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _apart(out: torch.Tensor, **tensors) -> None:
    """Refuses an output whose memory overlaps an input's."""
    low, high = _memory(out)
    for name, t in tensors.items():
        if t is not None:
            a, b = _memory(t)
            if a < high and low < b:
                raise ValueError(f"out must not overlap {name}")


def _state_apart(state: torch.Tensor, stride: int, **tensors) -> None:
    """Refuses a pool of states over an input: a state is written while other workgroups still read it.  Inputs may lie
    between the slots, as other columns of one matrix or in one row."""
    low, high = _memory(state)
    if low == high:
        return
    step, size = stride * state.element_size(), state[0].numel() * state.element_size()
    for name, t in tensors.items():
        if t is None or t.numel() == 0:
            continue
        a, b = _memory(t)
        if a >= high or low >= b:
            continue
        column, single = (a - low) % step, _memory(t[0])
        if column < size or not (column + b - a <= step or (t.stride(0) * t.element_size() == step and column + single[1] - a <= step)):
            raise ValueError(f"state must not overlap {name}")


def _heads(what: str, t: torch.Tensor, dtype: torch.dtype, tokens: int, heads: int, dim: int) -> torch.Tensor:
    """Rows [tokens, heads, dim] as the kernels read them, 16 bytes at a time; copied where they are not."""
    if t.dtype != dtype or tuple(t.shape) != (tokens, heads, dim):
        raise ValueError(f"{what} must be {dtype} {[tokens, heads, dim]}, got {t.dtype} {list(t.shape)}")
    if (t.stride(2) != 1 or t.data_ptr() % 16 or (tokens > 1 and t.stride(0) % 8) or (heads > 1 and t.stride(1) % 8)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t: torch.Tensor) -> tuple[int, int]:
    # the stride of a single token or head is read by nobody
    return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def _pool(what: str, state: torch.Tensor, dtype: torch.dtype, shape: tuple[int, ...]) -> int:
    """Checks a pool of states [slots, *shape] and returns the elements from one slot to the next."""
    if state.dtype != dtype or state.dim() != len(shape) + 1 or tuple(state.shape[1:]) != shape:
        raise ValueError(f"{what} must be {dtype} {['slots', *shape]}, got {state.dtype} {list(state.shape)}")
    size = 1
    for n, s in zip(reversed(shape), reversed(state.stride()[1:])):
        if n > 1 and s != size:
            raise ValueError(f"{what} must be contiguous in each slot, got strides {list(state.stride())}")
        size *= n
    if state.shape[0] > 1 and state.stride(0) < size:
        raise ValueError(f"{what}: slots overlap, got strides {list(state.stride())}")
    return state.stride(0) if state.shape[0] > 1 else size


def _check_span(what: str, span: StateSpan, tokens: int, device: torch.device) -> int:
    if span.device != device:
        raise RuntimeError(f"{what}: the span is on {span.device}, the tensors on {device}")
    if span._c.tokens != tokens:
        raise ValueError(f"{what}: the span holds {span._c.tokens} tokens, got {tokens}")
    return span._used()


# The host module takes the plain calls on the current device; it answers None to those that the general way
# below converts or refuses.
_host, _cuda_device, _raw_stream = _lib.host, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# ---------------------------------------------------------------- operators


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, state: torch.Tensor, span: StateSpan,
                  *, activation: str | None = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
    """Depthwise causal convolution of each sequence's tokens: x [tokens, channels] -> the same shape,

        out[t] = act(bias + sum_j weight[:, j] * x[t - width + 1 + j])

    with the rows of the sequence's state in front.  weight [channels, width], width 2 to 8; state [slots, width - 1,
    channels], the last inputs of every sequence, oldest first, updated in place; all of one type (bf16, fp16
    or fp32; sums in fp32).  x may be strided by rows (a slice of a projection).  activation: "silu" or None.  out must not overlap
    an input, and state neither."""
    if out is None and span is not None and x.is_cuda and _cuda_device() == span._index and (activation == "silu" or activation is None):
        got = _host().causal_conv1d(x, weight, bias, state, span._address, span._index, activation is not None, span._used())
        if got is not None:
            return got
    if x.dim() != 2 or x.dtype not in _lib._DTYPE_CODES:
        raise ValueError(f"x must be [tokens, channels] in bfloat16, float16 or float32, got {x.dtype} {list(x.shape)}")
    tokens, channels = x.shape
    if weight.dtype != x.dtype or weight.dim() != 2 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 8:
        raise ValueError(f"weight must be {x.dtype} [{channels}, 2 to 8], got {weight.dtype} {list(weight.shape)}")
    width = weight.shape[1]
    if bias is not None and (bias.dtype != x.dtype or tuple(bias.shape) != (channels,)):
        raise ValueError(f"bias must be {x.dtype} [{channels}], got {bias.dtype} {list(bias.shape)}")
    if activation not in ("silu", None):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if channels < 1:
        raise ValueError("x has no channels")
    stride = _pool("state", state, x.dtype, (width - 1, channels))
    _state_apart(state, stride, x=x, weight=weight, bias=bias)
    _lib.require_device(x)
    _on(x.device, x=x, weight=weight, bias=bias, state=state, out=out)
    stream = _check_span("causal_conv1d", span, tokens, x.device)
    if x.stride(1) != 1 and channels > 1 or tokens > 1 and x.stride(0) < channels:
        x = x.contiguous()
    if out is None:
        out = torch.empty((tokens, channels), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or out.shape != x.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {x.dtype} {list(x.shape)}")
    else:
        _apart(out, x=x, state=state, weight=weight, bias=bias)
    weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
    _call(x.device, "anna_mi_causal_conv1d", x.data_ptr(), _lib.dtype_code(x.dtype), channels, x.stride(0) if tokens > 1 else channels,
          weight.data_ptr(), width, _lib.ptr(bias), state.data_ptr(), state.shape[0], stride, int(activation == "silu"), span._ref,
          out.data_ptr(), channels, stream)
    _written(state, out)
    return out


def gated_delta_rule(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, decay: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, span: StateSpan, *, scaling: float, normalize: bool = True,
                     a_log: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """The gated delta rule over each sequence's tokens: for every token and value head

        u = beta (v - e^g S^T k),    S <- e^g S + k u^T,    out = scaling S^T q

    with k and q divided by sqrt(|.|^2 + 1e-6) first (``normalize``).  query and key [tokens, key_heads, key_dim],
    value [tokens, value_heads, value_dim] in bf16 or fp16 -> out as value; value head h reads key head
    h // (value_heads // key_heads).  key_dim 64 or 128, value_dim a multiple of 32 up to 256.  Strided slices
    of one projection are read where they lie.  state fp32 [slots, value_heads, key_dim, value_dim] is updated in place;
    it and out overlap no input.

    decay and beta [tokens, value_heads] (fp32 or 16 bits) are g, at most 0, and beta; with ``a_log`` and ``dt_bias``
    (fp32 [value_heads]) they are the projections that those are made from:
    g = -exp(a_log) softplus(decay + dt_bias), beta = sigmoid(beta).

    Sequences of up to 12 tokens go token by token, longer ones in chunks of 64 tokens.  The state is fp32, and sums and
    products are fp32 or as exact, at the size of what a token sees: values and states far larger that come later, or that
    a decay has made small, take nothing from it.  (Chunks that hold both are taken token by token, which takes longer.)
    Chunks need a workspace: each 256 * key_heads * key_dim + 26 KB * value_heads bytes, 1.4 MB at 16 and 32 heads of
    128, for all of the call's chunks together (1.4 GB for 64 K tokens)."""
    if out is None and span is not None and query.is_cuda and _cuda_device() == span._index:
        got = _host().gated_delta(query, key, value, decay, beta, state, a_log, dt_bias, span._address, span._index, scaling, normalize, span._used())
        if got is not None:
            return got
    if query.dim() != 3 or value.dim() != 3 or query.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"query and value must be [tokens, heads, dim] in bfloat16 or float16, got {query.dtype} "
                         f"{list(query.shape)} and {list(value.shape)}")
    tokens, key_heads, key_dim = query.shape
    value_heads, value_dim = value.shape[1:]
    if key_dim not in KEY_DIMS:
        raise ValueError(f"key_dim {key_dim}: 64 and 128 are supported")
    if not 32 <= value_dim <= 256 or value_dim % 32:
        raise ValueError(f"value_dim {value_dim}: multiples of 32 up to 256 are supported")
    if key_heads < 1 or value_heads < 1 or value_heads % key_heads:
        raise ValueError(f"value_heads ({value_heads}) must be a multiple of key_heads ({key_heads})")
    q = _heads("query", query, query.dtype, tokens, key_heads, key_dim)
    k = _heads("key", key, query.dtype, tokens, key_heads, key_dim)
    v = _heads("value", value, query.dtype, tokens, value_heads, value_dim)
    for name, t in (("decay", decay), ("beta", beta)):
        if t.dtype not in _lib._DTYPE_CODES or t.dtype != decay.dtype or tuple(t.shape) != (tokens, value_heads):
            raise ValueError(f"{name} must be [{tokens}, {value_heads}] in float32, bfloat16 or float16, decay and beta alike, got "
                             f"{t.dtype} {list(t.shape)}")
    if (a_log is None) != (dt_bias is None):
        raise ValueError("a_log and dt_bias go together")
    for name, t in (("a_log", a_log), ("dt_bias", dt_bias)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (value_heads,)):
            raise ValueError(f"{name} must be float32 [{value_heads}], got {t.dtype} {list(t.shape)}")
    scaling = float(scaling)
    if not -1e30 < scaling < 1e30:
        raise ValueError(f"scaling must be finite, got {scaling}")
    stride = _pool("state", state, torch.float32, (value_heads, key_dim, value_dim))
    if state.data_ptr() % 16 or stride % 4:
        raise ValueError("state must be 16-byte aligned in every slot")
    _state_apart(state, stride, query=query, key=key, value=value, decay=decay, beta=beta, a_log=a_log, dt_bias=dt_bias)
    device = query.device
    _lib.require_device(query)
    _on(device, query=query, key=key, value=value, decay=decay, beta=beta, a_log=a_log, dt_bias=dt_bias, state=state, out=out)
    stream = _check_span("gated_delta_rule", span, tokens, device)
    if out is None:
        out = torch.empty((tokens, value_heads, value_dim), dtype=query.dtype, device=device)
    elif out.dtype != query.dtype or out.shape != value.shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned {query.dtype} {list(value.shape)}")
    else:
        _apart(out, query=q, key=k, value=v, decay=decay, beta=beta, state=state, a_log=a_log, dt_bias=dt_bias)
    g, b = (t if t.stride(1) == 1 or value_heads == 1 else t.contiguous() for t in (decay, beta))
    a_log, dt_bias = (None if t is None else t.contiguous() for t in (a_log, dt_bias))
    args = _lib.GatedDeltaArgs(
        _lib.dtype_code(q.dtype), _lib.dtype_code(g.dtype), int(bool(normalize)), scaling, key_heads, value_heads, key_dim, value_dim,
        q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), g.data_ptr(), g.stride(0) if tokens > 1 else 0,
        b.data_ptr(), b.stride(0) if tokens > 1 else 0, _lib.ptr(a_log), _lib.ptr(dt_bias), state.data_ptr(), state.shape[0], stride,
        out.data_ptr(), None)
    if span._c.chunks:
        size = _lib.load().anna_mi_gated_delta_workspace(ctypes.byref(args), span._ref)
        workspace = torch.empty((size,), dtype=torch.uint8, device=device)
        args.workspace = workspace.data_ptr()
    _call(device, "anna_mi_gated_delta", ctypes.byref(args), span._ref, stream)
    _written(state, out)
    return out


def _rows(what: str, t: torch.Tensor, x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """[..., cols] as rows with one stride; copied where it has none."""
    cols = x.shape[-1]
    if t.dtype != x.dtype or t.shape != x.shape:
        raise ValueError(f"{what} must be {x.dtype} {list(x.shape)}, got {t.dtype} {list(t.shape)}")
    try:
        t = t.view(-1, cols)
    except RuntimeError:
        t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else cols)


def _rows_apart(a: torch.Tensor, a_stride: int, b: torch.Tensor, b_stride: int) -> bool:
    """Whether rows of a and b share no element: of other memory, or other columns of one matrix."""
    size, cols = a.element_size(), a.shape[-1]
    a_bytes, b_bytes = (((t.numel() // cols - 1) * s + cols) * size for t, s in ((a, a_stride), (b, b_stride)))
    between = b.data_ptr() - a.data_ptr()
    if between >= a_bytes or -between >= b_bytes:
        return True
    return a_stride == b_stride and between % size == 0 and cols <= between // size % a_stride <= a_stride - cols


def _norm(x, weight, eps, weight_offset, residual, gate, out, scales, group):
    if x.dim() < 1 or x.dtype not in _lib._DTYPE_CODES or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., cols] in bfloat16, float16 or float32, got {x.dtype} {list(x.shape)}")
    cols = x.shape[-1]
    if weight.dtype != x.dtype or tuple(weight.shape) != (cols,):
        raise ValueError(f"weight must be {x.dtype} [{cols}], got {weight.dtype} {list(weight.shape)}")
    if not 0.0 <= eps < 1e30:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if x.numel() == 0:
        _lib.require_device(x)
        return _on(x.device, x=x, weight=weight, residual=residual, gate=gate, out=out)
    rows, stride = _rows("x", x, x)
    if residual is not None:
        kept, residual_stride = _rows("residual", residual, x)
        if kept.data_ptr() != residual.data_ptr():
            raise ValueError("residual is written in place: its rows must lie at one stride, contiguous in the last dimension")
        same = residual.data_ptr() == x.data_ptr() and residual_stride == stride  # x is then doubled
        for name, t in (("x", None if same else rows), ("gate", gate), ("weight", weight)):
            if t is not None and not _rows_apart(kept, residual_stride, *((t, cols) if t is weight else _rows(name, t, x))):
                raise ValueError(f"residual must not overlap {name}")
    _lib.require_device(x)
    _on(x.device, x=x, weight=weight, residual=residual, gate=gate, out=out)
    args = _lib.RmsNormArgs(dtype=_lib.dtype_code(x.dtype), out_format=int(scales is not None), rows=rows.shape[0], cols=cols,
                            group=group, x=rows.data_ptr(), x_stride=stride, eps=eps, weight_offset=weight_offset)
    weight = weight.contiguous()
    args.weight = weight.data_ptr()
    if residual is not None:
        args.residual, args.residual_stride = kept.data_ptr(), residual_stride
    if gate is not None:
        gate, args.gate_stride = _rows("gate", gate, x)
        args.gate = gate.data_ptr()
    args.out, args.out_stride, args.scales = out.data_ptr(), cols, _lib.ptr(scales)
    _call(x.device, "anna_mi_rms_norm", ctypes.byref(args), _lib.stream_of(x))
    _written(residual, out)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, weight_offset: float = 0.0,
             residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * (weight + weight_offset) over the last dimension, times silu(gate) when
    a gate is given; bf16, fp16 or fp32, sums in fp32.

    residual (same shape): x is added to it first, in place, and the sum, as the type holds it, is what is
    normalised; it may be x itself, and overlaps nothing else.  out (contiguous) may be x or gate themselves, and overlaps nothing else."""
    if out is None:
        if x.is_cuda:
            device = _cuda_device()
            got = _host().rms_norm(x, weight, eps, weight_offset, residual, gate, device, _raw_stream(device))
            if got is not None:
                return got
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        if out.dtype != x.dtype or out.shape != x.shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {x.dtype} {list(x.shape)}")
        same = [n for n, t in (("x", x), ("gate", gate)) if t is not None and t.is_contiguous() and t.data_ptr() == out.data_ptr()]
        _apart(out, **{n: t for n, t in dict(x=x, gate=gate, residual=residual, weight=weight).items() if n not in same})
    _norm(x, weight, float(eps), float(weight_offset), residual, gate, out, None, 0)
    return out


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, weight_offset: float = 0.0,
                  residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  group_size: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """rms_norm in 8 bits: codes float8_e4m3fn of x's shape and scales fp32 [..., cols / group_size], codes * scales
    being the values.  A scale is the largest magnitude of its group / 448 (a group below 2^-100 is held as zeros);
    the values are quantized from fp32.  group_size 32, 64 or 128 (a divisor of cols), or cols (None): a scale a row."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., cols], got {list(x.shape)}")
    cols = x.shape[-1]
    group = cols if group_size is None else operator.index(group_size)
    if group != cols and (group not in E4M3_GROUPS or cols % group):
        raise ValueError(f"group_size {group} of {cols} columns: 32, 64 or 128 (a divisor) or all columns are supported")
    if x.is_cuda:
        device = _cuda_device()
        got = _host().rms_norm_e4m3(x, weight, eps, weight_offset, residual, gate, group, device, _raw_stream(device))
        if got is not None:
            return got
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((*x.shape[:-1], cols // group), dtype=torch.float32, device=x.device)
    _norm(x, weight, float(eps), float(weight_offset), residual, gate, codes, scales, group)
    return codes, scales
