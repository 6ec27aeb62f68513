"""Paged 4-bit KV cache: one pool of pages that sequences of any length share, with attention for any
number of new tokens.

Where TurboQuantBatchCache gives every sequence a fixed region and decodes one token a call, here a
sequence takes 64-token pages from a pool as it grows, sequences with a common beginning share its
pages (``fork``), and one call attends for single tokens, drafted tokens, prompts or chunks of them, mixed as
they come.  Keys and values are held in groups of 64 as 4-bit codes with a bf16 scale and a whole
zero, ``(code + zero) * scale``, 4.5 bits a value; the layout and the rounding are written down in
include/anna_mi.h.

    cache = PagedInt4Cache(num_layers=24, num_pages=4096, kv_heads=2, q_heads=16, head_dim=256,
                           max_sequences=64, max_length=32768)
    seqs = cache.add(2)
    span = cache.extend(seqs, [1000, 37])      # room for a prompt of each, once for all layers
    for layer in range(24):
        cache.store(layer, span, keys, values)  # [1037, kv_heads, head_dim], the prompts one after the other
        out = cache.attend(layer, span, query, scaling=1 / 16)
    span = cache.extend(seqs)                  # the next token of each
    answers = cache.fork([seqs[0]] * 4)        # four continuations of the first

The cache is for inference: tensors that require grad are refused outside ``torch.no_grad()``.  The host
counts pages and lengths; ``extend`` and ``span`` lay out the step's launches once for all layers.  Calls
that share a cache must not overlap on the GPU: run them on one stream, or order the streams.  A step can be
captured in a graph (``store``, ``read`` and ``attend``, not the calls that count): refill its span with
``extend(..., span=span)`` before every replay.
"""

from __future__ import annotations

import ctypes
import operator
import threading
import weakref

import torch

from . import _lib

PAGE_TOKENS = 64
HEAD_DIMS = (64, 128, 256)


def page_bytes(head_dim: int) -> int:
    """Bytes of a page of one KV head: codes, scales and offsets of 64 keys and 64 values."""
    return 72 * head_dim


def _ints(values, ctype):
    values = [operator.index(v) for v in values]
    lo, hi = (-(1 << 31), (1 << 31) - 1) if ctype is ctypes.c_int32 else (-(1 << 63), (1 << 63) - 1)
    for v in values:
        if not lo <= v <= hi:
            raise ValueError(f"{v} is out of range")
    return (ctype * len(values))(*values)


class PagedSpan:
    """Tokens ``starts[i] .. starts[i] + counts[i] - 1`` of sequences ``seqs[i]``, packed one sequence after
    the other: what ``store``, ``read`` and ``attend`` of every layer work on.  Made by
    ``PagedInt4Cache.extend`` and ``span``; it holds the device arrays and the workspace of their launches."""

    def __init__(self, cache: "PagedInt4Cache"):
        self.cache = cache
        self.seqs: list[int] = []
        self.starts: list[int] = []
        self.counts: list[int] = []
        self._c = _lib.PagedSpan()
        self._ref = ctypes.byref(self._c)
        self._address = ctypes.addressof(self._c)
        self._tensors: list[torch.Tensor] = []
        self._streams: set[int] = set()
        self._version = -1
        self._ended: list[int] = []

    @property
    def tokens(self) -> int:
        """Tokens of all sequences."""
        return self._c.tokens

    def _room(self, seqs, starts, counts) -> None:
        """A new span's memory; starts None: of an extend by counts."""
        cache, c = self.cache, self._c
        if c.buf is None:
            cache._call("anna_mi_paged_span_plan", len(seqs), seqs, starts, counts, self._ref)
            buf = torch.empty((c.words,), dtype=torch.int32, device=cache.device)
            c.buf = buf.data_ptr()
            self._tensors = [buf]
            if c.partial_rows > 0:
                stats = torch.empty((c.partial_rows, cache.kv_heads, 2), dtype=torch.float32, device=cache.device)
                values = torch.empty((c.partial_rows, cache.kv_heads, cache.head_dim), dtype=torch.float32,
                                     device=cache.device)
                c.partial_stats, c.partial_values = stats.data_ptr(), values.data_ptr()
                self._tensors += [stats, values]

    def _fill(self, seqs, starts, counts) -> None:
        cache = self.cache
        self._used_on(cache._stream())
        cache._call("anna_mi_paged_span_fill", len(seqs), seqs, starts, counts, self._ref, cache._stream())
        self.seqs, self.starts, self.counts = list(seqs), list(starts), list(counts)
        self._ended, self._version = [cache._ended[s] for s in self.seqs], cache._version

    def _fresh(self, seqs, starts, counts) -> bool:
        """A new span's fill by the host module, on the current device; False for calls that it leaves to the general way."""
        cache = self.cache
        stream = cache._stream()
        got = _lib.host().paged_span(cache._handle.value, self._address, seqs, starts, counts, cache.max_length,
                                     cache.kv_heads, cache.head_dim, cache.device.index, stream)
        if got is None:
            return False
        self.seqs, self.starts, self.counts, self._tensors = got
        self._ended, self._version = [cache._ended[s] for s in self.seqs], cache._version
        self._streams = {stream}
        return True

    def _used_on(self, stream: int) -> None:
        if stream not in self._streams:
            self._streams.add(stream)
            for t in self._tensors:
                t.record_stream(torch.cuda.current_stream(self.cache.device))

    @property
    def rows(self) -> torch.Tensor:
        """The sequences' rows of the page table (int32, on the device)."""
        return self._tensors[0][8:8 + self._c.sequences]


class PagedInt4Cache:
    """``num_pages`` pages of 64 tokens in every one of ``num_layers`` layers, shared by at most
    ``max_sequences`` sequences of at most ``max_length`` tokens.

    ``pool`` uint8 [layers, pages, kv_heads, page_bytes(head_dim)] and ``table`` int32 [max_sequences,
    pages of max_length] are on the device; sequences are named by their row of the table."""

    def __init__(self, *, num_layers: int, num_pages: int, kv_heads: int, q_heads: int, head_dim: int,
                 max_sequences: int, max_length: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"PagedInt4Cache supports head_dim 64, 128 and 256, got {head_dim}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PagedInt4Cache supports bfloat16 and float16, got {dtype}")
        if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads != 0:
            raise ValueError("q_heads must be a multiple of kv_heads")
        if min(num_layers, num_pages, max_sequences, max_length) < 1:
            raise ValueError("num_layers, num_pages, max_sequences and max_length must be positive")
        self.num_layers, self.num_pages = int(num_layers), int(num_pages)
        self.kv_heads, self.q_heads, self.head_dim = int(kv_heads), int(q_heads), int(head_dim)
        self.max_sequences, self.max_length, self.dtype = int(max_sequences), int(max_length), dtype
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedInt4Cache needs a ROCm device, got {device}")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        width = -(-self.max_length // PAGE_TOKENS)
        self.pool = self._new_pool(self.num_pages, zero=True)
        self.table = torch.zeros((self.max_sequences, width), dtype=torch.int32, device=self.device)
        self._version = 0  # counts the calls after which a span may name tokens that are no more
        self._ended = [0] * self.max_sequences  # how often a row's sequence has ended
        self._streams: set[int] = set()  # that the pool and the table are used on
        d = _lib.PagedDesc(_lib.dtype_code(dtype), self.num_layers, self.num_pages, self.kv_heads, self.q_heads,
                           self.head_dim, self.max_sequences, width, self.pool.data_ptr(), self.table.data_ptr())
        self._handle = ctypes.c_void_p()
        self._lock = threading.RLock()
        _lib.call("anna_mi_paged_create", ctypes.byref(d), ctypes.byref(self._handle))
        weakref.finalize(self, _lib.load().anna_mi_paged_destroy, self._handle)

    def _new_pool(self, pages: int, zero: bool) -> torch.Tensor:
        make = torch.zeros if zero else torch.empty
        return make((self.num_layers, pages, self.kv_heads, page_bytes(self.head_dim)), dtype=torch.uint8,
                    device=self.device)

    # ---- calls
    def _stream(self) -> int:
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        if stream not in self._streams:
            self._streams.add(stream)
            for t in (self.pool, self.table):
                t.record_stream(torch.cuda.current_stream(self.device))
        return stream

    def _call(self, name: str, *args) -> None:
        if self._here():
            _lib.call(name, self._handle, *args)
        else:
            with torch.cuda.device(self.device):
                _lib.call(name, self._handle, *args)

    def _here(self) -> bool:
        """Whether the cache's device is the current one, which the host module's calls take for granted."""
        return torch.cuda.current_device() == self.device.index

    def _capturing_there(self) -> bool:
        """Whether the current stream of the cache's device, which is not the current one, records a graph."""
        with torch.cuda.device(self.device):
            return torch.cuda.is_current_stream_capturing()

    def _counts(self, what: str) -> bool:
        """For calls that count on the host -> whether the cache's device is the current one."""
        here = self._here()
        if torch.cuda.is_current_stream_capturing() if here else self._capturing_there():
            # lengths and pages are counted on the host: a replay would not count again
            raise RuntimeError(f"PagedInt4Cache.{what} cannot be captured in a graph")
        return here

    # ---- sequences
    def add(self, n: int = 1) -> list[int]:
        """n new, empty sequences."""
        n = operator.index(n)
        if n < 0:
            raise ValueError(f"cannot add {n} sequences")
        seqs = (ctypes.c_int32 * n)()
        self._call("anna_mi_paged_add", n, seqs)
        return list(seqs)

    def fork(self, parents) -> list[int]:
        """A new sequence for every listed one (which may repeat), holding the same tokens in the same pages.
        A page is copied when one of the sequences that share it grows into it."""
        if self._counts("fork"):
            children = _lib.host().paged_fork(self._handle.value, parents, self._stream())
            if children is not None:
                return children
        parents = _ints(parents, ctypes.c_int32)
        children = (ctypes.c_int32 * len(parents))()
        self._call("anna_mi_paged_fork", len(parents), parents, children, self._stream())
        return list(children)

    def extend(self, seqs, counts=None, *, span: PagedSpan | None = None) -> PagedSpan:
        """Lengthens sequences by ``counts`` tokens (one each by default, 0 allowed) and returns the span of
        the new tokens, which the caller then stores in every layer.  Nothing changes if the pool has
        too few pages or the span no memory.  ``span``: an earlier span of as many sequences with the same counts, which is
        filled again in place (a captured graph holds its addresses)."""
        here = self._counts("extend")
        if here and span is None:
            span = PagedSpan(self)
            with self._lock:
                if span._fresh(seqs, None, counts):
                    return span
            span = None
        seqs = _ints(seqs, ctypes.c_int32)
        counts = _ints([1] * len(seqs) if counts is None else counts, ctypes.c_int64)
        if len(counts) != len(seqs):
            raise ValueError(f"{len(seqs)} sequences and {len(counts)} counts")
        if any(n < 0 for n in counts):
            raise ValueError("counts must not be negative")
        span = self._refilled(span, seqs, counts)
        with self._lock:
            starts = self._lengths(seqs)
            for s, have, n in zip(seqs, starts, counts):
                if have + n > self.max_length:
                    raise RuntimeError(f"sequence {s} would hold {have + n} tokens, max_length is {self.max_length}")
            span._room(seqs, None, counts)  # before anything changes
            self._call("anna_mi_paged_extend", len(seqs), seqs, counts, starts, self._stream())
            span._fill(seqs, starts, counts)
        return span

    def span(self, seqs, starts, counts, *, span: PagedSpan | None = None) -> PagedSpan:
        """The span of tokens that the sequences hold already: to store them anew, read them, or attend for them."""
        here = self._counts("span")
        if here and span is None:
            span = PagedSpan(self)
            with self._lock:
                if starts is not None and counts is not None and span._fresh(seqs, starts, counts):
                    return span
            span = None
        seqs, starts, counts = _ints(seqs, ctypes.c_int32), _ints(starts, ctypes.c_int64), _ints(counts, ctypes.c_int64)
        if not len(seqs) == len(starts) == len(counts):
            raise ValueError(f"{len(seqs)} sequences, {len(starts)} starts and {len(counts)} counts")
        span = self._refilled(span, seqs, counts)
        with self._lock:
            span._room(seqs, starts, counts)
            span._fill(seqs, starts, counts)
        return span

    def _refilled(self, span: PagedSpan | None, seqs, counts) -> PagedSpan:
        if span is None:
            return PagedSpan(self)
        if span.cache is not self:
            raise ValueError("the span belongs to another cache")
        if len(seqs) != len(span.seqs) or list(counts) != span.counts:
            raise ValueError("a span is filled again with as many sequences and the same counts")
        return span

    def truncate(self, seq: int, length: int) -> None:
        """Forgets the tokens of a sequence from ``length`` on (drafted tokens that were not accepted)."""
        self._counts("truncate")
        seqs, length = _ints([seq], ctypes.c_int32), _ints([length], ctypes.c_int64)
        with self._lock:
            self._call("anna_mi_paged_truncate", seqs[0], length[0], self._stream())
            self._version += 1

    def free(self, seqs) -> None:
        """Ends sequences; pages that no other sequence shares return to the pool."""
        here = self._counts("free")
        seqs = list(seqs)
        with self._lock:
            if not (here and _lib.host().paged_free(self._handle.value, seqs, self._stream())):
                seqs = _ints(seqs, ctypes.c_int32)
                self._call("anna_mi_paged_free", len(seqs), seqs, self._stream())
            for s in seqs:
                self._ended[s] += 1
            self._version += 1

    def _lengths(self, seqs):
        lengths = (ctypes.c_int64 * len(seqs))()
        _lib.call("anna_mi_paged_lengths", self._handle, len(seqs), seqs, lengths, None)
        for s, n in zip(seqs, lengths):
            if n < 0:
                raise RuntimeError(f"sequence {s} is not in use")
        return lengths

    def lengths(self, seqs) -> list[int]:
        """Tokens that the sequences hold."""
        return list(self._lengths(_ints(seqs, ctypes.c_int32)))

    @property
    def pages_in_use(self) -> int:
        live = ctypes.c_int64()
        _lib.call("anna_mi_paged_lengths", self._handle, 0, None, None, ctypes.byref(live))
        return live.value

    @property
    def free_pages(self) -> int:
        return self.num_pages - self.pages_in_use

    # ---- the pool
    def compact(self) -> int:
        """Moves the pages in use to the front of the pool, in place, and returns their number."""
        self._counts("compact")
        live = ctypes.c_int64()
        self._call("anna_mi_paged_compact", ctypes.byref(live), self._stream())
        return live.value

    def resize(self, num_pages: int) -> None:
        """A pool of another size: the pages in use, in the sequences' order, move to the front of a new
        ``pool``.  Graphs that were captured before hold the old one: capture them anew."""
        self._counts("resize")
        num_pages = operator.index(num_pages)
        with self._lock:
            if num_pages < max(1, self.pages_in_use):
                raise RuntimeError(f"{num_pages} pages asked, {self.pages_in_use} are in use")
            pool = self._new_pool(num_pages, zero=False)
            self._call("anna_mi_paged_resize", num_pages, pool.data_ptr(), self._stream())
            self.pool, self.num_pages, self._streams = pool, num_pages, {self._stream()}

    def page_table(self, span: PagedSpan) -> torch.Tensor:
        """The pages of the span's sequences, int32 [sequences, pages of max_length], 0 behind the last."""
        return self.table.index_select(0, span.rows)

    # ---- tokens
    def _check(self, what: str, layer: int, span: PagedSpan) -> int:
        if span.cache is not self:
            raise ValueError(f"{what}: the span belongs to another cache")
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"{what}: layer {layer} of {self.num_layers}")
        version = self._version
        if span._version != version:
            if span._ended != [self._ended[s] for s in span.seqs]:
                raise RuntimeError(f"{what}: a sequence of the span is not in use any more")
            lengths = self._lengths((ctypes.c_int32 * len(span.seqs))(*span.seqs))
            for s, start, n, have in zip(span.seqs, span.starts, span.counts, lengths):
                if start + n > have:
                    raise RuntimeError(f"{what}: sequence {s} holds {have} tokens, the span reaches to {start + n}")
            span._version = version
        stream = self._stream()
        span._used_on(stream)
        return stream

    def _rows(self, what: str, t: torch.Tensor, span: PagedSpan, heads: int) -> torch.Tensor:
        shape = (span._c.tokens, heads, self.head_dim)
        if t.dtype != self.dtype or tuple(t.shape) != shape:
            raise ValueError(f"{what} must be {self.dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
        if t.device != self.device:
            raise RuntimeError(f"{what} must be on {self.device}, got a tensor on {t.device}")
        self._no_grad(what, t)
        # rows are read 16 bytes at a time; the stride of a single token or head is read by nobody
        if (t.stride(2) != 1 or t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 8)
                or (heads > 1 and t.stride(1) % 8)):
            return t.clone(memory_format=torch.contiguous_format)
        return t

    @staticmethod
    def _no_grad(what: str, t: torch.Tensor) -> None:
        if t.requires_grad and torch.is_grad_enabled():
            # an answer without a graph would lose its gradient without a word
            raise RuntimeError(f"{what} requires grad, but the cache has no backward pass: call it under torch.no_grad()")

    @staticmethod
    def _strides(t: torch.Tensor) -> tuple[int, int]:
        return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)

    def store(self, layer: int, span: PagedSpan, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Quantizes the span's keys and values [tokens, kv_heads, head_dim] into the layer's pages.  Refused where
        tokens of two of the span's sequences stand in one page."""
        stream, here = self._check("store", layer, span), self._here()
        capturing = torch.cuda.is_current_stream_capturing() if here else self._capturing_there()
        if here and _lib.host().paged_store(self._handle.value, layer, span._address, keys, values, self.pool, self.dtype,
                                            self.head_dim, capturing, stream):
            return
        keys, values = self._rows("keys", keys, span, self.kv_heads), self._rows("values", values, span, self.kv_heads)
        self._call("anna_mi_paged_store", layer, span._ref, keys.data_ptr(), *self._strides(keys), values.data_ptr(),
                   *self._strides(values), capturing, stream)

    def read(self, layer: int, span: PagedSpan) -> tuple[torch.Tensor, torch.Tensor]:
        """The span's keys and values as the cache holds them, dense [tokens, kv_heads, head_dim]."""
        stream, here = self._check("read", layer, span), self._here()
        capturing = torch.cuda.is_current_stream_capturing() if here else self._capturing_there()
        if here:
            return _lib.host().paged_read(self._handle.value, layer, span._address, self.pool, self.dtype, self.head_dim,
                                          capturing, stream)
        keys, values = (torch.empty((span._c.tokens, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
                        for _ in range(2))
        self._call("anna_mi_paged_read", layer, span._ref, keys.data_ptr(), values.data_ptr(), capturing, stream)
        return keys, values

    def attend(self, layer: int, span: PagedSpan, query: torch.Tensor, *, scaling: float,
               gate: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention for the span's tokens: query [tokens, q_heads, head_dim] over all tokens of its
        sequence up to and with its own -> the same shape.  gate (optional, same shape as query): out *= sigmoid(gate).
        out may be the query or the gate."""
        stream, here = self._check("attend", layer, span), self._here()
        capturing = torch.cuda.is_current_stream_capturing() if here else self._capturing_there()
        if here:
            got = _lib.host().paged_attend(self._handle.value, layer, span._address, query, gate, out, self.pool, self.dtype,
                                           self.q_heads, self.head_dim, scaling, capturing, stream)
            if got is not None:
                return got
        if not 0.0 < scaling < 1e30:
            raise ValueError(f"scaling must be positive and finite, got {scaling}")
        query = self._rows("query", query, span, self.q_heads)
        if gate is not None:
            gate = self._rows("gate", gate, span, self.q_heads)
        if out is None:
            out = torch.empty((span._c.tokens, self.q_heads, self.head_dim), dtype=self.dtype, device=self.device)
        elif (out.dtype != self.dtype or tuple(out.shape) != tuple(query.shape) or out.device != self.device
              or not out.is_contiguous() or out.data_ptr() % 16):
            raise ValueError(f"out must be a contiguous, 16-byte aligned {self.dtype} tensor of the query's shape")
        else:
            self._no_grad("out", out)
        self._call("anna_mi_paged_attend", layer, span._ref, query.data_ptr(), *self._strides(query),
                   None if gate is None else gate.data_ptr(), *((0, 0) if gate is None else self._strides(gate)),
                   out.data_ptr(), scaling, capturing, stream)
        return out
