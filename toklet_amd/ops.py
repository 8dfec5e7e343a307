"""Device attention operators with the reference's operator interface.

Each function mirrors one toklet operator (same names, shape structs,
argument meaning and error behaviour) and calls libtokhip through its C ABI.
Tensors are torch tensors in device memory; torch supplies allocation and
the stream, the kernels are the library's.

    toklet                                   this module
    cpu::attention_cached (attention.rs:201)  attention_cached
    cpu::attention        (attention.rs:85)   attention
    cpu::window_attention (window_attention.rs:36)  window_attention
    cpu::span_attention   (span_attention.rs:42)    span_attention
    cpu::logit_softcap    (softcap.rs:16)     logit_softcap

Errors raise :class:`TkhError` carrying the code of the matching
``toklet::cpu::Error`` variant.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class TkhError(Exception):
    def __init__(self, err: _lib.Error):
        self.code = int(err.code)
        self.name = _lib.CODE_NAMES.get(self.code, str(self.code))
        self.tensor = err.tensor.decode(errors="replace")
        self.index = int(err.index)
        self.expected = int(err.expected)
        self.actual = int(err.actual)
        self.message = err.message.decode(errors="replace")
        super().__init__(f"{self.name}: {self.message}")


def _check(rc: int, err: _lib.Error):
    if rc != _lib.OK:
        raise TkhError(err)


class Context:
    """One device stream, workspace and status word (tkh_context)."""

    def __init__(self, device: int = 0, stream: Optional[torch.cuda.Stream] = None,
                 workspace_bytes: int = 0, synchronous: bool = True):
        lib = _lib.load()
        if stream is None:
            stream = torch.cuda.current_stream(device)
        self.device = device
        self.torch_stream = stream
        # Where the paged operators' errors go: a fresh structure per call costs as
        # much as the rest of the call, and a context serves one thread.
        self.paged_error = _lib.Error()
        handle = ctypes.c_void_p()
        err = _lib.Error()
        _check(lib.tkh_context_create(device, ctypes.c_void_p(stream.cuda_stream), workspace_bytes,
                                      int(synchronous), ctypes.byref(handle), ctypes.byref(err)), err)
        self.handle = handle
        _lib.track(self, _lib.CONTEXT)

    def synchronize(self):
        err = _lib.Error()
        _check(_lib.load().tkh_context_synchronize(self.handle, ctypes.byref(err)), err)

    def profile(self, enable: bool = True):
        """Start (and zero) or stop per-launch HIP-event timing of the kernels."""
        err = _lib.Error()
        _check(_lib.load().tkh_context_profile(self.handle, int(enable), ctypes.byref(err)), err)

    def profile_read(self) -> dict:
        """{'launches', 'attention_ms', 'combine_ms'} summed since profile(True)."""
        out = _lib.Profile()
        err = _lib.Error()
        _check(_lib.load().tkh_context_profile_read(self.handle, ctypes.byref(out),
                                                    ctypes.byref(err)), err)
        return {"launches": int(out.launches), "attention_ms": float(out.attention_ms),
                "combine_ms": float(out.combine_ms)}

    def close(self):
        if getattr(self, "handle", None):
            _lib.load().tkh_context_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- shape structs (reference field names) ----

@dataclass
class CachedAttentionShape:
    """src/cpu/attention.rs:180-189"""
    tokens: int
    query_heads: int
    kv_heads: int
    head_dim: int
    capacity: int
    offset: int


@dataclass
class AttentionShape:
    """src/cpu/attention.rs:67-72"""
    tokens: int
    query_heads: int
    kv_heads: int
    head_dim: int


@dataclass
class WindowAttentionShape:
    """src/cpu/window_attention.rs:6-17, plus the score softcap (0 disables)."""
    queries: int
    keys: int
    capacity: int
    query_heads: int
    kv_heads: int
    head_dim: int
    query_start: int
    key_start: int
    window: Optional[int]
    scale: float
    softcap: float = 0.0


@dataclass
class AttentionKvSegment:
    """src/cpu/span_attention.rs:9-16 (k/v are device tensors or None when keys == 0)."""
    k: Optional[torch.Tensor]
    v: Optional[torch.Tensor]
    keys: int
    head_stride: int
    key_start: int


@dataclass
class SpanAttentionShape:
    """src/cpu/span_attention.rs:18-28, plus the score softcap."""
    queries: int
    keys: int
    query_heads: int
    kv_heads: int
    head_dim: int
    query_start: int
    key_start: int
    window: Optional[int]
    scale: float
    softcap: float = 0.0


# A call through these bindings costs about as much as a launch, so the argument
# helpers avoid building ctypes objects: addresses go as plain integers.
def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _fptr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if t.dtype is not torch.float32:
        raise TypeError("outputs are float32 tensors")
    return t.data_ptr()


def _n(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.numel()


def dtype_of(*tensors: torch.Tensor) -> int:
    dt = None
    for t in tensors:
        if t is not None and t.dtype is not dt:
            if dt is not None:
                raise TypeError(f"q/k/v must share one dtype, got {({x.dtype for x in tensors if x is not None})}")
            dt = t.dtype
    code = _DTYPES.get(dt)
    if code is None:
        raise TypeError(f"unsupported dtype {dt}")
    return code


def _window(window):
    return (0, 0) if window is None else (1, int(window))


def attention_cached(ctx: Context, q, k, v, context, scores, probabilities,
                     shape: CachedAttentionShape):
    """Chunk queries over a head-major cache (reference: attention_cached)."""
    err = _lib.Error()
    s = _lib.CachedShape(shape.tokens, shape.query_heads, shape.kv_heads, shape.head_dim,
                         shape.capacity, shape.offset)
    rc = _lib.load().tkh_attention_cached(
        ctx.handle, ctypes.byref(s), dtype_of(q, k, v), _ptr(q), _n(q), _ptr(k), _n(k), _ptr(v),
        _n(v), _fptr(context), _n(context), _fptr(scores), _n(scores), _fptr(probabilities),
        _n(probabilities), ctypes.byref(err))
    _check(rc, err)


def attention_cached_static(device: int, q, k, v, context, shape: CachedAttentionShape,
                            stream: Optional[torch.cuda.Stream] = None,
                            status: Optional[torch.Tensor] = None):
    """attention_cached without a context or any allocation: split-K partials in
    the library's fixed per-GPU scratch (tkh_attention_cached_static).  `status`:
    an int32 device tensor of one element the kernels OR their status bits into
    (the call then returns once queued), or None to wait and raise on failure."""
    err = _lib.Error()
    s = _lib.CachedShape(shape.tokens, shape.query_heads, shape.kv_heads, shape.head_dim,
                         shape.capacity, shape.offset)
    if stream is None:
        stream = torch.cuda.current_stream(device)
    st = _ptr(status)
    rc = _lib.load().tkh_attention_cached_static(
        device, ctypes.c_void_p(stream.cuda_stream), ctypes.byref(s), dtype_of(q, k, v), _ptr(q),
        _n(q), _ptr(k), _n(k), _ptr(v), _n(v), _fptr(context), _n(context), st, ctypes.byref(err))
    _check(rc, err)


def attention(ctx: Context, q, k, v, context, scores, probabilities, shape: AttentionShape):
    """Full-prefix causal GQA with token-major K/V (reference: attention)."""
    err = _lib.Error()
    s = _lib.AttentionShape(shape.tokens, shape.query_heads, shape.kv_heads, shape.head_dim)
    rc = _lib.load().tkh_attention(
        ctx.handle, ctypes.byref(s), dtype_of(q, k, v), _ptr(q), _n(q), _ptr(k), _n(k), _ptr(v),
        _n(v), _fptr(context), _n(context), _fptr(scores), _n(scores), _fptr(probabilities),
        _n(probabilities), ctypes.byref(err))
    _check(rc, err)


def window_attention(ctx: Context, q, k, v, context, scores, probabilities,
                     shape: WindowAttentionShape):
    """Causal/sliding GQA with explicit scale (reference: window_attention)."""
    err = _lib.Error()
    hw, w = _window(shape.window)
    s = _lib.WindowShape(shape.queries, shape.keys, shape.capacity, shape.query_heads,
                         shape.kv_heads, shape.head_dim, shape.query_start, shape.key_start, hw, w,
                         shape.scale, shape.softcap)
    rc = _lib.load().tkh_window_attention(
        ctx.handle, ctypes.byref(s), dtype_of(q, k, v), _ptr(q), _n(q), _ptr(k), _n(k), _ptr(v),
        _n(v), _fptr(context), _n(context), _fptr(scores), _n(scores), _fptr(probabilities),
        _n(probabilities), ctypes.byref(err))
    _check(rc, err)


def span_attention(ctx: Context, q, segments: Sequence[AttentionKvSegment], context, scores,
                   probabilities, shape: SpanAttentionShape):
    """GQA over <=2 old ring spans plus the staged chunk (reference: span_attention)."""
    err = _lib.Error()
    segs = (_lib.Segment * 3)()
    tensors = [q] + [t for sg in segments for t in (sg.k, sg.v) if t is not None]
    for i, sg in enumerate(segments):
        segs[i] = _lib.Segment(_ptr(sg.k), _n(sg.k), _ptr(sg.v), _n(sg.v), sg.keys,
                               sg.head_stride, sg.key_start)
    hw, w = _window(shape.window)
    s = _lib.SpanShape(shape.queries, shape.keys, shape.query_heads, shape.kv_heads,
                       shape.head_dim, shape.query_start, shape.key_start, hw, w, shape.scale,
                       shape.softcap)
    rc = _lib.load().tkh_span_attention(
        ctx.handle, ctypes.byref(s), dtype_of(*tensors), _ptr(q), _n(q), segs, _fptr(context),
        _n(context), _fptr(scores), _n(scores), _fptr(probabilities), _n(probabilities),
        ctypes.byref(err))
    _check(rc, err)


def project_greedy(ctx: Context, context: torch.Tensor, weights: torch.Tensor,
                   tokens: torch.Tensor, logits: Optional[torch.Tensor] = None):
    """The o-projection of FP32 context rows [rows, hidden] by weights [vocab, hidden]
    in the reference matmul's FP32 order, then the greedy token of each row
    (reference: cpu::matmul + sampling::greedy).  tokens: int32 device tensor
    [rows] (holding the uint32 ids); logits: optional FP32 [rows, vocab]."""
    err = _lib.Error()
    rows, hidden = context.shape[0], context.shape[-1]
    vocab = weights.shape[0]
    if tokens.dtype != torch.int32:
        raise TypeError("tokens is an int32 tensor (uint32 ids)")
    rc = _lib.load().tkh_project_greedy(
        ctx.handle, rows, hidden, vocab, _fptr(context), _n(context), _fptr(weights), _n(weights),
        _fptr(logits), _n(logits), _ptr(tokens), _n(tokens), ctypes.byref(err))
    _check(rc, err)


def logit_softcap(ctx: Context, logits: torch.Tensor, cap: float):
    """In-place cap*tanh(x/cap) in FP64 rounded to FP32 (reference: logit_softcap)."""
    err = _lib.Error()
    rc = _lib.load().tkh_logit_softcap(ctx.handle, _fptr(logits), _n(logits), cap,
                                       ctypes.byref(err))
    _check(rc, err)


def _u64s(values):
    arr = (ctypes.c_uint64 * len(values))(*[int(x) for x in values])
    return arr


def decode_batch(ctx: Context, q, k_base, v_base, offsets, head_strides, lengths, context, *,
                 query_heads: int, kv_heads: int, head_dim: int, scale: float):
    """One query token per session over its own head-major cache (tkh_decode_batch)."""
    err = _lib.Error()
    batch = len(lengths)
    rc = _lib.load().tkh_decode_batch(
        ctx.handle, batch, query_heads, kv_heads, head_dim, dtype_of(q, k_base, v_base), _ptr(q),
        _ptr(k_base), _ptr(v_base), _u64s(offsets), _u64s(head_strides), _u64s(lengths), scale,
        _fptr(context), ctypes.byref(err))
    _check(rc, err)


def prefill_batch(ctx: Context, q, k_base, v_base, offsets, head_strides, positions, context, *,
                  tokens: int, query_heads: int, kv_heads: int, head_dim: int, scale: float):
    """A causal chunk of `tokens` queries per session at cache offset positions[b]."""
    err = _lib.Error()
    batch = len(positions)
    rc = _lib.load().tkh_prefill_batch(
        ctx.handle, batch, tokens, query_heads, kv_heads, head_dim, dtype_of(q, k_base, v_base),
        _ptr(q), _ptr(k_base), _ptr(v_base), _u64s(offsets), _u64s(head_strides),
        _u64s(positions), scale, _fptr(context), ctypes.byref(err))
    _check(rc, err)


# ---- producer: the step before attention (Model::run, src/model/mod.rs:611-662) ----

ROTARY_NONE, ROTARY_SPLIT_HALF, ROTARY_PROPORTIONAL, ROTARY_LLAMA3 = 0, 1, 2, 3


@dataclass
class ProducerShape:
    """Per-layer producer geometry: norm epsilon, rotary kind and its parameters
    (split-half theta; proportional base / rotated_dims / factor; Llama 3 theta,
    factor, low/high frequency factors and original context length, as
    Llama3Scaling::new takes them, src/cpu/llama3_rotary.rs:14-37)."""
    tokens: int
    query_heads: int
    kv_heads: int
    head_dim: int
    position: int
    norm_epsilon: float = 1e-6
    rotary: int = ROTARY_SPLIT_HALF
    theta: float = 1e6
    rotated_dims: int = 0
    factor: float = 1.0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    original_max_positions: int = 8192

    def c(self):
        return _lib.ProducerShape(self.tokens, self.query_heads, self.kv_heads, self.head_dim,
                                  self.position, self.norm_epsilon, self.rotary, self.theta,
                                  self.rotated_dims, self.factor, self.low_freq_factor,
                                  self.high_freq_factor, self.original_max_positions)


def produce_qkv(ctx: Context, shape: ProducerShape, q_proj, k_proj, v_proj, q_norm, k_norm,
                q_out, k_out, v_out, out_head_stride: int):
    """rmsnorm (optional) -> rotary -> rounding of Q, and the K/V append into head-major
    rows, in one launch.  k_out/v_out may be views into a cache at a row offset."""
    err = _lib.Error()
    s = shape.c()
    rc = _lib.load().tkh_produce_qkv(
        ctx.handle, ctypes.byref(s), dtype_of(q_out, k_out, v_out), _ptr(q_proj), _ptr(k_proj),
        _ptr(v_proj), _ptr(q_norm), _ptr(k_norm), _ptr(q_out), _ptr(k_out), _ptr(v_out),
        out_head_stride, ctypes.byref(err))
    _check(rc, err)


# ---- paged caches (no counterpart in the reference)

_ROPE_LAYOUTS = {"none": 0, "half": 1, "interleaved": 2}
_ROPE_SCALINGS = {"none": 0, "linear": 1, "bands": 2}


@dataclass
class PagedBatch:
    """A ragged batch over a paged cache (tkh_paged_batch).  The tensors are int32 on
    the device and are read by each launch: page_table [rows, columns] (rows may be
    strided), key_lens [rows], query_start [sequences + 1] or None (max_queries rows
    each), slots [sequences] (a sequence's table row) or None.  The integers bound
    what the tensors may hold."""
    page_table: torch.Tensor
    key_lens: torch.Tensor
    total_queries: int
    max_queries: int
    max_keys: int
    query_start: Optional[torch.Tensor] = None
    slots: Optional[torch.Tensor] = None

    def _c(self, device: int):
        table, lens, start, slots = self.page_table, self.key_lens, self.query_start, self.slots
        for t in (table, lens, start, slots):
            if t is not None and (t.dtype is not torch.int32 or t.get_device() != device):
                raise TypeError("a batch's tensors are int32 on the context's device")
        rows, columns = table.shape
        # Rows may lie further apart than their columns.
        stride, inner = table.stride()
        if rows == 1:
            stride = columns
        if (inner != 1 and columns > 1) or stride < columns:
            raise ValueError("page_table rows are contiguous and apart from each other")
        if lens.shape != (rows,) or not lens.is_contiguous():
            raise ValueError("page_table and key_lens have one row per sequence slot")
        sequences = rows
        if slots is not None:
            if slots.dim() != 1 or not slots.is_contiguous():
                raise ValueError("slots is contiguous [sequences]")
            sequences = slots.shape[0]
        if start is not None:
            if start.dim() != 1 or not start.is_contiguous() or start.shape[0] < 1:
                raise ValueError("query_start is contiguous [sequences + 1]")
            if slots is not None and start.shape[0] != sequences + 1:
                raise ValueError("slots and query_start disagree")
            sequences = start.shape[0] - 1
        if self.max_keys < 1 or self.max_queries < 1 or self.total_queries < 0:
            raise ValueError("a batch's bounds are positive")
        return _lib.PagedBatch(sequences, self.total_queries, self.max_queries, self.max_keys, rows, stride,
                               table.data_ptr(), lens.data_ptr(), None if start is None else start.data_ptr(),
                               None if slots is None else slots.data_ptr())


@dataclass
class RotaryPositions:
    """Rotary positions of a paged producer (tkh_rope).  layout: "none", "half" (pairs
    j, j + rotated_dims/2) or "interleaved" (2j, 2j + 1); rotated_dims 0: all of the
    head; scaling: "none", "linear" (frequencies / factor) or "bands" (kept, blended or
    divided by how many rotations original_max_positions hold); magnitude multiplies
    sine and cosine."""
    layout: str = "half"
    rotated_dims: int = 0
    theta: float = 1e6
    scaling: str = "none"
    factor: float = 1.0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    original_max_positions: int = 8192
    magnitude: float = 1.0

    def _c(self):
        if self.layout not in _ROPE_LAYOUTS or self.scaling not in _ROPE_SCALINGS:
            raise ValueError(f"rotary layout {self.layout!r}, scaling {self.scaling!r}")
        return _lib.Rope(_ROPE_LAYOUTS[self.layout], _ROPE_SCALINGS[self.scaling], self.rotated_dims,
                         self.theta, self.factor, self.low_freq_factor, self.high_freq_factor,
                         self.magnitude, self.original_max_positions)


def _paged_dtype(ctx: Context, t: torch.Tensor, *others) -> int:
    """The one dtype of tensors on the context's device."""
    dt, device = t.dtype, ctx.device
    if t.get_device() != device:
        raise ValueError("a tensor is not on the context's device")
    for x in others:
        if x.dtype is not dt:
            raise TypeError("the tensors share one dtype")
        if x.get_device() != device:
            raise ValueError("a tensor is not on the context's device")
    code = _DTYPES.get(dt)
    if code is None:
        raise TypeError(f"unsupported dtype {dt}")
    return code


def _paged_layout(k_pages: torch.Tensor, v_pages: torch.Tensor):
    """The layout of page tensors [pages, kv_heads, page_tokens, head_dim] (any strides
    with contiguous rows) and the elements from their first on."""
    shape, strides = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or strides != v_pages.stride():
        raise ValueError("k_pages and v_pages are [pages, kv_heads, page_tokens, head_dim] alike")
    pages, heads, tokens, dims = shape
    ps, hs, rs, inner = strides
    if inner != 1:
        raise ValueError("page rows are contiguous")
    if pages == 1:  # torch leaves these strides open
        ps = 0
    if heads == 1:
        hs = 0
    extent = (pages - 1) * ps + (heads - 1) * hs + (tokens - 1) * rs + dims if k_pages.numel() else 0
    return _lib.PagedLayout(pages, tokens, heads, dims, ps, hs, rs), heads, dims, extent


def _rows(t: torch.Tensor, tokens: int, heads: int, dims: int):
    """Stride and extent of a token-major [tokens, heads, dims] tensor whose tokens are contiguous."""
    if t.shape != (tokens, heads, dims):
        raise ValueError(f"a projection is [{tokens}, {heads}, {dims}], not {list(t.shape)}")
    stride, head, inner = t.stride()
    row = heads * dims
    if tokens <= 1:
        stride = row
    if tokens and (inner != 1 or (heads > 1 and head != dims)):
        raise ValueError("a projection's token has its heads side by side")
    return stride, (tokens - 1) * stride + row if tokens else 0


def paged_attention(ctx: Context, batch: PagedBatch, q, k_pages, v_pages, context, *, scale: float,
                    window: Optional[int] = None, softcap: float = 0.0):
    """Causal GQA of a ragged batch's new tokens over their pages (tkh_paged_attention).
    q/context: [total_queries, query_heads, head_dim], in the pages' dtype."""
    dt = _paged_dtype(ctx, q, k_pages, v_pages, context)
    layout, _, dims, extent = _paged_layout(k_pages, v_pages)
    shape = q.shape
    if len(shape) != 3 or shape[2] != dims or shape != context.shape:
        raise ValueError("q and context are [total_queries, query_heads, head_dim]")
    if not q.is_contiguous() or not context.is_contiguous():
        raise ValueError("q and context are contiguous")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError("window is at least 1 (None: no window)")
    n, err = shape[0] * shape[1] * dims, ctx.paged_error
    rc = _lib.load().tkh_paged_attention(
        ctx.handle, batch._c(ctx.device), layout, shape[1], dt, q.data_ptr(), n, k_pages.data_ptr(), extent,
        v_pages.data_ptr(), extent, scale, window, softcap, context.data_ptr(), n, err)
    if rc != _lib.OK:
        raise TkhError(err)


def paged_produce(ctx: Context, batch: PagedBatch, rotary: RotaryPositions, q_proj, k_proj, v_proj, q_norm,
                  k_norm, q_out, k_pages, v_pages, norm_epsilon: float = 1e-6):
    """RMSNorm (optional), rotary and rounding of a ragged batch's new rows: Q to q_out
    [total_queries, query_heads, head_dim], K and V into their pages (tkh_paged_produce).
    Projections: [total_queries, heads, head_dim] in one dtype, tokens at any stride."""
    dt = _paged_dtype(ctx, q_out, k_pages, v_pages)
    src = _paged_dtype(ctx, q_proj, k_proj, v_proj)
    layout, hkv, dims, extent = _paged_layout(k_pages, v_pages)
    if q_out.dim() != 3 or not q_out.is_contiguous():
        raise ValueError("q_out is contiguous [total_queries, query_heads, head_dim]")
    tokens, hq, _ = q_out.shape
    qs, qn = _rows(q_proj, batch.total_queries, hq, dims)
    ks, kn = _rows(k_proj, batch.total_queries, hkv, dims)
    vs, vn = _rows(v_proj, batch.total_queries, hkv, dims)
    norms = [None, None]
    for i, w in enumerate((q_norm, k_norm)):
        if w is None:
            continue
        if w.dtype is not torch.float32 or w.shape != (dims,) or not w.is_contiguous() or w.get_device() != ctx.device:
            raise ValueError("norm weights are float32 [head_dim] on the context's device")
        norms[i] = w.data_ptr()
    proj = _lib.PagedProjections(q_proj.data_ptr(), k_proj.data_ptr(), v_proj.data_ptr(), qs, ks, vs, qn, kn, vn,
                                 norms[0], norms[1], norm_epsilon)
    err = ctx.paged_error
    rc = _lib.load().tkh_paged_produce(
        ctx.handle, batch._c(ctx.device), layout, rotary._c(), hq, src, proj, dt, q_out.data_ptr(), tokens * hq * dims,
        k_pages.data_ptr(), extent, v_pages.data_ptr(), extent, err)
    if rc != _lib.OK:
        raise TkhError(err)


def copy_pages(ctx: Context, pool: torch.Tensor, src, dst):
    """pool[:, dst[i]] = pool[:, src[i]] for each i in order (tkh_copy_pages).  pool:
    [planes, pages, ...] with contiguous pages; src/dst: integers, or int64 CPU tensors."""
    _paged_dtype(ctx, pool)
    if pool.dim() < 3 or pool.numel() == 0 or not pool[0, 0].is_contiguous():
        raise ValueError("pool is [planes, pages, ...] with contiguous pages")
    lists = []
    for t in (src, dst):
        if not isinstance(t, torch.Tensor):
            t = torch.tensor(list(t), dtype=torch.int64)
        if t.dtype is not torch.int64 or t.get_device() != -1 or t.dim() != 1 or not t.is_contiguous():
            raise TypeError("page lists are integers or contiguous int64 CPU tensors")
        lists.append(t)  # a negative number is past the pool's pages as an unsigned one
    src, dst = lists
    count = src.shape[0]
    if dst.shape[0] != count:
        raise ValueError("src and dst have one entry per copy")
    es = pool.element_size()
    shape, strides = pool.shape, pool.stride()
    planes, pages = shape[:2]
    page = shape[2:].numel() * es
    page_stride = strides[1] * es if pages > 1 else page
    plane_stride = strides[0] * es if planes > 1 else page
    held = (planes - 1) * plane_stride + (pages - 1) * page_stride + page
    err = ctx.paged_error
    rc = _lib.load().tkh_copy_pages(ctx.handle, pool.data_ptr(), held, planes, plane_stride, pages, page_stride, page,
                                    src.data_ptr(), dst.data_ptr(), count, err)
    if rc != _lib.OK:
        raise TkhError(err)
