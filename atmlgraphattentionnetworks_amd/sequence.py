"""Operators over rows that are packed along one dimension, as a batch of graphs packs
its nodes: layer norm, embedding and (``packed_attention``) attention within each
sequence.  Each is a hand-written HIP kernel behind ``libgat_amd.so`` with a HIP
backward, next to :class:`GraphAttentionLayer`.

Common to all: tensors on one ROCm device (a CPU tensor raises ``RuntimeError``; there
is no CPU path), float32, bfloat16 or float16 where an operator does not say otherwise,
float32 sums and statistics, one rounding at the end.  Gradients are reverse mode only: a
tensor that carries a forward-mode tangent raises ``NotImplementedError``.
``torch.jit.trace`` keeps a call as one opaque function; ``make_fx`` could not, and is
refused (``RuntimeError``).  Work is enqueued on torch's current stream of the tensors'
device, nothing synchronises the host, and every workspace comes from torch's allocator
within the call, so calls can be captured in HIP graphs.  Results do not depend on timing:
no kernel adds floats with atomics.

When a step is captured in a graph, keep no autograd graph of an eager step on the same
leaves alive (detach what is kept of the warm-up steps): its gradient accumulators
belong to another stream.
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .layer import refuse_recording, refuse_tangents

__all__ = ["layer_norm", "embedding", "packed_attention", "LayerNorm", "Embedding"]

_DTYPES = {torch.float32: _lib.GAT_F32, torch.bfloat16: _lib.GAT_BF16,
           torch.float16: _lib.GAT_F16}
_NULL = contextlib.nullcontext()


def _on(device: torch.device):
    """Launches go to the device the tensors are on, whichever is current."""
    return _NULL if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _need_tensor(what: str, name: str, t, dtypes=_DTYPES) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch.Tensor, got {type(t).__name__}")
    if forward_ad._current_level >= 0:  # inside a dual_level(): elsewhere there are none
        refuse_tangents(what, t)
    if not t.is_cuda:
        raise RuntimeError(f"{what} needs ROCm device tensors ({name} is on {t.device}); "
                           "there is no CPU path")
    if t.dtype not in dtypes:
        names = ", ".join(str(d).replace("torch.", "") for d in dtypes)
        raise ValueError(f"{what}: {name} must be one of {names}, got {t.dtype}")
    return t


def _need_like(what: str, name: str, t, like: torch.Tensor, dtype=True) -> None:
    if t.device != like.device:
        raise ValueError(f"{what}: {name} is on {t.device}, the input on {like.device}")
    if dtype and t.dtype != like.dtype:
        raise ValueError(f"{what}: {name} is {t.dtype}, the input {like.dtype}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., C] as [rows, C] with adjacent columns; a copy only where no view does it."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _as_function(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call goes through its autograd function: where a gradient may be asked for,
    and under ``torch.jit.trace``, which keeps a function as one call (of a library call it
    would keep the empty output)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return torch._C._is_tracing()


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def _too_wide(cols: int) -> ValueError:
    return ValueError(f"layer_norm: {cols} columns are more than a row may have (16384, or 16377 "
                      "/ float32 16381 where rows are not 16-byte aligned)")


def _norm_forward(x2, w, b, eps, stats, shape):
    """``shape``: x's own.  The output has it from the start: a view made within an autograd
    function could not be changed in place."""
    lib = _lib.load()
    y = torch.empty(shape, dtype=x2.dtype, device=x2.device)
    with _on(x2.device):
        rc = lib.gat_layer_norm(x2.data_ptr(), x2.stride(0), x2.shape[0], x2.shape[1], _ptr(w),
                                _ptr(b), eps, y.data_ptr(), x2.shape[1], _ptr(stats),
                                _DTYPES[x2.dtype], _stream(x2.device))
    if rc == _lib.GAT_EUNSUPPORTED:
        raise _too_wide(x2.shape[1])
    if rc:
        _lib.check(rc, "gat_layer_norm")
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        x2 = _rows(x)
        stats = torch.empty(x2.shape[0], 2, dtype=torch.float32, device=x.device)
        y = _norm_forward(x2, w, b, eps, stats, x.shape)
        ctx.save_for_backward(x2, w, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x2, w, stats = ctx.saved_tensors
        n, c = x2.shape
        shape, g = g.shape, _rows(g)
        need = ctx.needs_input_grad
        dt = _DTYPES[x2.dtype]
        dx = x2.new_empty(n, c) if need[0] else None
        dw = x2.new_empty(c) if need[1] else None
        db = x2.new_empty(c) if need[2] else None
        size = _lib.layer_norm_workspace_size(n, c, dt) if need[1] or need[2] else 0
        ws = torch.empty(size, dtype=torch.uint8, device=x2.device)
        with _on(x2.device):
            rc = _lib.load().gat_layer_norm_backward(
                g.data_ptr(), g.stride(0), x2.data_ptr(), x2.stride(0), n, c, _ptr(w),
                stats.data_ptr(), _ptr(dx), c, _ptr(dw), _ptr(db), ws.data_ptr(), size, dt,
                _stream(x2.device))
        if rc:
            _lib.check(rc, "gat_layer_norm_backward")
        return dx if dx is None or len(shape) == 2 else dx.view(shape), dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x``
    (any leading shape and strides), as ``torch.nn.functional.layer_norm`` over one
    dimension.  ``weight`` and ``bias`` are ``[C]`` of ``x``'s type or None.
    Differentiable in all three; the gradients of ``weight`` and ``bias`` are summed
    over the rows in float32 in a fixed order.  Up to 16,384 columns (16,377 where the
    rows do not all start on 16-byte boundaries; float32: 16,381)."""
    refuse_recording("layer_norm")
    _need_tensor("layer_norm", "x", x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: x needs a last dimension of at least 1, got {tuple(x.shape)}")
    if x.shape[-1] > 16384:
        raise _too_wide(x.shape[-1])
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _need_like("layer_norm", name, _need_tensor("layer_norm", name, p), x)
            if p.shape != x.shape[-1:]:
                raise ValueError(f"layer_norm: {name} must have shape [{x.shape[-1]}], "
                                 f"got {tuple(p.shape)}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must be at least 0, got {eps}")
    if x.numel() // x.shape[-1] > 0x7FFFFFFF:
        raise ValueError("layer_norm: at most 2^31 - 1 rows")
    w, b = (None if p is None else p.contiguous() for p in (weight, bias))
    if _as_function(x, w, b):
        return _LayerNorm.apply(x, w, b, float(eps))
    return _norm_forward(_rows(x), w, b, float(eps), None, x.shape)


class LayerNorm(torch.nn.Module):
    """:func:`layer_norm` with ``torch.nn.LayerNorm``'s parameters and state_dict keys,
    over one trailing dimension."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True):
        super().__init__()
        self.normalized_shape, self.eps = int(normalized_shape), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.normalized_shape)) \
            if elementwise_affine else None
        self.bias = torch.nn.Parameter(torch.zeros(self.normalized_shape)) \
            if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.normalized_shape:
            raise ValueError(f"LayerNorm({self.normalized_shape}) got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape}, eps={self.eps}"


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------
def _embed_forward(ids, w, scale):
    w = _rows(w)
    ld = w.stride(0) if w.shape[0] > 1 else w.shape[1]  # one row: its stride says nothing
    if ld < w.shape[1]:  # a row repeated by expand()
        w, ld = w.contiguous(), w.shape[1]
    out = torch.empty(*ids.shape, w.shape[1], dtype=w.dtype, device=w.device)
    with _on(w.device):
        rc = _lib.load().gat_embedding(ids.data_ptr(), int(ids.dtype == torch.int64), ids.numel(),
                                       w.data_ptr(), ld, w.shape[0], w.shape[1], scale,
                                       out.data_ptr(), w.shape[1], _DTYPES[w.dtype],
                                       _stream(w.device))
    if rc:
        _lib.check(rc, "gat_embedding")
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, w, scale, padding):
        ctx.save_for_backward(ids)
        ctx.table, ctx.scale, ctx.padding = tuple(w.shape), scale, padding
        return _embed_forward(ids, w, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        v, c = ctx.table
        g = _rows(g)
        dw = torch.empty(v, c, dtype=g.dtype, device=g.device)
        size = _lib.embedding_grad_workspace_size(ids.numel(), v, c)
        ws = torch.empty(size, dtype=torch.uint8, device=g.device) if size else None
        with _on(g.device):
            rc = _lib.load().gat_embedding_grad(
                ids.data_ptr(), int(ids.dtype == torch.int64), ids.numel(), g.data_ptr(),
                g.stride(0), v, c, ctx.scale, ctx.padding, dw.data_ptr(), c, _ptr(ws), size,
                _DTYPES[g.dtype], _stream(g.device))
        if rc:
            _lib.check(rc, "gat_embedding_grad")
        return None, dw, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``: ``ids`` int32 or int64 of any shape, ``weight``
    ``[vocab, C]``.  Differentiable in ``weight`` (a dense gradient, float32 sums over
    each id's tokens in a fixed order); tokens with ``padding_idx`` take no gradient, their
    rows are read like any other.

    An id outside ``[0, vocab)`` gives a row of NaN and takes no gradient: checking on the
    host would cost a synchronisation per call.  At most 2^30 ids, 2^30 table rows and
    65,535 x 64 16-byte vectors a row (16.8 million float32 columns)."""
    refuse_recording("embedding")
    _need_tensor("embedding", "weight", weight)
    _need_tensor("embedding", "ids", ids, (torch.int64, torch.int32))
    _need_like("embedding", "ids", ids, weight, dtype=False)
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"embedding: weight must be [vocab, C] with both at least 1, "
                         f"got {tuple(weight.shape)}")
    v = weight.shape[0]
    if v > 1 << 30 or ids.numel() > 1 << 30:
        raise ValueError("embedding: at most 2^30 table rows and 2^30 ids")
    most = 65535 * 64 * (16 // weight.element_size())
    if weight.shape[1] > most:
        raise ValueError(f"embedding: {weight.shape[1]} columns are more than a row may have ({most})")
    pad = -1
    if padding_idx is not None:
        if not -v <= padding_idx < v:
            raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {v}")
        pad = int(padding_idx) % v
    ids = ids.contiguous()
    if _as_function(weight):
        return _Embedding.apply(ids, weight, float(scale), pad)
    return _embed_forward(ids, weight, float(scale))


class Embedding(torch.nn.Module):
    """:func:`embedding` with ``torch.nn.Embedding``'s parameter, initialisation and
    state_dict key, and a ``scale`` on what it looks up."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None,
                 scale: float = 1.0):
        super().__init__()
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx {padding_idx} is outside a table of {num_embeddings}")
        self.num_embeddings, self.embedding_dim = int(num_embeddings), int(embedding_dim)
        self.padding_idx, self.scale = padding_idx, float(scale)
        self.weight = torch.nn.Parameter(torch.empty(num_embeddings, embedding_dim))
        torch.nn.init.normal_(self.weight)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{self.num_embeddings}, {self.embedding_dim}, scale={self.scale}"


# ---------------------------------------------------------------------------
# Attention over packed sequences
# ---------------------------------------------------------------------------
def _vectors(t: torch.Tensor, query: bool = False) -> torch.Tensor:
    """[tokens, heads, dim] as the kernels read it: adjacent dimensions, rows of whole
    16-byte vectors on 16-byte boundaries, no two tokens in one place and strides that 31-bit
    offsets reach (of the heads for queries only: a key head's rows have a base of their own).
    ``t`` itself where it is that already (a view of a fused projection's output, say), else
    a copy padded with zeros."""
    n = 16 // t.element_size()
    d = t.shape[2]
    row, head, one = t.stride()
    if d % n == 0 and one == 1 and row % n == 0 and head % n == 0 and t.data_ptr() % 16 == 0 \
            and d <= row <= 1 << 22 and (not query or head * t.shape[1] <= 1 << 28):
        return t
    if d % n == 0:
        return t.clone(memory_format=torch.contiguous_format)
    return torch.nn.functional.pad(t, (0, -d % n))


def _attn_check(rc: int, count: int) -> None:
    if rc == _lib.GAT_EUNSUPPORTED:  # what the entry does not refuse itself
        raise ValueError(f"packed_attention: {count} sequences are more than one launch holds "
                         "(2^32 lanes: 64 to 256 for each sequence and 32 rows)")
    if rc:
        _lib.check(rc, "gat_packed_attention")


def _attn_forward(q, k, v, ptr, kv_ptr, causal, scale, want_lse, want_low=False):
    """``q``, ``k``, ``v`` as :func:`_vectors` gives them."""
    nq, h, d = q.shape
    nk, hk = k.shape[:2]
    dev, dt, count = q.device, _DTYPES[q.dtype], ptr.numel() - 1
    out = torch.empty(nq, h, d, dtype=q.dtype, device=dev)
    lse = torch.empty(nq, h, dtype=torch.float32, device=dev) if want_lse else None
    low = torch.empty_like(out) if want_low and dt != _lib.GAT_F32 else None
    size = _lib.packed_attention_workspace_size(False, nq, nk, count, h, hk, d, dt)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with _on(dev):
        rc = _lib.load().gat_packed_attention(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
            v.data_ptr(), v.stride(0), v.stride(1), ptr.data_ptr(), kv_ptr.data_ptr(),
            int(ptr.dtype == torch.int64), count, nq, nk, h, hk, d, scale, int(causal),
            out.data_ptr(), _ptr(low), _ptr(lse), _ptr(ws), size, dt, _stream(dev))
    _attn_check(rc, count)
    return out, lse, low


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, ptr, kv_ptr, causal, scale):
        d = q.shape[2]
        q, k, v = _vectors(q, True), _vectors(k), _vectors(v)
        out, lse, low = _attn_forward(q, k, v, ptr, kv_ptr, causal, scale, True, True)
        ctx.save_for_backward(q, k, v, out, low, lse, ptr, kv_ptr)
        ctx.causal, ctx.scale, ctx.dim = causal, scale, d
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)  # no zeros for lse
        return (out if out.shape[2] == d else out[..., :d].contiguous()), lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        q, k, v, out, low, lse, ptr, kv_ptr = ctx.saved_tensors
        if g is None:
            return (None,) * 7
        g = _vectors(g, True)
        nq, h, d = q.shape
        nk, hk = k.shape[:2]
        dev, dt, count = q.device, _DTYPES[q.dtype], ptr.numel() - 1
        dq = torch.empty(nq, h, d, dtype=q.dtype, device=dev)
        dk, dv = (torch.empty(nk, hk, d, dtype=q.dtype, device=dev) for _ in range(2))
        size = _lib.packed_attention_workspace_size(True, nq, nk, count, h, hk, d, dt)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        with _on(dev):
            rc = _lib.load().gat_packed_attention_backward(
                g.data_ptr(), g.stride(0), g.stride(1), q.data_ptr(), q.stride(0), q.stride(1),
                k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                out.data_ptr(), _ptr(low), lse.data_ptr(), ptr.data_ptr(), kv_ptr.data_ptr(),
                int(ptr.dtype == torch.int64), count, nq, nk, h, hk, d, ctx.scale,
                int(ctx.causal), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), size,
                dt, _stream(dev))
        _attn_check(rc, count)
        if ctx.dim != d:
            dq, dk, dv = (t[..., :ctx.dim] for t in (dq, dk, dv))
        return dq, dk, dv, None, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ptr: torch.Tensor,
                     kv_ptr: Optional[torch.Tensor] = None, causal: bool = False,
                     scale: Optional[float] = None, return_lse: bool = False):
    """Softmax attention of every query over the keys of its own sequence.

    ``q`` is ``[queries, heads, dim]``, ``k`` and ``v`` ``[keys, kv_heads, dim]`` (float32 or
    bfloat16; ``heads`` a multiple of ``kv_heads``, query head ``h`` reads key head
    ``h // (heads // kv_heads)``; ``dim`` up to 128, ``heads * dim`` up to 2^22).  Sequence ``b`` has the queries
    ``ptr[b]:ptr[b + 1]`` and the keys ``kv_ptr[b]:kv_ptr[b + 1]``; ``ptr`` is an ascending
    int32 or int64 device tensor of ``count + 1`` offsets (a batch of graphs:
    ``GraphData.ptr()``), ``kv_ptr`` defaults to it.  One query per sequence (a readout
    over a graph's nodes, the next token of a text) is the same call with
    ``ptr = arange(count + 1)``; a few queries over many keys are split over the keys, by the
    average lengths (one sequence far longer than all others of a large batch is not).

    ``causal``: the last query sees all keys of its sequence, each earlier one a key less
    (key ``j`` is visible to query ``i`` iff ``j <= i + keys - queries``).  ``scale``
    defaults to ``dim ** -0.5``.  Queries that see no key, and rows outside all sequences,
    give zeros.  Offsets are not checked on the host: values outside the tensors are held
    to them, descending ones give undefined results (but touch nothing outside).

    Returns the output ``[queries, heads, dim]``, with ``return_lse`` also the float32
    ``[queries, heads]`` logarithm of each softmax sum (-inf where no key is seen; not
    differentiable).  Differentiable in ``q``, ``k`` and ``v``.  Scores, softmax sums and
    accumulators are float32.  In bfloat16 a matrix product's second operand is rounded to
    bfloat16: the probabilities in the forward (not where a sequence's queries times the
    query heads of a key head are 32 or fewer on average), probabilities and scores'
    gradients in the backward (not for ``q``'s gradient with ``dim`` up to 32).  A call that
    records gradients keeps its output (which is therefore not to be changed in place) and,
    in bfloat16, a second tensor of the output's size.  The backward
    forms the probabilities again from the float32 ``lse``, whose rounding is a relative
    error of about ``|lse| * 2^-23``; rows where that leaves no digit (``|lse|`` over 2.9
    million) make their gradients NaN, unless the output's gradient is 0 there.  Inputs may
    be strided views (16-byte aligned rows are read in place, others are copied)."""
    refuse_recording("packed_attention")
    kinds = (torch.float32, torch.bfloat16)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need_tensor("packed_attention", name, t, kinds)
        if t.dim() != 3:
            raise ValueError(f"packed_attention: {name} must be [tokens, heads, dim], "
                             f"got {tuple(t.shape)}")
        if t is not q:
            _need_like("packed_attention", name, t, q)
    kv_ptr = ptr if kv_ptr is None else kv_ptr
    for name, t in (("ptr", ptr), ("kv_ptr", kv_ptr)):
        _need_tensor("packed_attention", name, t, (torch.int32, torch.int64))
        _need_like("packed_attention", name, t, q, dtype=False)
        if t.dim() != 1 or t.numel() < 1:
            raise ValueError(f"packed_attention: {name} must hold count + 1 offsets, "
                             f"got {tuple(t.shape)}")
    if ptr.numel() != kv_ptr.numel():
        raise ValueError(f"packed_attention: ptr has {ptr.numel()} offsets, kv_ptr {kv_ptr.numel()}")
    nq, h, d = q.shape
    nk, hk = k.shape[:2]
    if v.shape != k.shape or k.shape[2] != d:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and "
                         f"v {tuple(v.shape)} do not fit: k and v alike, dim as q's")
    if hk == 0 or h == 0 or h % hk:
        raise ValueError(f"packed_attention: {h} query heads over {hk} key heads")
    if not 1 <= d <= 128 or hk > 65535:
        raise ValueError(f"packed_attention: dim must be 1 to 128 and kv_heads at most 65535, "
                         f"got {d} and {hk}")
    n = 16 // q.element_size()
    if h * (-(-d // n) * n) > 1 << 22:
        raise ValueError(f"packed_attention: heads * dim must be at most 2^22 (dim in whole 16-byte "
                         f"vectors), got {h} * {d}")
    if max(nq * (h // hk), nk) >= 1 << 30:
        raise ValueError("packed_attention: queries * heads / kv_heads and keys must be "
                         "below 2^30")
    if ptr.dtype != kv_ptr.dtype:
        ptr, kv_ptr = ptr.long(), kv_ptr.long()
    ptr, kv_ptr = ptr.contiguous(), kv_ptr.contiguous()
    scale = float(d) ** -0.5 if scale is None else float(scale)
    if _as_function(q, k, v):
        out, lse = _PackedAttention.apply(q, k, v, ptr, kv_ptr, bool(causal), scale)
        return (out, lse) if return_lse else out
    out, lse, _ = _attn_forward(_vectors(q, True), _vectors(k), _vectors(v), ptr, kv_ptr, bool(causal),
                                scale, return_lse)
    out = out if out.shape[2] == d else out[..., :d].contiguous()
    return (out, lse) if return_lse else out
