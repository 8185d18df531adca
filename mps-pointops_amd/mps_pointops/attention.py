"""Attention for networks over ordered points.

A cloud whose points are ordered along a curve, or one that is written point
by point, is a sequence of tokens.  These operators are what a transformer
layer over such sequences asks for beside its matrix products:

* ``window_attention``: attention within a window of the order, with a few
  first tokens that every query sees and a bias learned by buckets of the
  offset, with its gradients;
* ``window_attention_step``: the same for one or a few new tokens over a cache;
* ``qk_norm_rotate``: the norm of each head's query and key and their rotation
  by the token's position in one pass, with its gradients;
* ``relative_bias``: the learned bias as a dense tensor, with its gradient.

Tensors are (batch, tokens, heads, width) in float32, float16 or bfloat16 on
``device='cuda'``, with any strides; fewer key heads than query heads are
shared by consecutive query heads.  Scores, softmax statistics, norms and sums
are float32 throughout, and no result depends on the order in which the GPU
happens to add.

float16 and bfloat16 are rounded to the type before a matrix product takes them:
``window_attention``'s weights (output and gradients) and the gradients of its
scores; its errors are about 1.4 times those of one rounding of the exact
result, and float16's weights and score gradients below 6e-5 keep fewer bits
(scale the loss).  ``window_attention_step`` keeps its weights' bits.  Callers
who need more take float32, whose exponentials and inverse roots are the
hardware's (errors of about 4e-7 and 3e-7 of a result's norm).
"""

from __future__ import annotations

import ctypes
import functools
import struct

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _native

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_HEAD = 128
_MAX_TOKENS = (1 << 30) - 1024
_MAX_REACH = 1024
_MAX_SIDE = 256
# pointops_attention of pointops_hip.h.
_ARGS = struct.Struct("@6Q9q6q2q5if")


# ------------------------------------------------------------------- buckets
def _root_above(n: int, m: int) -> int:
    """The smallest d with d ** m >= n."""
    low, high = 0, 1 << -(-n.bit_length() // m)  # low ** m < n <= high ** m
    while high - low > 1:
        mid = (low + high) // 2
        low, high = (mid, high) if mid ** m < n else (low, mid)
    return high


@functools.lru_cache(maxsize=256)
def bucket_edges(buckets: int, max_distance: int) -> tuple[int, ...]:
    """The smallest distance of each bucket but the first.

    Half of the ``buckets`` hold one distance each (0, 1, 2, ...), the others
    share the distances from there to ``max_distance`` in even steps of the
    logarithm, and all that lie farther are in the last one: with
    ``e = buckets // 2``, distance d >= e is in bucket
    ``min(buckets - 1, e + floor(log(d / e) / log(max_distance / e) * (buckets - e)))``,
    computed in whole numbers.
    """
    if buckets < 2:
        raise ValueError("at least 2 buckets are needed for each side")
    single = buckets // 2
    if max_distance <= single:
        raise ValueError(f"max_distance must be more than {single}, the distances that have a bucket of their own")
    steps = buckets - single
    return tuple(range(1, single + 1)) + tuple(
        _root_above(max_distance ** t * single ** (steps - t), steps) for t in range(1, steps))


@functools.lru_cache(maxsize=256)
def _edge_array(buckets: int, max_distance: int):
    edges = bucket_edges(buckets, max_distance)
    return (ctypes.c_int32 * len(edges))(*edges)


def _check_table(table: Tensor, heads: int | None, max_distance: int | None, causal: bool, limit: int, name: str):
    """The edges of a (buckets, heads) table's side."""
    if table.ndim != 2 or (heads is not None and table.shape[1] != heads):
        raise ValueError(f"{name} must have shape (buckets, heads)")
    if max_distance is None:
        raise ValueError(f"{name} needs max_distance")
    count = table.shape[0]
    if not causal and count % 2:
        raise ValueError(f"{name} must have an even number of buckets where both sides are seen")
    side = count if causal else count // 2
    if side > _MAX_SIDE:
        raise ValueError(f"{name} must have at most {_MAX_SIDE} buckets for each side")
    if max_distance > limit:
        raise ValueError(f"max_distance must be at most {limit}")
    return _edge_array(int(side), int(max_distance))  # (a trace has tensors for sizes)


# ----------------------------------------------------------------- arguments
def _like(t: Tensor) -> Tensor:
    """Memory for a contiguous result of the tensor's shape and type."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t: Tensor) -> Tensor:
    """The tensor with its last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_heads(tensors: dict[str, Tensor]) -> None:
    first = next(iter(tensors.values()))
    if not all(isinstance(t, Tensor) for t in tensors.values()):
        raise TypeError(f"{', '.join(tensors)} must be tensors")
    for name, t in tensors.items():
        if t.ndim != 4:
            raise ValueError(f"{name} must have shape (batch, tokens, heads, width)")
        if t.device != first.device:
            raise ValueError(f"{', '.join(tensors)} must be on the same device")
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} must be float32, float16 or bfloat16")
        if t.dtype != first.dtype:
            raise TypeError(f"{', '.join(tensors)} must have the same type")


def _check_attention(q: Tensor, k: Tensor, v: Tensor, window, sinks, causal, bias, max_distance, lengths):
    _check_heads({"q": q, "k": k, "v": v})
    batch, queries, heads, width = q.shape
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    if k.shape[0] != batch or k.shape[3] != width:
        raise ValueError("k and v must have q's batch size and head width")
    key_heads = k.shape[2]
    if heads and (key_heads == 0 or heads % key_heads):
        raise ValueError("the number of query heads must be a multiple of the number of key heads")
    if not 1 <= width <= _MAX_HEAD:
        raise ValueError(f"the head width must lie in [1, {_MAX_HEAD}]")
    if max(batch, queries, k.shape[1], heads) > _MAX_TOKENS:
        raise ValueError(f"sizes must be at most {_MAX_TOKENS}")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must be non-negative")
    edges = None
    if bias is not None:
        if not isinstance(bias, Tensor):
            raise TypeError("bias must be a tensor")
        if bias.dtype != q.dtype:
            raise TypeError("bias must have q's type")
        if bias.device != q.device:
            raise ValueError("bias must be on q's device")
        edges = _check_table(bias, heads, max_distance, causal, _MAX_REACH, "bias")
    if lengths is not None:
        if not isinstance(lengths, Tensor):
            raise TypeError("lengths must be a tensor")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError("lengths must be int32 or int64")
        if lengths.shape != (batch,):
            raise ValueError("lengths must have shape (batch,)")
        if lengths.device != q.device:
            raise ValueError("lengths must be on q's device")
    return edges


def _pack(q: Tensor, k: Tensor, v: Tensor, window, sinks, causal, bias, edges, lengths, scale) -> bytes:
    """The call as a pointops_attention."""
    batch, queries, heads, width = q.shape
    keys, key_heads = k.shape[1], k.shape[2]
    return _ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if lengths is None else lengths.data_ptr(), 0 if edges is None else ctypes.addressof(edges),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
        batch, queries, keys, heads, key_heads, width,
        keys + 1 if window is None else min(int(window), keys + 1), min(int(sinks), keys),
        0 if edges is None else len(edges), 0 if bias is None else bias.shape[0],
        0 if lengths is None else 8 * lengths.element_size(), bool(causal), _TYPES[q.dtype], scale)


def _tracked(*tensors: Tensor | None) -> bool:
    """Whether the call's graph is recorded."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _by_function(*tensors: Tensor | None) -> bool:
    """Whether a call goes through its autograd function: where its graph is
    recorded, and where more than the tensors' memory is asked for.  A trace
    records the function as a node, forward-mode differentiation and function
    transforms refuse it; the kernels' call alone they would not see."""
    return not _native.untraced() or _tracked(*tensors)


# ------------------------------------------------------------------ attention
def _attend(q, k, v, bias, lengths, edges, window, sinks, causal, scale, lse):
    out = _like(q)
    if out.numel():
        args = _pack(q, k, v, window, sinks, causal, bias, edges, lengths, scale)
        _native.call("pointops_attention_forward", args, out.data_ptr(), _native.ptr(lse), _native.stream(q.device))
    return out


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, lengths, edges, window, sinks, causal, scale):
        batch, queries, heads, _ = q.shape
        lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=q.device)
        out = _attend(q, k, v, bias, lengths, edges, window, sinks, causal, scale, lse)
        ctx.save_for_backward(q, k, v, bias, lengths, out, lse)
        ctx.rest = edges, window, sinks, causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        q, k, v, bias, lengths, out, lse = ctx.saved_tensors
        edges, window, sinks, causal, scale = ctx.rest
        grad = _rows(grad)
        dq, dk, dv = _like(q), _like(k), _like(v)
        dbias = None
        if bias is not None and ctx.needs_input_grad[3]:
            dbias = _like(bias)
        if dq.numel() or dk.numel() or dbias is not None:
            args = _pack(q, k, v, window, sinks, causal, bias, edges, lengths, scale)
            size = _native.size_query("pointops_attention_backward_workspace_bytes", args)
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            strides = (ctypes.c_int64 * 3)(*grad.stride()[:3])
            _native.call("pointops_attention_backward", args, out.data_ptr(), lse.data_ptr(), grad.data_ptr(),
                         strides, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _native.ptr(dbias),
                         workspace.data_ptr(), _native.stream(q.device))
        return dq, dk, dv, dbias, None, None, None, None, None, None


def window_attention(q: Tensor, k: Tensor, v: Tensor, *, window: int | None = None, sinks: int = 0,
                     causal: bool = False, bias: Tensor | None = None, max_distance: int | None = None,
                     lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """Attention of ``q (B, Q, H, D)`` over ``k, v (B, N, G, D)`` within a
    window of the order; H is a multiple of G, and D at most 128.

    The queries stand at the last Q of the N positions.  The query at position
    p sees the key at j when ``|p - j| < window`` (``None``: any) or
    ``j < sinks``, and only ``j <= p`` if ``causal``.  ``lengths (B,)`` (int32 or
    int64; values are clamped to [0, N]): positions from a cloud's length on do
    not exist.  A query that does not exist or sees no key yields zeros and has
    no gradient; what lies in keys and values that a query does not see
    (infinities and NaN too) reaches neither its output nor a gradient through it.

    Scores are ``scale * q . k`` (``D ** -0.5`` by default), plus
    ``bias[bucket(p - j), h]`` if a table ``bias (buckets, H)`` of q's type is
    given.  Its buckets are those of ``bucket_edges`` with ``max_distance`` (at
    most 1024): of ``p - j`` if ``causal``, else one half of them for
    ``p - j >= 0`` and the other, in the same way, for ``j - p``.  An entry of
    -inf masks its offsets, in the same way.

    Returns ``(B, Q, H, D)`` of q's type, differentiable in q, k, v and bias.
    """
    edges = _check_attention(q, k, v, window, sinks, causal, bias, max_distance, lengths)
    _native.require_device(q.device)
    if scale is None:
        scale = q.shape[3] ** -0.5
    args = (_rows(q), _rows(k), _rows(v), None if bias is None else bias.contiguous(),
            None if lengths is None else lengths.contiguous(), edges, window, sinks, causal, float(scale))
    return _WindowAttention.apply(*args) if _by_function(q, k, v, bias) else _attend(*args, None)


def _step(q, k_cache, v_cache, bias, lengths, edges, window, sinks, scale):
    out = _like(q)
    if out.numel():
        args = _pack(q, k_cache, v_cache, window, sinks, True, bias, edges, lengths, scale)
        size = _native.size_query("pointops_attention_step_workspace_bytes", args)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _native.call("pointops_attention_step", args, out.data_ptr(), _native.ptr(workspace), _native.stream(q.device))
    return out


class _WindowAttentionStep(torch.autograd.Function):
    """A node for traces; without gradients."""

    @staticmethod
    def forward(ctx, *args):
        return _step(*args)


def window_attention_step(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor | None = None, *,
                          window: int | None = None, sinks: int = 0, bias: Tensor | None = None,
                          max_distance: int | None = None, scale: float | None = None) -> Tensor:
    """``window_attention(..., causal=True)`` of one or a few new tokens a cloud
    over its cache, without gradients.

    ``k_cache, v_cache (B, N, G, D)`` hold the keys and values of the first
    ``lengths (B,)`` positions (int32 or int64, clamped to [0, N]; None: all N),
    the new tokens' own among them: ``q (B, Q, H, D)`` stands at the last Q of
    those.  What lies behind a length is not read.  A query before the first
    position yields zeros.
    """
    edges = _check_attention(q, k_cache, v_cache, window, sinks, True, bias, max_distance, lengths)
    _native.require_device(q.device)
    if _tracked(q, k_cache, v_cache, bias):
        raise ValueError("window_attention_step has no gradients: call it under torch.no_grad(), "
                         "or use window_attention")
    args = (_rows(q), _rows(k_cache), _rows(v_cache), None if bias is None else bias.contiguous(),
            None if lengths is None else lengths.contiguous(), edges, window, sinks,
            float(q.shape[3] ** -0.5 if scale is None else scale))
    return _step(*args) if _native.untraced() else _WindowAttentionStep.apply(*args)


# ------------------------------------------------------------- relative bias
_MAX_BIAS_QUERIES = 65535 * 64
_MAX_BIAS_KEYS = (1 << 22) - 1


def _dense_bias(table, edges, queries, keys):
    buckets, heads = table.shape
    out = torch.empty((heads, queries, keys), dtype=table.dtype, device=table.device)
    if out.numel():
        _native.call("pointops_relative_bias", table.data_ptr(), edges, len(edges), buckets, _TYPES[table.dtype],
                     out.data_ptr(), heads, queries, keys, _native.stream(table.device))
    return out


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, edges, queries, keys):
        ctx.rest = edges, table.shape[0]
        return _dense_bias(table, edges, queries, keys)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        edges, buckets = ctx.rest
        heads, queries, keys = grad.shape
        grad = _rows(grad)
        grad_table = torch.empty((buckets, heads), dtype=grad.dtype, device=grad.device)
        size = _native.size_query("pointops_relative_bias_backward_workspace_bytes", heads, queries, keys,
                                  buckets)
        workspace = torch.empty(size, dtype=torch.uint8, device=grad.device)
        _native.call("pointops_relative_bias_backward", grad.data_ptr(), grad.stride(0), grad.stride(1), edges,
                     len(edges), buckets, _TYPES[grad.dtype], grad_table.data_ptr(), workspace.data_ptr(),
                     heads, queries, keys, _native.stream(grad.device))
        return grad_table, None, None, None


def relative_bias(table: Tensor, queries: int, keys: int, *, max_distance: int, causal: bool = False) -> Tensor:
    """The bias that ``window_attention`` takes from ``table (buckets, H)``, as a
    tensor ``(H, queries, keys)``: entry (h, i, j) is ``table[b, h]`` with b the
    bucket of ``keys - queries + i - j`` (the queries stand at the last
    positions).  ``max_distance`` may be up to 2**30 here.  Differentiable in the
    table.
    """
    if not isinstance(table, Tensor):
        raise TypeError("table must be a tensor")
    if table.dtype not in _TYPES:
        raise TypeError("table must be float32, float16 or bfloat16")
    edges = _check_table(table, None, max_distance, causal, 1 << 30, "table")
    if queries < 0 or keys < 0:
        raise ValueError("queries and keys must be non-negative")
    if queries > _MAX_BIAS_QUERIES or keys > _MAX_BIAS_KEYS or table.shape[1] > 65535:
        raise ValueError(f"relative_bias supports at most {_MAX_BIAS_QUERIES} queries, {_MAX_BIAS_KEYS} keys and 65535 heads")
    _native.require_device(table.device)
    args = table.contiguous(), edges, int(queries), int(keys)
    return _RelativeBias.apply(*args) if _by_function(table) else _dense_bias(*args)


# --------------------------------------------------------- norm and rotation
# pointops_qk_norm of pointops_hip.h.
_NORM_ARGS = struct.Struct("@6Q8q6q2if")


def _pack_norm(q, k, q_weight, k_weight, cos, sin, eps) -> bytes:
    batch, tokens, heads, width = q.shape
    weight = q_weight if q_weight is not None else k_weight
    return _NORM_ARGS.pack(
        q.data_ptr(), k.data_ptr(), 0 if q_weight is None else q_weight.data_ptr(),
        0 if k_weight is None else k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], 0 if cos.ndim == 2 else cos.stride(0), cos.stride(-2),
        batch, tokens, heads, k.shape[2], width, 2 * cos.shape[-1],
        _TYPES[q.dtype], _TYPES[q.dtype if weight is None else weight.dtype], eps)


def _norm(q, k, q_weight, k_weight, cos, sin, eps):
    q_out, k_out = _like(q), _like(k)
    if q_out.numel() + k_out.numel():
        _native.call("pointops_qk_norm_rotate", _pack_norm(q, k, q_weight, k_weight, cos, sin, eps),
                     q_out.data_ptr(), k_out.data_ptr(), _native.stream(q.device))
    return q_out, k_out


class _QkNormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin)
        ctx.eps = eps
        return _norm(q, k, q_weight, k_weight, cos, sin, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, q_grad: Tensor, k_grad: Tensor):
        q, k, q_weight, k_weight, cos, sin = ctx.saved_tensors
        q_grad, k_grad = _rows(q_grad), _rows(k_grad)
        dq, dk = _like(q), _like(k)
        weights = [w if need else None for w, need in zip((q_weight, k_weight), ctx.needs_input_grad[2:4])]
        dwq, dwk = (None if w is None else torch.empty_like(w) for w in weights)
        if q.numel() + k.numel() or dwq is not None or dwk is not None:
            args = _pack_norm(q, k, q_weight, k_weight, cos, sin, ctx.eps)
            workspace = None
            if dwq is not None or dwk is not None:
                size = _native.size_query("pointops_qk_norm_rotate_backward_workspace_bytes", args)
                workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            three = ctypes.c_int64 * 3
            _native.call("pointops_qk_norm_rotate_backward", args, q_grad.data_ptr(), three(*q_grad.stride()[:3]),
                         k_grad.data_ptr(), three(*k_grad.stride()[:3]), dq.data_ptr(), dk.data_ptr(),
                         _native.ptr(dwq), _native.ptr(dwk), _native.ptr(workspace), _native.stream(q.device))
        return dq, dk, dwq, dwk, None, None, None


def qk_norm_rotate(q: Tensor, k: Tensor, q_weight: Tensor | None, k_weight: Tensor | None, cos: Tensor, sin: Tensor, *,
                   eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """Norm and rotation of queries ``q (B, N, H, D)`` and keys ``k (B, N, G, D)``.

    Each head's row x becomes ``y = x / sqrt(mean(x ** 2) + eps) * weight``
    (weights ``(D,)`` of q's type or float32; None: ones), and of the first
    ``R = 2 * cos.shape[-1] <= D`` values, y[i] and y[i + R / 2] turn by the
    token's angle i::

        out[i] = y[i] * cos[i] - y[i + R/2] * sin[i]
        out[i + R/2] = y[i + R/2] * cos[i] + y[i] * sin[i]

    ``cos, sin`` are float32, ``(N, R / 2)`` or ``(B, N, R / 2)``: angles of a
    place in the order, or of a point's coordinates (a share of the R / 2 for each
    axis).  They have no gradient.  Returns both in q's type, differentiable in
    q, k and the weights.
    """
    _check_heads({"q": q, "k": k})
    batch, tokens, heads, width = q.shape
    if k.shape[:2] != q.shape[:2] or k.shape[3] != width:
        raise ValueError("k must have q's batch size, tokens and head width")
    if not 1 <= width <= _MAX_HEAD:
        raise ValueError(f"the head width must lie in [1, {_MAX_HEAD}]")
    if max(batch, tokens, heads, k.shape[2]) > _MAX_TOKENS:
        raise ValueError(f"sizes must be at most {_MAX_TOKENS}")
    if not isinstance(cos, Tensor) or not isinstance(sin, Tensor):
        raise TypeError("cos and sin must be tensors")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    if cos.shape != sin.shape or cos.ndim not in (2, 3) or cos.shape[:-1] not in ((tokens,), (batch, tokens)):
        raise ValueError("cos and sin must have shape (tokens, R / 2) or (batch, tokens, R / 2)")
    if 2 * cos.shape[-1] > width:
        raise ValueError("cos and sin must have at most half as many values as the head width")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError("cos and sin must be on q's device")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise ValueError("cos and sin have no gradients here: detach them")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not isinstance(w, Tensor):
            raise TypeError(f"{name} must be a tensor")
        if w.shape != (width,):
            raise ValueError(f"{name} must have shape (width,)")
        if w.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"{name} must have q's type or be float32")
        if w.device != q.device:
            raise ValueError(f"{name} must be on q's device")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight must have the same type")
    _native.require_device(q.device)
    cos, sin = _rows(cos), _rows(sin)
    if cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    args = (_rows(q), _rows(k), None if q_weight is None else q_weight.contiguous(),
            None if k_weight is None else k_weight.contiguous(), cos, sin, float(eps))
    return _QkNormRotate.apply(*args) if _by_function(q, k, q_weight, k_weight) else _norm(*args)


__all__ = ["bucket_edges", "qk_norm_rotate", "relative_bias", "window_attention", "window_attention_step"]
