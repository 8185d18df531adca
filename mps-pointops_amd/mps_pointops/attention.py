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
* ``relative_bias``: the learned bias as a dense tensor, with its gradient;
* ``QuantizedCache``, ``cache_write``, ``cache_read``: keys and values kept in 8
  or 4 bits, and ``quantized_attention_step``, the step over them;
* ``prefix_attention_step``: the step of a batch whose clouds continue one common
  start, which is kept and read once for all.

Tensors are (batch, tokens, heads, width) in float32, float16 or bfloat16 on
``device='cuda'``, with any strides; fewer key heads than query heads are
shared by consecutive query heads.  Scores, softmax statistics, norms and sums
are float32 throughout, and no result depends on the order in which the GPU
happens to add.

float16 and bfloat16 are rounded to the type before a matrix product takes them:
``window_attention``'s weights (output and gradients) and the gradients of its
scores; its errors are about 1.4 times those of one rounding of the exact
result, and float16's weights and score gradients below 6e-5 keep fewer bits
(scale the loss).  ``window_attention_step`` and the steps over kept keys keep
their weights' bits (over float16 tensors to 2 ** -37 of a row's largest).  Callers
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


# ------------------------------------------------------------ quantized cache
# pointops_cache, pointops_keys and pointops_cache_attention of pointops_hip.h; of the
# last, with both keys given as they are or packed.
_CACHE = struct.Struct("@4Q6qi4x")
_KEYS = struct.Struct("@4Q7q")
_STEP_RAW = struct.Struct("@Q4Q7q4Q7q3Q3q5q2q5if")
_STEP_CODED = struct.Struct("@Q88s88s3Q3q5q2q5if")
_NO_KEYS = bytes(_KEYS.size)
_THREE = struct.Struct("@3q")
_GROUP = 32


class QuantizedCache:
    """Keys and values of ``batch`` clouds of up to ``tokens`` positions, in 8 or
    4 bits a value.

    Each row of ``width`` values (at most 128) of one of the ``heads`` key heads is
    held as codes and a scale ``2 ** x`` for each 32 of them: the smallest one,
    x >= -127, with which the group's largest magnitude is at most 448 (8 bits: 3
    fraction bits, exponents from -6 to 8, even steps of 2 ** -9 below) or 6 (4 bits:
    0, 0.5, 1, 1.5, 2, 3, 4, 6) times it.  Quotients are rounded to the nearest value,
    to even codes at ties: by at most 1/16 of a value in 8 bits, 1/4 in 4 (below the
    smallest exponents by half a step).  A group with an infinity or NaN reads as NaN, and
    a magnitude whose nearest value is 2 ** 128 (from 1.75 * 2 ** 127 on in 4 bits, 1.9375 in 8) as an infinity.

    ``k_codes, v_codes (batch, heads, tokens, bytes)`` and ``k_scales, v_scales (batch,
    heads, tokens, groups)`` are uint8 and zeros (values of zero) at first; a row's
    bytes are ``width`` rounded up to a multiple of 32, or half of that.  Their contents
    may be copied and changed, the tensors themselves stay.
    """

    __slots__ = ("k_codes", "v_codes", "k_scales", "v_scales", "batch", "tokens", "heads", "width", "bits", "device",
                 "_pointers", "_keys", "_packed")

    def __init__(self, batch: int, tokens: int, heads: int, width: int, *, bits: int = 8,
                 device: torch.device | str = "cuda"):
        if bits not in (8, 4):
            raise ValueError("bits must be 8 or 4")
        if not 1 <= width <= _MAX_HEAD:
            raise ValueError(f"the head width must lie in [1, {_MAX_HEAD}]")
        if min(batch, tokens, heads) < 0 or max(batch, tokens, heads) > _MAX_TOKENS:
            raise ValueError(f"sizes must lie in [0, {_MAX_TOKENS}]")
        groups = -(-width // _GROUP)
        self._hold([torch.zeros((batch, heads, tokens, size), dtype=torch.uint8, device=device)
                    for size in (groups * _GROUP * bits // 8, groups * _GROUP * bits // 8, groups, groups)], width, bits)

    def _hold(self, tensors: list[Tensor], width: int, bits: int) -> None:
        shape = tensors[0].shape
        pointers = tuple(t.data_ptr() for t in tensors)
        row = tensors[2].shape[3]
        batch, head = (stride // row for stride in tensors[2].stride()[:2])  # in rows, of all four alike
        values = (*tensors, shape[0], shape[2], shape[1], int(width), int(bits), tensors[0].device, pointers,
                  _KEYS.pack(*pointers, batch, 1, head, batch, 1, head, shape[2]),
                  _CACHE.pack(*pointers, batch, head, shape[0], shape[2], shape[1], width, bits))
        for name, value in zip(self.__slots__, values):
            object.__setattr__(self, name, value)

    def __setattr__(self, name: str, value) -> None:
        raise AttributeError(f"a cache's {name} stays as it was made: copy into its tensors")

    def _view(self, dim: int, first: int, count: int) -> QuantizedCache:
        if first < 0 or count < 0 or first + count > self.k_codes.shape[dim]:
            raise ValueError(f"there are {self.k_codes.shape[dim]} of these")
        view = object.__new__(QuantizedCache)
        view._hold([t.narrow(dim, first, count) for t in (self.k_codes, self.v_codes, self.k_scales, self.v_scales)],
                   self.width, self.bits)
        return view

    def positions(self, start: int, stop: int) -> QuantizedCache:
        """Positions start .. stop - 1 as a cache, in the same memory."""
        return self._view(2, start, stop - start)

    def cloud(self, index: int) -> QuantizedCache:
        """One cloud's cache (a batch of one), in the same memory."""
        return self._view(0, index, 1)

    def __reduce__(self):
        return _restore, (self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.width, self.bits)

    def __repr__(self) -> str:
        return (f"QuantizedCache(batch={self.batch}, tokens={self.tokens}, heads={self.heads}, width={self.width}, "
                f"bits={self.bits}, device='{self.device}')")


def _restore(*args) -> QuantizedCache:
    """A cache of four tensors, from a copy or a file."""
    cache = object.__new__(QuantizedCache)
    cache._hold([t.contiguous() for t in args[:4]], *args[4:])
    return cache


def _check_cache(cache, name: str = "cache") -> None:
    if type(cache) is not QuantizedCache:
        raise TypeError(f"{name} must be a QuantizedCache")
    if cache._pointers != (cache.k_codes.data_ptr(), cache.v_codes.data_ptr(), cache.k_scales.data_ptr(),
                           cache.v_scales.data_ptr()):
        raise ValueError(f"{name}'s tensors have lost their memory")


def _check_places(name: str, places, batch: int, device: torch.device) -> None:
    if not isinstance(places, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if places.dtype not in _PLACES:
        raise TypeError(f"{name} must be int32 or int64")
    if places.shape != (batch,):
        raise ValueError(f"{name} must have shape (batch,)")
    if places.device != device:
        raise ValueError(f"{name} must be on the same device")


_PLACES = {torch.int32: 32, torch.int64: 64}


def _place_args(places: Tensor | None) -> tuple[Tensor | None, int, int]:
    """The tensor, its address and its bits."""
    if places is None:
        return None, 0, 0
    places = places.contiguous()
    return places, places.data_ptr(), _PLACES[places.dtype]


def _check_unrecorded(name: str, *args) -> None:
    """Of a call with these tensors and pairs of them."""
    if _native.untraced():
        return
    every = (t for arg in args for t in (arg if isinstance(arg, (tuple, list)) else (arg,)))
    if _native.recorded(*(t for t in every if isinstance(t, Tensor))):
        raise RuntimeError(f"{name} works on kept memory: traces, transforms and forward-mode differentiation "
                           "do not see it")


def cache_write(cache: QuantizedCache, k: Tensor, v: Tensor, lengths: Tensor | None = None, *,
                starts: Tensor | None = None) -> None:
    """Writes the keys and values of new tokens ``k, v (B, T, G, D)`` to a cache.

    The T tokens of a cloud are the last of its first ``lengths (B,)`` positions
    (int32 or int64, clamped to [0, tokens]; None: all), or, with ``starts (B,)``, token t
    goes to position ``starts + t`` where that lies in [0, lengths): a batch of
    prompts padded to T has starts of 0 and their own lengths.  All other positions
    stay as they are.  k and v are float32, float16 or bfloat16 with any strides; the
    rounding to codes has no gradient.
    """
    _check_unrecorded("cache_write", k, v)
    _check_cache(cache)
    if not isinstance(k, Tensor) or not isinstance(v, Tensor):
        raise TypeError("k and v must be tensors")
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.ndim != 4:
        raise ValueError("k and v must have shape (batch, tokens, heads, width)")
    if v.shape != shape:
        raise ValueError("k and v must have the same shape")
    if dtype not in _TYPES:
        raise TypeError("k and v must be float32, float16 or bfloat16")
    if v.dtype != dtype:
        raise TypeError("k and v must have the same type")
    batch, tokens, heads, width = shape
    if batch != cache.batch or heads != cache.heads or width != cache.width:
        raise ValueError("k and v must have the cache's batch size, heads and width")
    if tokens > _MAX_TOKENS:
        raise ValueError(f"sizes must be at most {_MAX_TOKENS}")
    device = k.device
    if device != cache.device or v.device != device:
        raise ValueError("k and v must be on the cache's device")
    if lengths is not None:
        _check_places("lengths", lengths, batch, device)
    if starts is not None:
        _check_places("starts", starts, batch, device)
    _native.require_device(device)
    if _tracked(k, v):
        raise ValueError("cache_write has no gradients: call it under torch.no_grad()")
    if not (batch and tokens and heads and cache.tokens):
        return
    k, v = _rows(k), _rows(v)
    lengths, length_at, length_bits = _place_args(lengths)
    starts, start_at, start_bits = _place_args(starts)
    _native.call_on(device, "pointops_cache_write", cache._packed, k.data_ptr(), _THREE.pack(*k.stride()[:3]), v.data_ptr(),
                    _THREE.pack(*v.stride()[:3]), tokens, length_at, length_bits, start_at, start_bits, _TYPES[dtype],
                    _native.stream(device))


def cache_read(cache: QuantizedCache, *, dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """All keys and values of a cache (of a part: ``cache.positions(start, stop)``),
    ``(B, tokens, G, D)`` each, in float32, float16 or bfloat16, rounded once; float32
    and bfloat16 hold every value exactly but those below their smallest normal
    numbers, float16 those from 2 ** -14 to 65504.
    """
    _check_unrecorded("cache_read")
    _check_cache(cache)
    if dtype not in _TYPES:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    device = cache.device
    _native.require_device(device)
    shape = cache.batch, cache.tokens, cache.heads, cache.width
    k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    if k.numel():
        _native.call_on(device, "pointops_cache_read", cache._packed, k.data_ptr(), v.data_ptr(), _TYPES[dtype],
                        _native.stream(device))
    return k, v


def _check_step(q, key_heads: int, tokens: int, window, sinks, bias, max_distance, lengths):
    """The bias's edges."""
    batch, queries, heads, width = q.shape
    if not 1 <= width <= _MAX_HEAD:
        raise ValueError(f"the head width must lie in [1, {_MAX_HEAD}]")
    if heads and (key_heads == 0 or heads % key_heads):
        raise ValueError("the number of query heads must be a multiple of the number of key heads")
    if batch * queries * heads > _MAX_TOKENS or max(batch, queries, heads, tokens) > _MAX_TOKENS:
        raise ValueError(f"queries of all heads and keys must be at most {_MAX_TOKENS}")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must be non-negative")
    if lengths is not None:
        _check_places("lengths", lengths, batch, q.device)
    if bias is None:
        return None
    if not isinstance(bias, Tensor):
        raise TypeError("bias must be a tensor")
    if bias.dtype != q.dtype:
        raise TypeError("bias must have q's type")
    if bias.device != q.device:
        raise ValueError("bias must be on q's device")
    return _check_table(bias, heads, max_distance, True, _MAX_REACH, "bias")


def _check_query(q) -> None:
    if not isinstance(q, Tensor):
        raise TypeError("q must be a tensor")
    if q.ndim != 4:
        raise ValueError("q must have shape (batch, tokens, heads, width)")
    if q.dtype not in _TYPES:
        raise TypeError("q must be float32, float16 or bfloat16")


def _kept_step(q, keys, key_heads, tokens, bits, lengths, window, sinks, bias, edges, scale) -> Tensor:
    """The step over checked keys: the arguments of pointops_keys of the start and of the
    clouds' own, in one list, or both packed."""
    out = _like(q)
    shape, device = q.shape, q.device
    if not out.numel():
        return out
    q = _rows(q)
    if bias is not None:
        bias = bias.contiguous()
    lengths, length_at, length_bits = _place_args(lengths)
    stride = q.stride()
    args = (_STEP_CODED if bits else _STEP_RAW).pack(
        q.data_ptr(), *keys, 0 if bias is None else bias.data_ptr(), length_at,
        0 if edges is None else ctypes.addressof(edges), stride[0], stride[1], stride[2], shape[0], shape[1], shape[2],
        key_heads, shape[3], tokens + 1 if window is None else min(int(window), tokens + 1), min(int(sinks), tokens),
        0 if edges is None else len(edges), 0 if bias is None else bias.shape[0], length_bits, _TYPES[q.dtype], bits,
        float(shape[3] ** -0.5 if scale is None else scale))
    size = _native.size_query("pointops_cache_attention_step_workspace_bytes", args)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _native.call_on(device, "pointops_cache_attention_step", args, out.data_ptr(), _native.ptr(workspace), _native.stream(device))
    return out


def _check_coded(q: Tensor, cache, name: str, batch: int) -> None:
    _check_cache(cache, name)
    if cache.device != q.device:
        raise ValueError(f"{name} must be on q's device")
    if cache.batch != batch:
        raise ValueError(f"{name} must have a batch of {batch}")
    if cache.width != q.shape[3]:
        raise ValueError(f"{name} must have q's head width")


def quantized_attention_step(q: Tensor, cache: QuantizedCache, lengths: Tensor | None = None, *,
                             window: int | None = None, sinks: int = 0, bias: Tensor | None = None,
                             max_distance: int | None = None, scale: float | None = None) -> Tensor:
    """``window_attention_step`` over keys and values in 8 or 4 bits: of the values
    that the cache holds, without a further rounding of them, of the queries or of
    the weights.  ``q (B, Q, H, D)`` is float32, float16 or bfloat16.
    """
    _check_unrecorded("quantized_attention_step", q, bias)
    _check_query(q)
    _check_coded(q, cache, "cache", q.shape[0])
    edges = _check_step(q, cache.heads, cache.tokens, window, sinks, bias, max_distance, lengths)
    _native.require_device(q.device)
    if _tracked(q, bias):
        raise ValueError("quantized_attention_step has no gradients: call it under torch.no_grad()")
    return _kept_step(q, (_NO_KEYS, cache._keys), cache.heads, cache.tokens, cache.bits, lengths, window, sinks, bias,
                      edges, scale)


def prefix_attention_step(q: Tensor, prefix, cache, lengths: Tensor | None = None, *, window: int | None = None,
                          sinks: int = 0, bias: Tensor | None = None, max_distance: int | None = None,
                          scale: float | None = None) -> Tensor:
    """``window_attention_step`` of a batch whose clouds continue one common start.

    ``prefix`` is the start's keys and values, two tensors ``(P, G, D)``, and
    ``cache`` each cloud's own behind them, two tensors ``(B, N, G, D)`` of which the
    first ``lengths (B,)`` hold tokens, the new ones' own among them: the cloud's
    positions are 0 .. P + lengths - 1, and ``q (B, Q, H, D)`` stands at the last Q.
    Or both are a ``QuantizedCache`` of the same bits, the prefix with a batch of one.
    Where they are long, the start's keys are read once for up to 64 queries of the batch
    at a time.  Tensors are best aligned to 16 bytes, and the head width a multiple of 8 (float32:
    of 4): of others, also if only one is, rows are read value by value, for up to 32 queries
    at a time, and a call takes many times as long.  Without gradients.
    """
    _check_unrecorded("prefix_attention_step", q, prefix, cache, bias)
    _check_query(q)
    if type(prefix) is QuantizedCache or type(cache) is QuantizedCache:
        if type(prefix) is not type(cache):
            raise TypeError("prefix and cache must both be a QuantizedCache, or both pairs of tensors")
        _check_coded(q, prefix, "prefix", 1)
        _check_coded(q, cache, "cache", q.shape[0])
        if prefix.bits != cache.bits or prefix.heads != cache.heads:
            raise ValueError("prefix and cache must have the same bits and heads")
        tokens = prefix.tokens + cache.tokens
        edges = _check_step(q, cache.heads, tokens, window, sinks, bias, max_distance, lengths)
        _native.require_device(q.device)
        if _tracked(q, bias):
            raise ValueError("prefix_attention_step has no gradients: call it under torch.no_grad()")
        return _kept_step(q, (prefix._keys, cache._keys), cache.heads, tokens, cache.bits, lengths, window, sinks, bias,
                          edges, scale)
    dtype, device = q.dtype, q.device
    for name, pair, dims, shape in (("prefix", prefix, 3, "(tokens, heads, width)"),
                                    ("cache", cache, 4, "(batch, tokens, heads, width)")):
        if not isinstance(pair, (tuple, list)) or len(pair) != 2:
            raise TypeError(f"{name} must be a pair of tensors or a QuantizedCache")
        for t in pair:
            if not isinstance(t, Tensor):
                raise TypeError(f"{name} must be a pair of tensors or a QuantizedCache")
            if t.ndim != dims:
                raise ValueError(f"{name} must be two tensors of shape {shape}")
            if t.dtype is not dtype:
                raise TypeError(f"{name} must have the same type as q")
            if t.device != device:
                raise ValueError(f"{name} must be on q's device")
    (pk, pv), (ck, cv) = prefix, cache
    start, own = pk.shape, ck.shape
    if pv.shape != start or cv.shape != own:
        raise ValueError("keys and values must have the same shape")
    if own[0] != q.shape[0]:
        raise ValueError("cache must have q's batch size")
    if start[1] != own[2]:
        raise ValueError("prefix and cache must have the same heads")
    if start[2] != q.shape[3] or own[3] != q.shape[3]:
        raise ValueError("prefix and cache must have q's head width")
    tokens = start[0] + own[1]
    edges = _check_step(q, own[2], tokens, window, sinks, bias, max_distance, lengths)
    _native.require_device(device)
    if _tracked(q, bias, pk, pv, ck, cv):
        raise ValueError("prefix_attention_step has no gradients: call it under torch.no_grad()")
    a, b, c, d = pk.stride(), pv.stride(), ck.stride(), cv.stride()
    if own[3] > 1 and not a[2] == b[2] == c[3] == d[3] == 1:
        pk, pv, ck, cv = _rows(pk), _rows(pv), _rows(ck), _rows(cv)
        a, b, c, d = pk.stride(), pv.stride(), ck.stride(), cv.stride()
    keys = (pk.data_ptr(), pv.data_ptr(), 0, 0, 0, a[0], a[1], 0, b[0], b[1], start[0],
            ck.data_ptr(), cv.data_ptr(), 0, 0, c[0], c[1], c[2], d[0], d[1], d[2], own[1])
    return _kept_step(q, keys, own[2], tokens, 0, lengths, window, sinks, bias, edges, scale)


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


__all__ = ["QuantizedCache", "bucket_edges", "cache_read", "cache_write", "prefix_attention_step", "qk_norm_rotate",
           "quantized_attention_step", "relative_bias", "window_attention", "window_attention_step"]
