"""Gradients of window_attention where a row's scores are large: all of its keys
under a mask of the type's lowest value, or tokens that repeat with scores of
thousands.  The weights of such a row still add up to 1.

Queries under a mask are zeros, and repeated tokens have the same score, so that
the definition's weights are equal shares whatever the scores' own rounding;
tolerances as in test_gpu_attention.py.  A row's ds add up to zero, so that dq
cancels where keys repeat: its error is allowed that much of the sum of its
terms' magnitudes, as the bias's gradient."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, close, definition, tensors, visible

pytestmark = pytest.mark.gpu


def sizes_of_dq(q, k, v, g, window, sinks, causal):
    """|ds| |k| of rows whose keys share the weight evenly, in 64 bits."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    (_, Q, H, D), (_, N, G, _) = q.shape, k.shape
    p = visible(Q, N, window, sinks, causal, N).double()
    p = p / p.sum(1, keepdim=True)
    size = torch.zeros_like(q)
    for h in range(H):
        dp = g[0, :, h] @ v[0, :, h * G // H].t()
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        size[0, :, h] = D ** -0.5 * ds.abs() @ k[0, :, h * G // H].abs()
    return size


def check(kind, q, k, v, g, copies=1, cancels=False, **how):
    """One cloud against the definition; `copies` of it side by side give the
    same, and their sum for the bias."""
    from mps_pointops.attention import window_attention

    bias = how.pop("bias", None)
    many = [t.expand(copies, -1, -1, -1).contiguous() for t in (q, k, v, g)]
    leaves = [t.requires_grad_() for t in many[:3]] + ([] if bias is None else [bias.clone().requires_grad_()])
    more = {} if bias is None else {"bias": leaves[3]}
    print(kind, tuple(many[0].shape), how, flush=True)
    out = window_attention(*leaves[:3], **more, **how)
    got = torch.autograd.grad(out, leaves, many[3])
    want = definition(q, k, v, g, bias=bias, **how)
    for n, (x, y) in enumerate(zip((out, *got[:3]), want)):
        assert all(torch.equal(x[0], x[b]) for b in range(copies))
        close(x[:1], y, LIMIT[kind], sizes_of_dq(q, k, v, g, how["window"], how["sinks"], how["causal"]) if cancels and n == 1 else None)
    if bias is not None:
        close(got[3], want[4] * copies, LIMIT[kind], want[5] * copies)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("low", ["lowest", -6e4, -3000.0])
@pytest.mark.parametrize("N,D,copies,window,sinks,causal", [
    (90, 32, 1, None, 0, True), (300, 40, 1, 200, 5, True), (170, 33, 1, 160, 40, False), (290, 24, 180, 280, 3, True),
    (140, 128, 1, None, 0, False),
])
def test_rows_under_a_mask(cuda_device, kind, low, N, D, copies, window, sinks, causal):
    """Head 0: the lowest value for all but the keys farthest away, which few
    rows see; head 1: for every key."""
    q, k, v, g, bias = tensors(31, 1, N, N, 2, 2, D, TYPES[kind], 8)
    low = torch.finfo(TYPES[kind]).min if low == "lowest" else low
    q[:] = 0
    bias[:, 1] = low
    bias[:, 0] = low
    bias[3 if causal else 2, 0] = 0.5
    check(kind, q, k, v, g, copies, False, window=window, sinks=sinks, causal=causal, bias=bias, max_distance=100)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("N,D,copies,window,sinks,causal", [
    (100, 32, 1, None, 0, True), (400, 64, 1, 150, 2, True), (200, 20, 1, 30, 0, False), (290, 128, 180, None, 0, True),
])
@pytest.mark.parametrize("size", [20.0, 200.0])
def test_repeated_tokens(cuda_device, kind, N, D, copies, window, sinks, causal, size):
    q, k, v, g, _ = tensors(32, 1, N, N, 2, 1, D, TYPES[kind])
    k[:] = (size * k[:, :1].sign()).expand_as(k)
    q[:] = size * q.sign()
    check(kind, q, k, v, g, copies, True, window=window, sinks=sinks, causal=causal)
