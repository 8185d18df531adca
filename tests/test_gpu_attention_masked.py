"""Gradients of window_attention where a token is no number: what does not see
it, or is not seen by it, keeps its gradient.

Tolerances as in test_gpu_attention.py; entries of the definition that are not
finite must not be finite here either, and the others are compared."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, definition, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("which,value", [("q", math.nan), ("k", math.nan), ("v", math.nan), ("v", math.inf), ("grad", math.nan),
                                         ("grad", -math.inf)])
@pytest.mark.parametrize("D", [40, 33])  # rows in 16-byte pieces, and not
@pytest.mark.parametrize("window,sinks,causal,buckets,where", [
    (30, 2, True, 8, 120), (11, 0, False, 0, 64), (20, 3, False, 8, 1), (17, 40, True, 0, 30),
])
def test_gradients_beside_a_token_that_is_no_number(cuda_device, kind, which, value, D, window, sinks, causal, buckets, where):
    from mps_pointops.attention import window_attention

    q, k, v, g, bias = tensors(11, 1, 200, 200, 2, 1, D, TYPES[kind], buckets)
    {"q": q, "k": k, "v": v, "grad": g}[which][0, where, 0, 5] = value
    how = dict(window=window, sinks=sinks, causal=causal, max_distance=16 if buckets else None)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    print(kind, which, value, D, window, sinks, causal, flush=True)
    out = window_attention(*leaves, bias=bias, **how)
    got = torch.autograd.grad(out, leaves, g)
    want = definition(q, k, v, g, bias=bias, **how)
    for name, x, y in zip(("out", "q", "k", "v"), (out, *got), want):
        x = x.detach().cpu().double()
        rows = torch.isfinite(y).all(-1)
        # (A first key is seen by all: then nothing of some results is left.)
        assert torch.isfinite(x[rows]).all(), name
        assert (x[rows] - y[rows]).norm() <= LIMIT[kind] * y[rows].norm(), name
        assert not torch.isfinite(x[~rows]).all(-1).any(), name


@pytest.mark.parametrize("kind", TYPES)
def test_everything_is_no_number(cuda_device, kind):
    """A diverged model's call ends, and says so everywhere."""
    from mps_pointops.attention import window_attention

    q, k, v, g, _ = tensors(12, 1, 150, 150, 2, 1, 32, TYPES[kind])
    leaves = [t.fill_(math.nan).requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window=40, sinks=2, causal=True)
    assert torch.isnan(out).all()
    assert all(torch.isnan(x).all() for x in torch.autograd.grad(out, leaves, g))
