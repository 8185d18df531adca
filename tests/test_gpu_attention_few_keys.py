"""Gradients of window_attention where queries see few keys, in 16 bits.

The output's rounding, which delta = do . o would carry into every ds of a row,
is as large there as that of ds itself.  What is left are two roundings of one
relative size, of ds and of the result: sqrt(2) = 1.414 times the error of the
exact gradient rounded once; limit 1.5, the rest for the spread over some 10^5
values.  With delta from the rounded output alone the shapes below have 1.6 to 1.8.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import TYPES, definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,N,H,G,D,window,causal", [
    (150, 30, 6, 2, 20, None, False),   # small clouds, one wave's rows
    (150, 14, 4, 4, 64, None, True),
    (3, 600, 4, 2, 32, 4, True),        # a narrow window
    (2, 333, 4, 1, 40, 3, False),       # few blocks: two waves share rows
    (2, 777, 2, 2, 128, 5, True),
])
def test_gradients_of_few_keys(cuda_device, kind, B, N, H, G, D, window, causal):
    from mps_pointops.attention import window_attention

    gen = torch.Generator().manual_seed(N + D)
    make = lambda heads: torch.randn(B, N, heads, D, generator=gen).to(TYPES[kind])  # noqa: E731
    q, k, v, grad = make(H), make(G), make(G), make(H)
    on = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    out = window_attention(*on, window=window, causal=causal)
    got = torch.autograd.grad(out, on, grad.to(cuda_device))
    _, dq, *_ = definition(q, k, v, grad, window=window, causal=causal)
    once = (dq.to(TYPES[kind]).double() - dq).norm()
    assert (got[0].cpu().double() - dq).norm() <= 1.5 * once
