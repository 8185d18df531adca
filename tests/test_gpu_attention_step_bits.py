"""window_attention_step's 16-bit outputs carry one rounding: the weights' own
would add as much again.

The limit is the error of the definition's result rounded once, in 64 bits, and
a twentieth of it for the 32-bit sums, whose errors are 2^-13 (bfloat16 2^-16) of
a rounding each, and for the spread where a value lies near the middle between
two.  With the weights rounded the error is 1.2 to 1.4 times one rounding's."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import TYPES
from test_gpu_attention_step import make, step_definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,Q,N,H,G,D,window,buckets", [
    (4, 1, 600, 8, 2, 64, None, 0), (4, 1, 3000, 8, 2, 64, 512, 16), (2, 1, 5000, 32, 8, 128, None, 0), (6, 3, 40, 4, 4, 33, None, 8),
    (3, 2, 1500, 12, 1, 96, 70, 0),
])
def test_one_rounding(cuda_device, kind, B, Q, N, H, G, D, window, buckets):
    from mps_pointops.attention import window_attention_step

    q, k, v, bias = make(91, B, Q, N, H, G, D, TYPES[kind], buckets)
    how = dict(window=window, bias=bias, max_distance=100 if buckets else None)
    with torch.no_grad():
        out = window_attention_step(q, k, v, **how)
    want = step_definition(q, k, v, None, **how)
    once = (want.to(TYPES[kind]).double() - want).norm()
    assert (out.cpu().double() - want).norm() <= 1.05 * once
