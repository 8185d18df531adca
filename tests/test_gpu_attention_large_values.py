"""window_attention over values near the largest of 32 bits, whose means are finite, also where a sum of
them is not.  Tolerances as in test_gpu_attention.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, close, definition
from test_gpu_attention_step import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,H,G,D,window,causal", [(2, 300, 4, 2, 64, None, False), (2, 700, 4, 2, 128, 200, True), (3, 200, 2, 2, 33, None, True)])
@pytest.mark.parametrize("largest", [1e37, 2e38])
def test_large_values(cuda_device, kind, B, N, H, G, D, window, causal, largest):
    """Scores that rise from key to key by less than 8 (in units of log 2) in all."""
    from mps_pointops.attention import window_attention

    print(kind, B, N, H, G, D, window, causal, largest, flush=True)
    q, k, v, _ = make(23, B, N, N, H, G, D, TYPES[kind])
    q *= 0.125
    q[..., 0] = 1.0
    k[..., 0] = torch.linspace(0, 5.4 * D ** 0.5, N, device="cuda")[None, :, None]
    v[..., 1::3] = v[..., 1::3].abs().clamp(max=1.0) * largest
    v[..., 2::3] = v[..., 2::3].sign() * largest
    got, want = window_attention(q, k, v, window=window, causal=causal), definition(q, k, v, None, window=window, causal=causal)[0]
    close(got, want, LIMIT[kind])
    close(got[..., ::3], want[..., ::3], LIMIT[kind])
