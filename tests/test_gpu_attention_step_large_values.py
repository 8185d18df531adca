"""window_attention_step over values near the largest of 32 bits, whose means are finite, also where
a sum of them is not.  Tolerances as in test_gpu_attention_step.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, close
from test_gpu_attention_step import make, step_definition

pytestmark = pytest.mark.gpu

SIZES = [(3, 1, 400, 4, 2, 64), (1, 1, 6000, 4, 2, 64), (3, 5, 3000, 8, 2, 32), (4, 1, 500, 4, 2, 33), (2, 1, 5000, 4, 2, 128)]


def check(q, k, v, lengths, kind):
    from mps_pointops.attention import window_attention_step

    with torch.no_grad():
        got, want = window_attention_step(q, k, v, lengths), step_definition(q, k, v, lengths)
    close(got, want, LIMIT[kind])
    close(got[..., ::3], want[..., ::3], LIMIT[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("B,Q,N,H,G,D", SIZES)
@pytest.mark.parametrize("largest", [1e37, 2e38])
def test_large_values(cuda_device, kind, B, Q, N, H, G, D, largest):
    """Scores that rise from key to key by less than 8 (in units of log 2) in all."""
    print(kind, B, Q, N, H, G, D, largest, flush=True)
    q, k, v, _ = make(21, B, Q, N, H, G, D, TYPES[kind])
    q *= 0.125
    q[..., 0] = 1.0
    k[..., 0] = torch.linspace(0, 5.4 * D ** 0.5, N, device="cuda")[None, :, None]
    v[..., 1::3] = v[..., 1::3].abs().clamp(max=1.0) * largest
    v[..., 2::3] = v[..., 2::3].sign() * largest
    check(q, k, v, N - torch.arange(B, device="cuda") % 3, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("B,Q,N,H,G,D", SIZES)
def test_few_keys_of_large_values(cuda_device, kind, B, Q, N, H, G, D):
    """Some keys of equal scores far above the others', so that each split's sum is finite, and that
    of all splits is not."""
    print(kind, B, Q, N, H, G, D, flush=True)
    q, k, v, _ = make(22, B, Q, N, H, G, D, TYPES[kind])
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    some = k[:, ::max(1, N // 5)]
    some.zero_()
    some[..., 0] = 5.0 * D ** 0.5
    v[:, ::max(1, N // 5), :, 1::3] = 3e38
    check(q, k, v, None, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,window", [(3, 400, 300), (2, 6000, 4000)])
def test_columns_beside_those_formed_again(cuda_device, kind, B, N, window):
    """A masked value that is no number has one column formed again: the others, near the type's smallest
    numbers, keep their bits."""
    from mps_pointops.attention import window_attention_step

    q, k, v, _ = make(23, B, 1, N, 4, 2, 64, TYPES[kind])
    v *= 1e-33
    with torch.no_grad():
        want = window_attention_step(q, k, v, window=window, sinks=1)
        v[:, N - window - 3:N - window, :, 5] = float("nan")
        got = window_attention_step(q, k, v, window=window, sinks=1)
    some = [c for c in range(64) if c != 5]
    assert torch.equal(got[..., some], want[..., some]) and torch.isfinite(got).all()
    assert (got.double() - want.double()).norm() <= 2 * LIMIT[kind] * want.double().norm()
