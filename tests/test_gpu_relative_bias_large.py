"""relative_bias at the largest number of queries that its launches hold."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_most_queries(cuda_device, kind):
    """Entries by an independent expression; the gradient of ones counts each
    bucket's offsets (exact in float32, rounded once in bfloat16)."""
    from mps_pointops.attention import bucket_edges, relative_bias

    Q, N = 4194240, 3
    table = torch.arange(1, 9, device=cuda_device, dtype=kind)[:, None].requires_grad_()
    out = relative_bias(table, Q, N, max_distance=1 << 20, causal=True)
    edges = torch.tensor(bucket_edges(8, 1 << 20), device=cuda_device)
    offset = torch.arange(N - Q, N, device=cuda_device)[:, None] - torch.arange(N, device=cuda_device)
    bucket = (offset.clamp(min=0)[..., None] >= edges).sum(-1)
    assert torch.equal(out[0], table.detach()[bucket, 0])
    grad, = torch.autograd.grad(out, [table], torch.ones_like(out))
    assert torch.equal(grad[:, 0], torch.bincount(bucket.flatten(), minlength=8).to(kind))
