"""relative_bias against its definition: values exactly, gradients in 64 bits.

A gradient is a sum of up to queries * keys values, in float32 by parts: its
error is allowed 64 units of 2^-24 of the sum of magnitudes, and for 16-bit
tables half the spacing of the result besides."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import bucket_matrix

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("H,Q,N,buckets,reach,causal", [
    (1, 1, 1, 2, 2, True), (3, 5, 5, 4, 3, False), (2, 64, 64, 16, 40, False), (4, 65, 300, 32, 128, True),
    (2, 300, 65, 20, 90, False), (1, 1, 3000, 32, 1000, True), (3, 700, 1025, 50, 5000, False), (2, 1030, 1028, 8, 16, True),
    (6, 333, 1001, 20, 500, True), (1, 2000, 3, 256, 100000, True), (1, 200, 200, 512, 100000, False),
])
def test_bias(cuda_device, kind, H, Q, N, buckets, reach, causal):
    from mps_pointops.attention import relative_bias

    gen = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(buckets, H, generator=gen, device="cuda").to(TYPES[kind]).requires_grad_()
    print(kind, H, Q, N, buckets, reach, causal, flush=True)
    out = relative_bias(table, Q, N, max_distance=reach, causal=causal)
    offset = torch.arange(N - Q, N)[:, None] - torch.arange(N)
    bucket = bucket_matrix(offset, buckets, reach, causal)
    want = table.detach().cpu()[bucket].permute(2, 0, 1)
    assert out.dtype == table.dtype and torch.equal(out.detach().cpu(), want)
    wide = torch.randn(H, Q, N + 3, generator=gen, device="cuda").to(TYPES[kind])
    for grad in (wide[..., :N].contiguous(), wide[..., 2:N + 2], wide[:1, :, :N].expand(H, -1, -1),
                 wide[..., :N].transpose(1, 2).contiguous().transpose(1, 2)):
        got, = torch.autograd.grad(out, [table], grad, retain_graph=True)
        again, = torch.autograd.grad(out, [table], grad, retain_graph=True)
        assert got.dtype == table.dtype and torch.equal(got, again)
        g = grad.cpu().double()
        sums, sizes = torch.zeros(buckets, H, dtype=torch.float64), torch.zeros(buckets, H, dtype=torch.float64)
        sums.index_add_(0, bucket.flatten(), g.reshape(H, -1).t())
        sizes.index_add_(0, bucket.flatten(), g.abs().reshape(H, -1).t())
        off = (got.cpu().double() - sums).abs()
        assert (off <= 64 * 2.0 ** -24 * sizes + ROUND[kind] * sums.abs()).all(), (off / sizes).max()


def test_masks_and_empty(cuda_device):
    """Entries of -inf are copied; empty sides have gradients of zeros."""
    from mps_pointops.attention import relative_bias

    table = torch.full((4, 2), -torch.inf, device="cuda", requires_grad=True)
    assert (relative_bias(table, 9, 9, max_distance=8) == -torch.inf).all()
    for Q, N in ((0, 5), (5, 0), (0, 0)):
        out = relative_bias(table, Q, N, max_distance=8)
        assert out.shape == (2, Q, N)
        assert (torch.autograd.grad(out.sum(), [table])[0] == 0).all()


def test_is_the_bias_that_attention_takes(cuda_device):
    """Attention with the table equals attention with the dense bias added to
    the scores, to float32's rounding (64 units, as there)."""
    from mps_pointops.attention import relative_bias, window_attention

    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(2, 120, 3, 32, generator=gen, device="cuda") for _ in range(3))
    table = torch.randn(16, 3, generator=gen, device="cuda")
    out = window_attention(q, k, v, bias=table, max_distance=50).double()
    dense = relative_bias(table, 120, 120, max_distance=50).double()
    score = torch.matmul(q.double().transpose(1, 2), k.double().permute(0, 2, 3, 1).contiguous()) * 32 ** -0.5 + dense
    want = torch.matmul(score.softmax(-1), v.double().transpose(1, 2).contiguous()).transpose(1, 2)
    assert (out - want).norm() <= 64 * 2.0 ** -24 * want.norm()
