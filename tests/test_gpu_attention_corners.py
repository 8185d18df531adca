"""Corners of the attention operators: one key, the largest tables together with
the widest heads, rows that see a key that is no number, and every operator's
gradient on a stream of its own.  Tolerances as in test_gpu_attention.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, check, close, definition, tensors, visible
from test_gpu_attention_step import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B,Q,N,H,G,D,window", [
    (1, 1, 1, 1, 1, 1, None), (3, 1, 1, 4, 2, 64, None), (2, 5, 1, 2, 1, 33, None), (2, 300, 300, 2, 2, 40, 1), (1, 70, 200, 2, 1, 128, 1),
])
@pytest.mark.parametrize("causal", [False, True])
def test_one_key(cuda_device, kind, B, Q, N, H, G, D, window, causal):
    """Its weight is 1: the output is its value, and the gradients of q and k are
    zero.  What is left of them is the difference of two 32-bit sums of the D
    products do v, at most 2 D 2^-24 of their magnitudes, times scale and k (q,
    over the heads that share the key); float16 rounds to multiples of 2^-24."""
    from mps_pointops.attention import window_attention

    q, k, v, g, _ = tensors(81, B, Q, N, H, G, D, TYPES[kind])
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window=window, causal=causal)
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    want = definition(q, k, v, g, window=window, causal=causal)
    close(out, want[0], LIMIT[kind])
    close(dv, want[3], LIMIT[kind])
    most = 2 * D * 2.0 ** -24 * D ** -0.5 * D * (g.abs().amax() * v.abs().amax()).item()
    least = 2.0 ** -24 if kind == "f16" else 0.0
    assert dq.abs().amax().item() <= most * k.abs().amax().item() + least
    assert dk.abs().amax().item() <= (H // G) * most * q.abs().amax().item() + least


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("D", [128, 127])  # rows in 16-byte pieces, and not
@pytest.mark.parametrize("causal,buckets", [(True, 256), (False, 512)])
def test_largest_tables_and_widest_heads(cuda_device, kind, D, causal, buckets):
    q, k, v, g, bias = tensors(82, 1, 130, 1300, 2, 1, D, TYPES[kind], buckets)
    check(kind, q, k, v, g, causal=causal, bias=bias, max_distance=1024, window=1200, sinks=2)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("D,H,G", [(128, 40, 1), (128, 2, 2), (24, 8, 2)])
@pytest.mark.parametrize("N", [700, 2500])
def test_largest_tables_in_a_step(cuda_device, kind, D, H, G, N):
    q, k, v, bias = make(83, 2, 1, N, H, G, D, TYPES[kind], 256)
    run(kind, q, k, v, torch.tensor([N, N - 333], device=cuda_device), bias=bias, max_distance=1024, window=1500, sinks=1)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("window,sinks,causal", [(30, 2, True), (11, 0, False)])
def test_rows_that_see_a_nan_key(cuda_device, kind, window, sinks, causal):
    from mps_pointops.attention import window_attention

    q, k, v, _, bias = tensors(84, 1, 200, 200, 2, 1, 40, TYPES[kind], 8)
    k[0, 100, 0, 3] = math.nan
    out = window_attention(q, k, v, window=window, sinks=sinks, causal=causal, bias=bias, max_distance=16)
    seen = visible(200, 200, window, sinks, causal, 200)[:, 100].to(cuda_device)
    assert torch.isnan(out[:, seen]).all() and torch.isfinite(out[:, ~seen]).all()


def test_streams(cuda_device):
    """Each operator and its gradient on a side stream, behind work that writes
    its input there, give what they gave on the default one."""
    from mps_pointops import attention

    q, k, v, g, bias = tensors(85, 2, 500, 500, 4, 2, 64, torch.bfloat16, 16)
    angle = torch.randn(500, 32, device=cuda_device)
    weight = torch.randn(64, device=cuda_device)
    dense = torch.randn(4, 500, 500, device=cuda_device).bfloat16()

    def attend(q):
        out = attention.window_attention(q, k, v, window=100, sinks=3, causal=True, bias=bias, max_distance=60)
        return out, *torch.autograd.grad(out, [q], g)

    def norm(q):
        w = weight.clone().requires_grad_()
        outs = attention.qk_norm_rotate(q, k, w, w, angle.cos(), angle.sin())
        return *outs, *torch.autograd.grad(outs, [q, w], (g, k))

    def step(q):
        with torch.no_grad():
            return attention.window_attention_step(q[:, -2:], k, v, window=100, bias=bias, max_distance=60),

    def table(q):
        t = (bias + 0 * q.detach().amax()).requires_grad_()
        out = attention.relative_bias(t, 500, 500, max_distance=60)
        return out, *torch.autograd.grad(out, [t], dense)

    for call in (attend, norm, step, table):
        want = call(q.detach().requires_grad_())
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            late = torch.full_like(q, math.nan)
            big = torch.randn(4096, 4096, device=cuda_device)
            for _ in range(4):
                big = big @ big * 1e-2
            late.copy_(q)  # behind the products
            got = call(late.requires_grad_())
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), call.__name__
