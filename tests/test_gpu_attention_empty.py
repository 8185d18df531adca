"""Gradients of window_attention where a side is empty are zeros, all of them
written: memory that held other values before shows none of them."""

from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

SIDES = [(0, 4, 5, 2), (2, 0, 5, 2), (2, 3, 0, 2), (2, 0, 0, 2), (2, 3, 5, 0), (0, 0, 0, 2), (2, 0, 0, 0)]


@pytest.mark.parametrize("B,Q,N,H", SIDES)
@pytest.mark.parametrize("causal", [False, True])
def test_through_autograd(cuda_device, B, Q, N, H, causal):
    from mps_pointops.attention import window_attention

    q = torch.ones(B, Q, H, 8, device=cuda_device, requires_grad=True)
    k, v = (torch.ones(B, N, 2 if H else 3, 8, device=cuda_device, requires_grad=True) for _ in range(2))
    bias = torch.ones(16, H, device=cuda_device, requires_grad=True)
    out = window_attention(q, k, v, window=3, sinks=1, causal=causal, bias=bias, max_distance=20)
    used = [torch.full((16, 2), torch.nan, device=cuda_device) for _ in range(64)]  # the next small blocks
    torch.cuda.synchronize()
    del used
    got = torch.autograd.grad(out, (q, k, v, bias), torch.ones_like(out))
    for t, g in zip((q, k, v, bias), got):
        assert g.shape == t.shape and (g == 0).all()


@pytest.mark.parametrize("B,Q,N,H", SIDES)
def test_the_entry_point_writes_everything(cuda_device, B, Q, N, H):
    """As a caller in C would: buffers that hold NaN."""
    from mps_pointops import _native, attention

    G, D = 2, 8
    new = lambda *s: torch.full(s, torch.nan, device=cuda_device)  # noqa: E731
    q, grad, out, dq, lse = new(B, Q, H, D), new(B, Q, H, D), new(B, Q, H, D), new(B, Q, H, D), new(B, H, Q)
    k, v, dk, dv = new(B, N, G, D), new(B, N, G, D), new(B, N, G, D), new(B, N, G, D)
    bias, dbias = new(8, H), new(8, H)
    edges = attention._edge_array(8, 20)
    args = attention._pack(q, k, v, 3, 1, True, bias, edges, None, 1.0)
    workspace = torch.empty(_native.size_query("pointops_attention_backward_workspace_bytes", args), dtype=torch.uint8,
                            device=cuda_device)
    _native.call("pointops_attention_backward", args, out.data_ptr(), lse.data_ptr(), grad.data_ptr(),
                 (ctypes.c_int64 * 3)(*grad.stride()[:3]), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dbias.data_ptr(),
                 workspace.data_ptr(), _native.stream(cuda_device))
    for t in (dq, dk, dv, dbias):
        assert (t == 0).all()


@pytest.mark.parametrize("B,N,H,G", [(0, 4, 2, 1), (3, 0, 2, 1), (3, 4, 0, 0), (0, 0, 0, 0), (3, 4, 0, 2)])
@pytest.mark.parametrize("D,R", [(8, 8), (33, 6), (128, 128), (1, 0)])
def test_weights_of_no_rows(cuda_device, B, N, H, G, D, R):
    """qk_norm_rotate's weights, through the entry point and through autograd."""
    from mps_pointops import _native, attention

    q, k = torch.ones(B, N, H, D, device=cuda_device), torch.ones(B, N, G, D, device=cuda_device)
    angle = torch.zeros(B, N, R // 2, device=cuda_device)
    w = torch.ones(D, device=cuda_device)
    dwq, dwk = (torch.full((D,), torch.nan, device=cuda_device) for _ in range(2))
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    args = attention._pack_norm(q, k, w, w, angle, angle, 1e-6)
    size = _native.size_query("pointops_qk_norm_rotate_backward_workspace_bytes", args)
    workspace = torch.empty(size, dtype=torch.uint8, device=cuda_device)
    three = ctypes.c_int64 * 3
    _native.call("pointops_qk_norm_rotate_backward", args, q.data_ptr(), three(*q.stride()[:3]), k.data_ptr(),
                 three(*k.stride()[:3]), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
                 workspace.data_ptr(), _native.stream(cuda_device))
    leaves = [t.requires_grad_() for t in (q, k, w, w.clone())]
    outs = attention.qk_norm_rotate(*leaves, angle, angle)
    grads = torch.autograd.grad(outs, leaves, [torch.zeros_like(t) for t in outs])
    assert all((t == 0).all() for t in (dwq, *grads))
    if not k.numel():
        assert (dwk == 0).all()
