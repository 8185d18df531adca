"""Traced calls of the attention operators, without gradients, on new tensors
and on clouds of another length give what the calls themselves give."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import tensors

pytestmark = pytest.mark.gpu


@pytest.mark.filterwarnings("ignore")
def test_traces(cuda_device):
    from mps_pointops import attention

    def layer(q, k, v, table, cos, sin):
        q, k = attention.qk_norm_rotate(q, k, None, None, cos, sin)
        whole = attention.window_attention(q, k, v, window=30, sinks=2, causal=True, bias=table, max_distance=20)
        last = attention.window_attention_step(q[:, -1:], k, v, window=30, sinks=2, bias=table, max_distance=20)
        return whole, last, attention.relative_bias(table, 7, 9, max_distance=20)

    def inputs(seed, N):
        q, k, v, _, table = tensors(seed, 2, N, N, 4, 2, 32, torch.bfloat16, 8)
        angle = torch.arange(N, device=cuda_device)[:, None] / torch.arange(1, 17, device=cuda_device)
        return q, k, v, table, angle.cos(), angle.sin()

    with torch.no_grad():
        traced = torch.jit.trace(layer, inputs(51, 70), check_trace=False)
        for seed, N in ((51, 70), (52, 70), (53, 41)):
            args = inputs(seed, N)
            for x, y in zip(traced(*args), layer(*args)):
                assert torch.equal(x, y)
