"""A gradient's bits do not depend on which other gradients are asked for."""

from __future__ import annotations

import itertools

import pytest
import torch

from test_gpu_attention import TYPES, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("N,window,sinks,causal", [(90, None, 0, True), (400, None, 0, False), (500, 200, 5, True)])
def test_any_of_the_inputs(cuda_device, kind, N, window, sinks, causal):
    from mps_pointops.attention import window_attention

    *given, g, bias = tensors(71, 2, N, N, 4, 2, 40, TYPES[kind], 16)
    given.append(bias)

    def grads(wanted):
        leaves = [t.detach().requires_grad_(w) for t, w in zip(given, wanted)]
        out = window_attention(*leaves[:3], bias=leaves[3], max_distance=60, window=window, sinks=sinks, causal=causal)
        return iter(torch.autograd.grad(out, [t for t, w in zip(leaves, wanted) if w], g))

    whole = list(grads((True,) * 4))
    for wanted in itertools.product((False, True), repeat=4):
        if any(wanted):
            got = grads(wanted)
            assert all(torch.equal(next(got), x) for x, w in zip(whole, wanted) if w), wanted
