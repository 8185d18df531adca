"""Places that a bias of -inf masks hold infinities and NaN: they reach no output
and no gradient, the bias's own included.

The definition is that with zeros in those places (a pair of weight zero adds
nothing); tolerances as in test_gpu_attention.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, close, definition, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [40, 33])  # rows in 16-byte pieces, and not
@pytest.mark.parametrize("window,sinks,causal", [(None, 0, True), (120, 4, True), (None, 0, False), (90, 140, False)])
def test_gradients(cuda_device, kind, value, D, window, sinks, causal):
    """40 queries at the end of 200 keys; offsets of 54 and more are masked, and
    key 101 is no number.  Head 1 sees nothing at all, and its output's gradient
    is no number either."""
    from mps_pointops.attention import window_attention

    Q, N, where = 40, 200, 101
    for which in ("k", "v"):
        q, k, v, g, bias = tensors(41, 2, Q, N, 2, 2, D, TYPES[kind], 16)
        bias[slice(14, 16) if causal else 7, 0] = -math.inf  # earlier keys from 54, or 45, on
        bias[:, 1] = -math.inf
        clean_g = g.clone()
        clean_g[:, :, 1] = 0
        g[:, :, 1] = value
        clean = {"k": k, "v": v}
        bad = {x: t.clone() for x, t in clean.items()}
        clean[which][:, where] = 0
        bad[which][:, where] = value
        how = dict(window=window, sinks=sinks, causal=causal, max_distance=100)
        leaves = [t.detach().requires_grad_() for t in (q, bad["k"], bad["v"], bias)]
        print(kind, which, value, D, window, sinks, causal, flush=True)
        out = window_attention(*leaves[:3], bias=leaves[3], **how)
        got = torch.autograd.grad(out, leaves, g)
        want = definition(q, clean["k"], clean["v"], clean_g, bias=bias, **how)
        for x, y in zip((out, *got[:3]), want):
            close(x, y, LIMIT[kind])
        close(got[3], want[4], LIMIT[kind], want[5])
        assert (got[3][bias == -math.inf] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("N", [300, 3000])  # one block a cloud, and several
def test_step(cuda_device, kind, value, N):
    from mps_pointops.attention import window_attention_step

    for which in (0, 1):
        q, k, v, _, bias = tensors(42, 2, 1, N, 2, 2, 40, TYPES[kind], 8)
        bias[-1, 0] = -math.inf  # offsets from 45 on
        clean = [k, v]
        bad = [t.clone() for t in clean]
        clean[which][:, N - 150] = 0
        bad[which][:, N - 150] = value
        with torch.no_grad():
            out = window_attention_step(q, *bad, bias=bias, max_distance=100)
        close(out[:, :, :1], definition(q, *clean, None, causal=True, bias=bias, max_distance=100)[0][:, :, :1], LIMIT[kind])
        assert not torch.isfinite(out[:, :, 1]).all(-1).any()  # which has no mask
