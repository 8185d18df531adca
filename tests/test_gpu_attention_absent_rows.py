"""Queries that do not exist (behind their cloud's length, or before the first
position) have no gradient, whatever lies in the tiles of keys that their block
reads.

Rows that exist are compared as in test_gpu_attention_masked.py, with the
tolerances of test_gpu_attention.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, definition, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [40, 33])  # rows in 16-byte pieces, and not
@pytest.mark.parametrize("Q,N,length,window,sinks,causal,where", [
    (200, 200, 150, 30, 0, True, 120),   # seen by rows of the wave in which the length lies
    (200, 200, 150, 30, 0, True, 118),   # within the last existing rows' tile
    (200, 200, 147, 9, 0, False, 146),
    (200, 200, 150, 20, 3, True, 60),    # in the first keys' tile, seen by a few
    (60, 200, 170, 12, 0, True, 129),    # a chunk of queries: no query sees the key
    (200, 120, 120, 10, 0, True, 2),     # queries before the first position
    (200, 120, 100, 10, 0, False, 30),
])
def test_absent_rows_have_no_gradient(cuda_device, kind, value, D, Q, N, length, window, sinks, causal, where):
    from mps_pointops.attention import window_attention

    for which in ("k", "v"):
        q, k, v, g, _ = tensors(21, 1, Q, N, 2, 1, D, TYPES[kind])
        {"k": k, "v": v}[which][0, where, 0, 5] = value
        how = dict(window=window, sinks=sinks, causal=causal, lengths=torch.tensor([length], device=cuda_device))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        print(kind, which, value, D, Q, N, length, window, sinks, causal, where, flush=True)
        out = window_attention(*leaves, **how)
        got = torch.autograd.grad(out, leaves, g)
        place = torch.arange(N - Q, N)
        absent = (place < 0) | (place >= length)
        assert absent.any() and not absent.all()
        assert (got[0][:, absent.to(cuda_device)] == 0).all()
        assert (got[1][:, length:] == 0).all() and (got[2][:, length:] == 0).all()
        want = definition(q, k, v, g, **how)
        for name, x, y in zip(("out", "q", "k", "v"), (out, *got), want):
            x = x.detach().cpu().double()
            rows = torch.isfinite(y).all(-1)
            assert torch.isfinite(x[rows]).all(), name
            assert (x[rows] - y[rows]).norm() <= LIMIT[kind] * y[rows].norm(), name
            # (A seen key of +-inf with a score of -inf has no weight and is left out; the definition has 0 * inf.)
            if which == "v" or math.isnan(value):
                assert not torch.isfinite(x[~rows]).all(-1).any(), name
