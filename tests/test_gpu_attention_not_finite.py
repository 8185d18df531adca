"""Where places are no numbers: columns of values that they do not reach keep
their results, and calls that are full of them (a gradient that overflowed, a
model that diverged) take about as long as others.

Tolerances as in test_gpu_attention.py, column by column; times against the same
call on finite values, of which a pass over every pair one by one would take
hundreds."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, definition, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("D", [40, 33, 96])
@pytest.mark.parametrize("window,sinks,causal,buckets", [(40, 3, True, 8), (25, 0, False, 0), (30, 50, False, 8)])
def test_columns(cuda_device, kind, D, window, sinks, causal, buckets):
    """Values of two tokens and a gradient, in one column each."""
    from mps_pointops.attention import window_attention

    q, k, v, g, bias = tensors(61, 1, 200, 200, 2, 1, D, TYPES[kind], buckets)
    v[0, 60, 0, 5], v[0, 130, 0, D - 1] = math.nan, math.inf
    g[0, 170, 0, 2] = -math.inf
    how = dict(window=window, sinks=sinks, causal=causal, max_distance=16 if buckets else None)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, bias=bias, **how)
    got = torch.autograd.grad(out, leaves, g)
    want = definition(q, k, v, g, bias=bias, **how)
    for name, x, y in zip(("out", "q", "k", "v"), (out, *got), want):
        x, y = x.detach().cpu().double(), y
        there = torch.isfinite(y)
        assert torch.equal(torch.isfinite(x), there), name
        assert (x[there] - y[there]).norm() <= LIMIT[kind] * y[there].norm(), name


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("sinks", [0, 4])
def test_times(cuda_device, kind, biased, sinks):
    from mps_pointops.attention import window_attention, window_attention_step

    N = 2048
    q, k, v, g, bias = tensors(62, 2, N, N, 4, 2, 64, TYPES[kind], 16 if biased else 0)
    how = dict(bias=bias, max_distance=100 if biased else None, window=1024, sinks=sinks)

    def train(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = window_attention(*leaves, causal=True, **how)
        return out, *torch.autograd.grad(out, leaves, g)

    def step(q, k, v, g):
        with torch.no_grad():
            return window_attention_step(q[:, -1:], k, v, **how),

    def best(call, *args):
        times = []
        for _ in range(4):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            results = call(*args)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times[1:]), results

    usual, _ = best(train, q, k, v, g)
    for value in (math.nan, math.inf):
        for what in ("gradient", "its column", "all"):
            bad = [t.clone() for t in (q, k, v, g)]
            if what == "its column":
                bad[3][..., 7] = value
            else:
                for t in bad[3 if what == "gradient" else 0:]:
                    t.fill_(value)
            print(kind, biased, sinks, value, what, flush=True)
            took, results = best(train, *bad)
            assert took < 10 * usual + 0.5, (what, took, usual)
            for x in results[0 if what == "all" else 1:3]:
                assert not torch.isfinite(x[:, :-1]).any()  # (no query sees the last key but its own)
    usual, _ = best(step, q, k, v, g)
    for value in (math.nan, math.inf):
        took, results = best(step, *[torch.full_like(t, value) for t in (q, k, v, g)])
        assert took < 10 * usual + 0.5
        assert not torch.isfinite(results[0]).any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("biased", [False, True])
def test_one_token(cuda_device, kind, biased):
    """A NaN token in the middle, with a finite gradient: all that meets it is NaN,
    which is found without going through the pairs before it; what does not keeps its
    values, those of the clouds without it."""
    from mps_pointops.attention import window_attention

    N, at = 4096, 2048
    q, k, v, g, bias = tensors(63, 1, N, N, 4, 2, 64, TYPES[kind], 16 if biased else 0)
    how = dict(bias=bias, max_distance=100 if biased else None, causal=True)

    def train(*tensors):
        leaves = [t.detach().requires_grad_() for t in tensors]
        out = window_attention(*leaves, **how)
        return out, *torch.autograd.grad(out, leaves, g)

    def best(*tensors):
        times = []
        for _ in range(4):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            results = train(*tensors)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times[1:]), results

    usual, whole = best(q, k, v)
    for t in (q, k, v):
        t[:, at] = math.nan
    took, got = best(q, k, v)
    assert took < 10 * usual + 0.5, (took, usual)
    for x, y in zip(got[:2], whole):  # rows before it do not see it
        assert torch.isnan(x[:, at:]).all()
        assert (x[:, :at].double() - y[:, :at].double()).norm() <= LIMIT[kind] * y[:, :at].double().norm()
    assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()  # every key is seen by its row or a later one
