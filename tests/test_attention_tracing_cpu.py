"""Traces and forward-mode differentiation of the attention operators, without
gradients: a trace records a node that computes, and a tangent, for which the
operators have no rule, is refused and not lost.  The launch is replaced by one
that marks its outputs."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from mps_pointops import _native, attention

HEADS, ANGLE, TABLE = (2, 5, 2, 8), (5, 4), (8, 2)


def shape(*s):
    return torch.zeros(s)


CALLS = {  # operator: its tensors, the call
    "window_attention": ((HEADS,) * 3 + (TABLE,), lambda q, k, v, t: attention.window_attention(q, k, v, bias=t, max_distance=9)),
    "window_attention_step": ((HEADS,) * 3 + (TABLE,),
                              lambda q, k, v, t: attention.window_attention_step(q, k, v, window=3, bias=t, max_distance=9)),
    "relative_bias": ((TABLE,), lambda t: attention.relative_bias(t, 5, 6, max_distance=9)),
    "qk_norm_rotate": ((HEADS, HEADS, (8,), (8,), ANGLE, ANGLE), attention.qk_norm_rotate),
}
# The outputs' places among a launch's arguments, and their sizes.
OUTPUTS = {
    "pointops_attention_forward": {1: 160}, "pointops_attention_step": {1: 160}, "pointops_relative_bias": {5: 60},
    "pointops_qk_norm_rotate": {1: 160, 2: 160},
}


@pytest.fixture
def launches(monkeypatch):
    made = []

    def call(name, *args):
        made.append(name)
        for at, size in OUTPUTS[name].items():
            (ctypes.c_float * size).from_address(args[at])[:] = [float(len(made))] * size

    monkeypatch.setattr(_native, "call", call)
    monkeypatch.setattr(_native, "require_device", lambda device: 0)
    monkeypatch.setattr(_native, "stream", lambda device: 0)
    return made


def outputs(x):
    return x if isinstance(x, tuple) else (x,)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_computes(launches, name, grad):
    shapes, call = CALLS[name]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, tuple(shape(*s) for s in shapes), check_trace=False)
        for _ in range(2):
            before = len(launches)
            got = outputs(traced(*(shape(*s) for s in shapes)))
            assert len(launches) == before + 1
            assert all((t == before + 1).all() for t in got)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(launches, name, grad):
    shapes, call = CALLS[name]
    for which in range(len(shapes)):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            args = [shape(*s) for s in shapes]
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
                call(*args)


@pytest.mark.parametrize("name", CALLS)
def test_no_tangent_no_refusal(launches, name):
    """Inside a dual level, a call whose tensors have none computes."""
    shapes, call = CALLS[name]
    with forward_ad.dual_level():
        assert all((t == 1).all() for t in outputs(call(*(shape(*s) for s in shapes))))
    assert len(launches) == 1


@pytest.mark.parametrize("name", CALLS)
def test_other_calls_leave_the_function_out(launches, monkeypatch, name):
    for function in ("_WindowAttention", "_WindowAttentionStep", "_RelativeBias", "_QkNormRotate"):
        monkeypatch.setattr(getattr(attention, function), "apply", None)
    shapes, call = CALLS[name]
    call(*(shape(*s) for s in shapes))
    assert len(launches) == 1


@pytest.mark.parametrize("name", CALLS)
def test_transforms_are_refused(launches, name):
    shapes, call = CALLS[name]
    args = tuple(torch.zeros(3, *s) for s in shapes)
    with pytest.raises(RuntimeError):
        torch.vmap(call)(*args)
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.grad(lambda x, *rest: outputs(call(x, *rest))[0].sum())(*(shape(*s) for s in shapes))
    assert not launches
