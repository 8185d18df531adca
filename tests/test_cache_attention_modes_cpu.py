"""The quantised cache and the steps over kept keys under dispatch modes that look at a
program's operations, and in a dual level without tangents: they compute, as
window_attention_step does.  Modes without memory are refused.  Launches are replaced by a list."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.flop_counter import FlopCounterMode

from mps_pointops import _native, attention


class Log(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def cache(batch=2):
    return attention.QuantizedCache(batch, 3, 2, 8, device="cpu")


CALLS = {
    "cache_write": lambda q: attention.cache_write(cache(), q, q),
    "cache_read": lambda q: attention.cache_read(cache()),
    "quantized_attention_step": lambda q: attention.quantized_attention_step(q, cache()),
    "prefix_attention_step": lambda q: attention.prefix_attention_step(q, (q[0], q[0]), (q, q)),
    "prefix_attention_step of caches": lambda q: attention.prefix_attention_step(q, cache(1), cache()),
    "window_attention_step": lambda q: attention.window_attention_step(q, q, q),
}


@pytest.fixture
def launches(monkeypatch):
    made = []
    monkeypatch.setattr(_native, "call", lambda name, *args: made.append(name))
    monkeypatch.setattr(_native, "require_device", lambda device: 0)
    monkeypatch.setattr(_native, "stream", lambda device: 0)
    return made


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", [lambda: FlopCounterMode(display=False), Log, torch.inference_mode, torch.no_grad, forward_ad.dual_level])
def test_modes_that_look_on(launches, name, mode):
    with mode():
        CALLS[name](torch.zeros(2, 3, 2, 8))
    assert len(launches) == 1


@pytest.mark.parametrize("name", [n for n in CALLS if n != "window_attention_step"])
def test_modes_without_memory(launches, name):
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match=name.split()[0]):
        CALLS[name](torch.zeros(2, 3, 2, 8))
    with pytest.raises(RuntimeError, match=name.split()[0]):
        make_fx(CALLS[name])(torch.zeros(2, 3, 2, 8))
    assert not launches


def test_tangents(launches):
    """Of any of a call's tensors."""
    q, k = torch.zeros(2, 1, 4, 8), torch.zeros(2, 3, 2, 8)
    bias, start = torch.zeros(8, 4), torch.zeros(5, 2, 8)
    calls = [(lambda k, v: attention.cache_write(cache(), k, v), (k, k)),
             (lambda q, bias: attention.quantized_attention_step(q, cache(), bias=bias, max_distance=9), (q, bias)),
             (lambda q, a, b, c, d, bias: attention.prefix_attention_step(q, (a, b), [c, d], bias=bias, max_distance=9), (q, start, start, k, k, bias))]
    for call, tensors in calls:
        for which in range(len(tensors)):
            with forward_ad.dual_level():
                args = [t.clone() for t in tensors]
                args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
                with pytest.raises(RuntimeError, match="tangents|forward-mode"):
                    call(*args)
    assert not launches
