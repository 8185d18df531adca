"""The example of examples/ordered_points.py: training lowers the loss, single
steps over the cache give the whole pass's logits, and the attention's weights
seen through the dense bias are those that the fused call applies."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("ordered_points", ROOT / "examples" / "ordered_points.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_trains_and_continues(cuda_device, example):
    torch.manual_seed(0)
    model = example.Generator().cuda()
    losses = example.train(model, 30, 160)
    assert losses[0] > 8.0  # about log 4096 at the start
    assert sum(losses[-5:]) / 5 < losses[0] - 1.0
    token = example.clouds(3, 160, 12345)
    with torch.no_grad():
        whole, single = model(token), example.replay(model, token)
    # Float32 throughout: two layers of sums in another order.
    assert (whole - single).norm() <= 2e-5 * whole.norm()
    made = example.generate(model, token[:, :80], 160)
    assert made.shape == (3, 160) and torch.equal(made[:, :80], token[:, :80])


def test_weights_are_those_of_the_fused_call(cuda_device, example):
    from mps_pointops import attention

    torch.manual_seed(1)
    layer = example.Layer().cuda()
    with torch.no_grad():
        layer.bias.normal_()
        token = example.clouds(2, 150, 7)
        x = torch.randn(2, 150, example.WIDTH, device="cuda")
        turn = example.angles(example.place(token))
        q, k, v = layer.heads(x, *turn)
        out = attention.window_attention(q, k, v, window=example.WINDOW, sinks=example.FIRST, causal=True,
                                         bias=layer.bias, max_distance=example.REACH)
        weights = layer.weights(x, *turn)
        wide = v.repeat_interleave(example.HEADS // example.KEY_HEADS, 2).transpose(1, 2).contiguous()
        want = (weights.double() @ wide.double()).transpose(1, 2)
    assert (out.double() - want).norm() <= 1e-5 * want.norm()


def test_parameters_all_learn(cuda_device, example):
    torch.manual_seed(2)
    model = example.Generator(layers=1).cuda()
    token = example.clouds(2, 100, 3)
    model(token).float().square().mean().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.abs().sum() > 0, name
