"""The example's caches: steps over keys and values in 8 and 4 bits, several tokens
at once, and continuations that share their start's cache."""

from __future__ import annotations

import pytest
import torch

from test_gpu_ordered_points import example  # noqa: F401

pytestmark = pytest.mark.gpu

# Float32 throughout: two layers of sums in another order.  A key or value that lies on a code's
# border may take the one beside it by that, 1/8 (8 bits) or 1/2 (4 bits) of one of 64 values of a
# token that up to 66 others weigh: below 2^-9 and 2^-7 of all logits' norm.
LIMIT = {32: 2e-5, 8: 2.0 ** -9, 4: 2.0 ** -7}


@pytest.fixture(scope="module")
def model(example):  # noqa: F811
    torch.manual_seed(3)
    return example.Generator().cuda()


@pytest.mark.parametrize("bits", [8, 4])
def test_steps_over_codes(cuda_device, example, model, bits):  # noqa: F811
    """One token after another gives what a chunk of all gives."""
    token = example.clouds(2, 120, 5)
    single = example.replay(model, token, bits)
    whole = model.step(token, model.cache(2, 120, bits), 0)
    assert (single - whole).norm() <= LIMIT[bits] * whole.norm()
    assert example.generate(model, token[:, :60], 90, bits).shape == (2, 90)


@pytest.mark.parametrize("bits", [32, 8, 4])
def test_a_shared_start(cuda_device, example, model, bits):  # noqa: F811
    """Continuations of one start give the logits of the same tokens with the start repeated for
    each."""
    start = example.clouds(1, 100, 6)[0]
    many = example.continue_many(model, start, 5, 40, bits)
    assert many.shape == (5, 140) and torch.equal(many[:, :100], start.expand(5, -1))
    assert len({tuple(row.tolist()) for row in many}) > 1
    prefix = model.cache(1, 100, bits)
    model.step(start[None], prefix, 0)
    if bits == 32:
        prefix = [(k[0], v[0]) for k, v in prefix]
    cache = model.cache(5, 40, bits)
    got = torch.cat([model.step(many[:, 100 + n:101 + n], cache, n, prefix) for n in range(40)], 1)
    want = example.replay(model, many, bits)[:, 100:]
    assert (got - want).norm() <= LIMIT[bits] * want.norm()
    assert torch.equal(many, example.continue_many(model, start, 5, 40, bits))
