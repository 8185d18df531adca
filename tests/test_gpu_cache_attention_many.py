"""Caches and steps of more blocks than a launch holds along one dimension (2^32 threads: 2^24
blocks), of a token or two each, whose results are the values kept: exact numbers."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def values(*shape, dtype=torch.bfloat16):
    """Whole numbers of either sign that 4 bits hold exactly beside others of their size."""
    new = torch.randint(0, 2, shape, device="cuda", dtype=torch.int8)
    return (4 + 2 * new).to(dtype)


@pytest.mark.parametrize("bits", [8, 4])
def test_write_and_read(cuda_device, bits):
    from mps_pointops.attention import QuantizedCache, cache_read, cache_write

    B, G, D = (1 << 18) + 3, 32, 7  # 2^24 + 192 blocks
    cache = QuantizedCache(B, 2, G, D, bits=bits)
    k, v = values(B, 1, G, D), values(B, 1, G, D)
    cache_write(cache, k, -v)
    got = cache_read(cache)
    assert torch.equal(got[0][:, 1:], k) and torch.equal(got[1][:, 1:], -v) and not got[0][:, 0].any()
    cache_write(cache, -k, v, starts=torch.zeros(B, dtype=torch.int64, device="cuda"))
    got = cache_read(cache)
    assert torch.equal(got[0], torch.cat([-k, k], 1)) and torch.equal(got[1], torch.cat([v, -v], 1))


@pytest.mark.parametrize("bits", [8, 0])
def test_steps(cuda_device, bits):
    """One key a sequence; over codes without a start, over rows behind one of a key that
    weighs nothing."""
    from mps_pointops.attention import QuantizedCache, cache_write, prefix_attention_step, quantized_attention_step

    B, G, D = (1 << 19) + 3, 32, 8  # 2^24 + 96 blocks
    q, k, v = torch.ones(B, 1, G, D, device="cuda", dtype=torch.bfloat16), values(B, 1, G, D), values(B, 1, G, D)
    with torch.no_grad():
        if bits:
            cache = QuantizedCache(B, 1, G, D, bits=bits)
            cache_write(cache, k, v)
            got = quantized_attention_step(q, cache)
        else:
            start = [torch.full((1, G, D), x, device="cuda", dtype=torch.bfloat16) for x in (-1000.0, 5.0)]
            got = prefix_attention_step(q, start, (k, v))
    assert torch.equal(got, v)


def test_joins(cuda_device):
    """2^26 rows and some, whose parts a second launch joins."""
    from mps_pointops.attention import prefix_attention_step

    B, G, D = (1 << 21) + 3, 32, 1
    q, k, v = torch.ones(B, 1, G, D, device="cuda", dtype=torch.bfloat16), values(B, 1, G, D), values(B, 1, G, D)
    start = [torch.full((1, G, D), x, device="cuda", dtype=torch.bfloat16) for x in (-1000.0, 5.0)]
    with torch.no_grad():
        got = prefix_attention_step(q, start, (k, v))
    assert torch.equal(got, v)
