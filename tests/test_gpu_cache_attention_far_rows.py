"""Steps over rows as far apart as one buffer's offsets reach (a tile of 64 rows within 2 GiB), just
below the limit and at it, where other kernels take them, with no numbers between the rows."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cache_attention import LIMIT, close, make, step, want_of
from test_gpu_quantized_cache import TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def room():
    """Two buffers of 129 rows of 2^25 bytes and one of ordinary length."""
    size = 129 * 2 ** 25 + 4096
    return [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]


def apart(t, buffer, stride):
    """A copy of (tokens, heads, width) whose tokens lie `stride` bytes apart."""
    flat = buffer.view(t.dtype)
    flat.fill_(math.nan)
    out = flat.as_strided(t.shape, (stride // t.element_size(), t.shape[2], 1))
    out.copy_(t)
    return out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("stride", [2 ** 25 - 16, 2 ** 25])
@pytest.mark.parametrize("B,N", [(40, 1300), (2, 1300), (2, 60)])  # keys that waves share, parts, one block a sequence
def test_starts(cuda_device, room, kind, stride, B, N):
    q, start, own, _ = make(31, kind, B, 1, 130, N, 4, 2, 128)
    lengths = 1 + torch.arange(B, device="cuda") % 7
    far = [apart(t, x, stride) for t, x in zip(start, room)]
    for how in (dict(), dict(window=90, sinks=3)):
        got = step(q, far, own, lengths, 0, **how)
        close(got, want_of(q, start, own, lengths, 0, **how), LIMIT[kind])
        if stride < 2 ** 25:
            assert torch.equal(got, step(q, start, own, lengths, 0, **how))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("stride", [2 ** 25 - 16, 2 ** 25])
@pytest.mark.parametrize("P", [9, 3000])  # one block a sequence, parts
def test_caches(cuda_device, room, kind, stride, P):
    q, start, own, _ = make(32, kind, 1, 1, P, 130, 4, 2, 128)
    far = [apart(t[0], x, stride)[None] for t, x in zip(own, room)]
    for n in (130, 128, 97, 1):
        lengths = torch.tensor([n], device="cuda")
        got = step(q, start, far, lengths, 0)
        close(got, want_of(q, start, own, lengths, 0), LIMIT[kind])
        if stride < 2 ** 25:
            assert torch.equal(got, step(q, start, own, lengths, 0))
