"""window_attention_step in float16 where one key holds nearly all of a row's weight and its
value is zero: limit and derivation as in test_gpu_cache_attention_weights.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention_step import step_definition
from test_gpu_cache_attention import LIMIT, close
from test_gpu_cache_attention_weights import make

pytestmark = pytest.mark.gpu


def step(*args, **how):
    from mps_pointops.attention import window_attention_step

    with torch.no_grad():
        return window_attention_step(*args, **how)


@pytest.mark.parametrize("gap", [8, 10, 12, 14, 16])
@pytest.mark.parametrize("B,Q,N,H,G,D,where,window", [
    (3, 1, 400, 4, 2, 64, 0, None), (2, 1, 6000, 8, 2, 128, 0, None), (2, 5, 3000, 8, 2, 64, -9, None), (4, 1, 700, 4, 2, 36, 0, None),
    (2, 1, 3000, 4, 1, 96, 0, 600),
])
def test_small_weights(cuda_device, gap, B, Q, N, H, G, D, where, window):
    print(gap, B, Q, N, H, G, D, where, window, flush=True)
    q, start, own = make(2, gap, B, Q, 1, N, H, G, D, -1)
    if where != -1:
        for t in own:
            t[:, [where, -1]] = t[:, [-1, where]]
    how = {} if window is None else dict(window=window, sinks=1)
    close(step(q, *own, None, **how), step_definition(q, *own, None, **how), LIMIT["f16"])


@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 11, 2.0 ** 17, 2.0 ** 24, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28])
@pytest.mark.parametrize("N", [200, 3000])
def test_large_scores(cuda_device, size, N):
    """Three equal scores of `size` (in units of log 2) share a row, two with values of 1 and one of
    0; then one of the first grows by 2^-11, or by a step of 32 bits."""
    q = torch.zeros(2, 1, 2, 64, device="cuda", dtype=torch.float16)
    k, v = (torch.full((2, N, 1, 64), x, device="cuda", dtype=torch.float16) for x in (0.0, 1.0))
    for t in (q, k[:, 5], k[:, N - 7], k[:, N // 2]):
        t[..., :2] = 4096.0  # products of 2^25
    v[:, N // 2] = 0.0
    scale = size / 2 ** 25 * math.log(2)
    assert (step(q, k, v, None, scale=scale) == torch.tensor(2 / 3).half().item()).all()
    k[:, 5, :, 1] = 4100.0
    more = 2.0 ** min(size / 2 ** 11, 100.0)
    # The result's rounding, and as much for the scores' (2^-24 of `size`, in the exponent).
    limit = 2.0 ** -11 + (size * 2.0 ** -23 if size < 2.0 ** 17 else 0.0)
    assert (step(q, k, v, None, scale=scale).double() - (more + 1) / (more + 2)).abs().max() <= limit
    k[:, 5, :, 1] = 4096.0
    k[:, 5, :, 2], q[..., 2] = 1.0, 4.0  # a product of 2^25 + 4, the next of 32 bits
    got = step(q, k, v, None, scale=scale)
    more = 2.0 ** min(size / 2 ** 23, 100.0)
    # (Scores rounded to a step of 32 bits: the difference may be nothing or two steps.)
    low, high = (min(max(x, 0.0), 1.0) for x in (2 / 3 - 2.0 ** -11, (more ** 2 + 1) / (more ** 2 + 2) + 2.0 ** -11))
    assert (got >= low).all() and (got <= high).all() and torch.isfinite(got).all()
