"""prefix_attention_step in float16 where one key holds nearly all of a row's weight and its
value is zero, as first keys do that a model's heads rest on: the result is what the other
keys' small weights make of their values.

Limit: that of test_gpu_cache_attention.py, one rounding of the result.  A weight is the sum of
two float16 values, off by at most 2^-37 of the row's largest (half a step of 2^-24, the largest
being 2^12 and more).  With the others' scores of a deviation of 1, a gap of g to their mean and
values of one size, the roundings' share of the result is at most 2^-37 / (e^(1 - g)), for g = 16 2^-15.4:
beside a rounding of 2^-11 (at most; their squares add) below the limit's 2 %."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cache_attention import LIMIT, close, step, want_of

pytestmark = pytest.mark.gpu


def make(seed, gap, B, Q, P, N, H, G, D, where):
    """Key `where` (of the start, or, negative, of the caches from the end) has scores of `gap` and values of zero, the
    others scores of deviation 1 and values whose weighted sums are normal numbers of float16."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    q, start, own = new(B, Q, H, D), [new(P, G, D), 2000 * new(P, G, D)], [new(B, N, G, D), 2000 * new(B, N, G, D)]
    q[..., 0] = 4
    for keys in (start[0], own[0]):
        keys[..., 0] = 0
    k, v = ((t[where] for t in start) if where >= 0 else (t[:, where] for t in own))
    k.zero_()
    k[..., 0] = gap * D ** 0.5 / 4
    v.zero_()
    return q.half(), [t.half() for t in start], [t.half() for t in own]


@pytest.mark.parametrize("gap", [8, 10, 12, 14, 16])
@pytest.mark.parametrize("B,Q,P,N,H,G,D,where", [
    (3, 1, 400, 60, 4, 2, 64, 0),  # one block a sequence
    (1, 1, 6000, 300, 4, 2, 64, 3), (2, 1, 40, 5000, 8, 2, 128, 0),  # parts
    (12, 1, 4000, 30, 4, 2, 64, 0), (40, 1, 3000, 20, 4, 2, 128, 0), (40, 1, 3000, 20, 4, 2, 96, 2999),  # keys that waves share
    (3, 5, 3000, 70, 8, 2, 64, 1),  # more than 16 rows a key head
    (4, 1, 500, 40, 4, 2, 36, 0), (2, 1, 2000, 3000, 4, 2, 33, -1),  # rows of no whole pieces
])
def test_small_weights(cuda_device, gap, B, Q, P, N, H, G, D, where):
    print(gap, B, Q, P, N, H, G, D, where, flush=True)
    q, start, own = make(1, gap, B, Q, P, N, H, G, D, where)
    close(step(q, start, own, None, 0), want_of(q, start, own, None, 0), LIMIT["f16"])


@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 11, 2.0 ** 17, 2.0 ** 24, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28])
@pytest.mark.parametrize("P,B", [(200, 2), (3000, 40)])
def test_large_scores(cuda_device, size, P, B):
    """Scores whose steps in 32 bits reach the weights' range: three equal ones of `size` (in units
    of log 2) share a row, two with values of 1 and one of 0; then one of the first grows by 2^-11."""
    q = torch.zeros(B, 1, 2, 64, device="cuda", dtype=torch.float16)
    start = [torch.full((P, 1, 64), x, device="cuda", dtype=torch.float16) for x in (0.0, 1.0)]
    own = [torch.zeros(B, 9, 1, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    for t in (q, start[0][5], start[0][P - 7], own[0][:, 2]):
        t[..., :2] = 4096.0  # products of 2^25
    scale = size / 2 ** 25 * math.log(2)
    got = step(q, start, own, None, 0, scale=scale)
    assert (got == torch.tensor(2 / 3).half().item()).all()
    start[0][5, :, 1] = 4100.0
    more = 2.0 ** min(size / 2 ** 11, 100.0)
    got = step(q, start, own, None, 0, scale=scale)
    # The result's rounding, and as much for the scale's in the exponent (2^-23 of an eighth to one).
    assert (got.double() - (more + 1) / (more + 2)).abs().max() <= 2.0 ** -11
