"""Steps over kept keys whose values are near the largest of 32 bits: a weighted mean of them is
finite, also where a sum of them is not.  Tolerances as in test_gpu_cache_attention.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_cache_attention import LIMIT, close, kept, make, step, want_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("B,Q,P,N,H,G,D", [
    (3, 1, 400, 60, 4, 2, 64), (1, 1, 6000, 300, 4, 2, 64), (40, 1, 3000, 20, 4, 2, 128), (3, 5, 3000, 70, 8, 2, 32), (4, 1, 500, 40, 4, 2, 33),
])
@pytest.mark.parametrize("largest", [1e37, 2e38])
def test_large_values(cuda_device, kind, bits, B, Q, P, N, H, G, D, largest):
    """Scores that rise from key to key by less than 8 (in units of log 2) in all, over the start and the
    caches; some columns of the values large, others of ordinary size, and signs of both kinds."""
    print(kind, bits, B, Q, P, N, H, G, D, largest, flush=True)
    q, start, own, _ = make(21, kind, B, Q, P, N, H, G, D)
    q *= 0.125
    q[..., 0] = 1.0
    rise = torch.linspace(0, 5.4 * D ** 0.5, P + N, device="cuda")
    start[0][..., 0] = rise[:P, None]
    own[0][..., 0] = rise[None, P:, None]
    for k, v in (start, own):
        v[..., 1::3] = v[..., 1::3].abs().clamp(max=1.0) * largest
        v[..., 2::3] = v[..., 2::3].sign() * largest
    lengths = N - torch.arange(B, device="cuda") % 3
    a, b = kept(start, bits), kept(own, bits)
    got, want = step(q, a, b, lengths, bits), want_of(q, start, own, lengths, bits)
    close(got, want, LIMIT[kind])
    close(got[..., ::3], want[..., ::3], LIMIT[kind])
    if bits:
        close(step(q, None, a if B == 1 else b, None, bits), want_of(q, None, [t[None] for t in start] if B == 1 else own, None, bits), LIMIT[kind])
    # The same with a value that is no number, which only its own column shows.
    start[1][P - 3, :, 0] = float("nan")
    got = step(q, kept(start, bits), b, lengths, bits)
    if not bits:
        assert torch.isnan(got[..., 0]).all() and torch.isfinite(got[..., 1:]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("B,P,N,D", [(1, 6000, 300, 64), (2, 40, 5000, 128), (40, 3000, 20, 128), (4, 500, 40, 64)])
def test_few_keys_of_large_values(cuda_device, kind, bits, B, P, N, D):
    """Some keys of equal scores far above the others', with the same large value: each part's sum is
    finite, and that of all parts is not."""
    print(kind, bits, B, P, N, D, flush=True)
    large = 1.5e38 if bits == 4 else 3e38  # (3e38 is 3.53 x 2^126, which 4 bits round to 2^128)
    q, start, own, _ = make(22, kind, B, 1, P, N, 4, 2, D)
    q[..., 0] = 8.0
    for k, v in (start, own):
        keys = k.shape[-3]
        k[..., 0] = 0.0
        some = k[..., ::max(1, keys // 5), :, :]
        some.zero_()
        some[..., 0] = 5.0 * D ** 0.5
        v[..., ::max(1, keys // 5), :, 1::2] = large
    got = step(q, kept(start, bits), kept(own, bits), None, bits)
    want = want_of(q, start, own, None, bits)
    close(got, want, LIMIT[kind])
    close(got[..., ::2], want[..., ::2], LIMIT[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("B,P,N,window", [(3, 400, 60, 300), (2, 6000, 90, 4000), (40, 3000, 20, 2500)])
def test_columns_beside_those_formed_again(cuda_device, kind, bits, B, P, N, window):
    """A masked value that is no number has one column formed again: the others, near the type's smallest
    numbers, keep their bits."""
    q, start, own, _ = make(23, kind, B, 1, P, N, 4, 2, 64)
    start[1].mul_(1e-33)
    own[1].mul_(1e-33)
    how = dict(window=window, sinks=1)
    a, b = kept(start, bits), kept(own, bits)
    want = step(q, a, b, None, bits, **how)
    low = P + N - window
    start[1][low - 3:low, :, 5] = float("nan")  # in the tile of the first keys that are seen
    got = step(q, kept(start, bits), b, None, bits, **how)
    some = [c for c in range(64) if c != 5] if not bits else list(range(32, 64))
    assert torch.equal(got[..., some], want[..., some])
    assert torch.isfinite(got).all()
    assert (got.double() - want.double()).norm() <= 2 * LIMIT[kind] * want.double().norm()
