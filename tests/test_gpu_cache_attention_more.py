"""More of quantized_attention_step and prefix_attention_step: parts of caches, other
layouts, places and sizes.  Tolerances as in test_gpu_cache_attention.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cache_attention import FORMS, LIMIT, close, kept, make, run, step, want_of
from test_gpu_quantized_cache import TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [20, 64, 96, 128])
def test_parts_of_caches(cuda_device, kind, bits, D):
    """A start from the middle of one cloud's cache, own keys from a range of a batch's, and
    lengths with a stride."""
    from mps_pointops.attention import QuantizedCache, cache_write

    q, prefix, own, _ = make(1, kind, 3, 1, 301, 77, 4, 2, D)
    big = QuantizedCache(2, 400, 2, D, bits=bits)
    cache_write(big.cloud(1).positions(5, 306), *(t[None] for t in prefix))
    caches = QuantizedCache(3, 99, 2, D, bits=bits)
    cache_write(caches.positions(11, 88), *own)
    lengths = torch.tensor([77, -1, 30, -1, 1, -1], device="cuda")[::2]
    for how in (dict(), dict(window=50, sinks=2)):
        got = step(q, big.cloud(1).positions(5, 306), caches.positions(11, 88), lengths, bits, **how)
        close(got, want_of(q, prefix, own, lengths, bits, **how), LIMIT[kind])
        got = step(q, None, caches.positions(11, 88), lengths, bits, **how)
        close(got, want_of(q, None, own, lengths, bits, **how), LIMIT[kind])
    many = make(2, kind, 40, 1, 0, 9, 4, 2, D)
    got = step(many[0], big.cloud(1).positions(5, 306), kept(many[2], bits), None, bits)
    close(got, want_of(many[0], prefix, many[2], None, bits), LIMIT[kind])


@pytest.mark.parametrize("bits", FORMS)
def test_shared_keys_beyond_32_bits(cuda_device, bits):
    """Rows of many sequences at the end of a start of more than 2^32 values (4 bits:
    bytes)."""
    P = (1 << 25) + 40 if bits != 4 else (1 << 26) + 40
    q, tail, own, _ = make(3, "bf16", 24, 1, 200, 6, 2, 1, 128)
    from mps_pointops.attention import QuantizedCache, cache_write
    if bits:
        long = QuantizedCache(1, P, 1, 128, bits=bits)
        cache_write(long, *(t[None] for t in tail))
    else:
        long = [torch.zeros(P, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        for t, x in zip(long, tail):
            t[-200:] = x
    lengths = torch.arange(24, device="cuda") % 7
    got = step(q, long, kept(own, bits), lengths, bits, window=150)
    close(got, want_of(q, tail, own, lengths, bits, window=150), LIMIT["bf16"])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B,Q,P,N,H,G,D", [(2, 1, 90, 700, 4, 2, 64), (20, 1, 1500, 40, 4, 2, 128), (3, 1, 2000, 60, 4, 1, 40)])
def test_layouts(cuda_device, kind, B, Q, P, N, H, G, D):
    """Tokens before sequences, one key for all places or all heads, keys and values of
    different strides, and rows far apart; through every kernel that reads rows."""
    q, prefix, own, _ = make(4, kind, B, Q, P, N, H, G, D)
    want = run(kind, q, prefix, own, None, 0)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in own]
    assert torch.equal(run(kind, q, prefix, turned, None, 0), want)
    assert torch.equal(run(kind, q, (prefix[0], prefix[1].transpose(0, 1).contiguous().transpose(0, 1)), (own[0], turned[1]), None, 0), want)
    wide = [torch.zeros(*t.shape[:-1], 2 * D, dtype=t.dtype, device="cuda") for t in prefix]
    for x, t in zip(wide, prefix):
        x[..., D:] = math.nan  # beside the rows
        x[..., :D] = t
    assert torch.equal(run(kind, q, [x[..., :D] for x in wide], own, None, 0), want)
    same = [t[:1].expand(P, -1, -1) for t in prefix]
    run(kind, q, same, [t[:, :1].expand(-1, N, -1, -1) for t in own], None, 0)
    run(kind, q, [t[:, :1].expand(-1, G, -1) for t in prefix], [t[:1].expand(B, -1, -1, -1) for t in own], None, 0)


@pytest.mark.parametrize("bits", FORMS)
def test_many_small_sequences(cuda_device, bits):
    """More sequences than a launch of whole rows takes, of a token or none each."""
    B = 2100
    q, prefix, own, _ = make(5, "f16", B, 1, 300, 3, 2, 1, 32)
    lengths = torch.arange(B, device="cuda") % 4
    got = step(q, kept(prefix, bits), kept(own, bits), lengths, bits)
    some = torch.cat([torch.arange(8), torch.arange(B - 8, B)]).cuda()
    close(got[some], want_of(q[some], prefix, [t[some] for t in own], lengths[some], bits), LIMIT["f16"])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
def test_scores_that_rise_and_fall(cuda_device, kind, bits):
    """Maxima that grow from tile to tile, by little and by much, that fall, and a first
    tile whose scores are far below zero."""
    q, prefix, own, _ = make(6, kind, 5, 1, 700, 90, 4, 2, 64)
    for shape in (torch.linspace(0, 1, 700), torch.linspace(1, 0, 700), torch.linspace(0, 1, 700) ** 8):
        k = prefix[0].float() * (0.1 + 8 * shape.cuda()[:, None, None])
        run(kind, q, (k.to(TYPES[kind]), prefix[1]), own, None, bits)
    k = prefix[0].clone()
    k[:64] = -q[0, 0, 0] * 20  # about -160 for one row, anything for the others
    run(kind, q, (k, prefix[1]), own, None, bits)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("D", [8, 48, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("P", [1281, 1312, 1344, 2111])
def test_shared_rows_of_all_widths(cuda_device, kind, D, P):
    """A start that many sequences' blocks read, inside a longer one: no numbers before it,
    behind it and beside its rows, and in the keys that the window leaves out."""
    q, prefix, own, _ = make(7, kind, 70, 1, P, 5, 4, 2, D)
    wide = [torch.full((P + 70, 2, D + 16), math.nan, dtype=t.dtype, device="cuda") for t in prefix]
    inside = [x[5:P + 5, :, :D] for x in wide]
    for x, t in zip(inside, prefix):
        x.copy_(t)
    lengths = torch.arange(70, device="cuda") % 6
    for window, sinks in ((None, 0), (1290, 3)):
        how = {} if window is None else dict(window=window, sinks=sinks)
        want = want_of(q, prefix, own, lengths, 0, **how)
        if window is not None:
            for x in inside:
                x[sinks:max(sinks, P - window - 3)] = math.nan
        close(step(q, inside, own, lengths, 0, **how), want, LIMIT[kind])
