"""quantized_attention_step and prefix_attention_step against attention's
definition in 64 bits, over the values that a cache holds and over each cloud's
start and own keys one behind the other.

Tolerances, as the 2-norm of the difference over that of the result: queries,
keys, weights and values keep their bits, so that a 16-bit result carries its own
rounding, at most u = eps / 2 of each value, and the 32-bit sums' below 2^-12 u; 1.02 u
and room for the hardware's exponential (2^-20).  Float32, as window_attention_step's: sums of
a few hundred terms and an exponent below 2^4, well below 64 u.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import definition
from test_gpu_quantized_cache import TYPES, held

pytestmark = pytest.mark.gpu

LIMIT = {"f32": 64 * 2.0 ** -24, "f16": 1.02 * 2.0 ** -11 + 2.0 ** -20, "bf16": 1.02 * 2.0 ** -8 + 2.0 ** -20}
FORMS = [0, 8, 4]


def close(got, want, limit):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    assert (got - want).norm() <= limit * want.norm(), ((got - want).norm() / want.norm()).item()


def make(seed, kind, B, Q, P, N, H, G, D, buckets=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda").to(TYPES[kind])  # noqa: E731
    return (new(B, Q, H, D), (new(P, G, D), new(P, G, D)), (new(B, N, G, D), new(B, N, G, D)),
            new(buckets, H) if buckets else None)


def kept(pair, bits):
    """The pair itself, or a cache that holds it."""
    from mps_pointops.attention import QuantizedCache, cache_write

    if not bits:
        return pair
    k, v = (t[None] if t.ndim == 3 else t for t in pair)
    cache = QuantizedCache(*k.shape, bits=bits)
    cache_write(cache, k, v)
    return cache


def want_of(q, prefix, own, lengths, bits, **how):
    """Each cloud's start and own keys, cut to its length."""
    if bits:
        prefix, own = (None if pair is None else [held(t, bits)[0] for t in pair] for pair in (prefix, own))
    else:
        prefix, own = (None if pair is None else [t.cpu().double() for t in pair] for pair in (prefix, own))
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(q.shape[0]):
        n = own[0].shape[1] if lengths is None else min(max(int(lengths[b]), 0), own[0].shape[1])
        k, v = (t[b:b + 1, :n] for t in own)
        if prefix is not None:
            k, v = (torch.cat([t[None], x], 1) for t, x in zip(prefix, (k, v)))
        if k.shape[1]:
            out[b] = definition(q[b:b + 1], k, v, None, causal=True, **how)[0][0]
    return out


def step(q, prefix, own, lengths, bits, **how):
    from mps_pointops.attention import prefix_attention_step, quantized_attention_step

    with torch.no_grad():
        if prefix is None:
            return quantized_attention_step(q, own, lengths, **how)
        return prefix_attention_step(q, prefix, own, lengths, **how)


def run(kind, q, prefix, own, lengths, bits, **how):
    print(kind, bits, tuple(q.shape), None if prefix is None else tuple(prefix[0].shape), tuple(own[0].shape),
          {n: x for n, x in how.items() if n != "bias"}, flush=True)
    held_prefix = None if prefix is None else kept(prefix, bits)
    held_own = kept(own, bits)
    got = step(q, held_prefix, held_own, lengths, bits, **how)
    assert got.dtype == q.dtype and got.is_contiguous()
    close(got, want_of(q, prefix, own, lengths, bits, **how), LIMIT[kind])
    assert torch.equal(got, step(q, held_prefix, held_own, lengths, bits, **how))
    return got


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("B,Q,N,H,G,D,window,sinks", [
    (2, 1, 1, 1, 1, 1, None, 0), (3, 1, 33, 4, 2, 64, None, 0), (1, 1, 5000, 8, 2, 128, None, 0),
    (2, 1, 3000, 4, 4, 40, 500, 4), (2, 1, 3000, 4, 1, 33, 64, 70), (1, 5, 700, 6, 3, 96, None, 0),
    (2, 3, 1000, 40, 1, 32, 100, 2), (1, 40, 30, 2, 2, 16, None, 0), (1, 7, 2500, 2, 1, 80, 1, 0), (5, 1, 300, 33, 33, 24, 17, 1),
])
@pytest.mark.parametrize("biased", [False, True])
def test_quantized(cuda_device, kind, bits, B, Q, N, H, G, D, window, sinks, biased):
    q, _, own, bias = make(1, kind, B, Q, 0, N, H, G, D, 16 if biased else 0)
    run(kind, q, None, own, None, bits, window=window, sinks=sinks, **(dict(bias=bias, max_distance=50) if biased else {}))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
@pytest.mark.parametrize("B,Q,P,N,H,G,D,window,sinks", [
    (1, 1, 1, 1, 1, 1, 1, None, 0), (3, 1, 65, 9, 4, 2, 64, None, 0), (8, 1, 3000, 40, 8, 2, 128, None, 0), (2, 1, 700, 300, 4, 4, 40, 500, 4),
    (4, 1, 500, 90, 4, 1, 33, 64, 70), (2, 5, 300, 100, 6, 3, 96, None, 0), (6, 3, 400, 11, 40, 1, 32, 100, 2), (3, 40, 20, 50, 2, 2, 16, None, 0),
    (5, 2, 1000, 7, 2, 1, 80, 1, 0), (21, 1, 130, 60, 66, 33, 24, 100, 1), (40, 1, 257, 31, 6, 2, 56, None, 0), (2, 1, 40, 3000, 4, 2, 128, None, 3),
])
@pytest.mark.parametrize("biased", [False, True])
def test_prefix(cuda_device, kind, bits, B, Q, P, N, H, G, D, window, sinks, biased):
    q, prefix, own, bias = make(2, kind, B, Q, P, N, H, G, D, 16 if biased else 0)
    gen = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, N + 1, (B,), generator=gen).cuda()
    run(kind, q, prefix, own, lengths, bits, window=window, sinks=sinks, **(dict(bias=bias, max_distance=50) if biased else {}))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
@pytest.mark.parametrize("bits_of_lengths", [torch.int32, torch.int64])
def test_lengths(cuda_device, kind, bits, bits_of_lengths):
    """Caches of no, one and any number of tokens, fewer than the queries, lengths
    out of range, and no numbers behind them; with a start of one key, of none, and
    (over codes) without one."""
    lengths = torch.tensor([0, 1, 2, 64, 65, 400, 777, -3, 10 ** 6], dtype=bits_of_lengths, device="cuda")
    for P in (0, 1, 90):
        q, prefix, own, bias = make(3, kind, 9, 3, P, 777, 4, 2, 48, 12)
        for b, n in enumerate(lengths.clamp(0, 777).tolist()):
            own[0][b, n:] = math.nan
            own[1][b, n:] = math.inf
        for how in (dict(), dict(window=40, sinks=5), dict(bias=bias, max_distance=300)):
            run(kind, q, prefix, own, lengths, bits, **how)
            if bits and P == 0:
                run(kind, q, None, own, lengths, bits, **how)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
def test_masked_places_that_are_no_numbers(cuda_device, kind, bits):
    """Keys and values outside the window, in the tiles of those that are seen, in
    the start and in the caches; and one that some rows see and others do not."""
    q, prefix, own, bias = make(4, kind, 3, 1, 600, 90, 4, 2, 64, 8)
    lengths = torch.tensor([90, 50, 1], device="cuda")  # windows from 590, 550, 501
    for value in (math.nan, math.inf, -math.inf):
        for t in prefix:
            t[480:499, :, 5] = value
            t[7] = value
        for how in (dict(), dict(bias=bias, max_distance=64)):
            run(kind, q, prefix, own, lengths, bits, window=100, sinks=3, **how)
        k, v = (t.clone() for t in prefix)
        v[520] = value  # seen by the last cloud alone
        got = step(q, kept((k, v), bits), kept(own, bits), lengths, bits, window=100, sinks=3)
        want = want_of(q, (k, v), own, lengths, bits, window=100, sinks=3)
        close(got[:2], want[:2], LIMIT[kind])
        assert not torch.isfinite(got[2]).any()
        mine = own[0].clone(), own[1].clone()
        mine[0][0, 40], mine[1][1, 30, 1] = value, value
        got = step(q, kept(prefix, bits), kept(mine, bits), lengths, bits, window=30, sinks=3)
        want = want_of(q, prefix, mine, lengths, bits, window=30, sinks=3)
        close(got[0], want[0], LIMIT[kind])
        close(got[1, :, :2], want[1, :, :2], LIMIT[kind])
        assert not torch.isfinite(got[1, :, 2:]).any()


@pytest.mark.parametrize("bits", FORMS)
def test_bias_masks(cuda_device, bits):
    """A bias of -inf for all that is seen leaves zeros, for some leaves them out, no
    numbers there too; the type's lowest value for all keys weighs them alike."""
    q, prefix, own, bias = make(5, "f32", 3, 2, 130, 60, 4, 2, 32, 8)
    bias[:, 0] = -math.inf
    bias[4:, 1] = -math.inf
    bias[:, 2] = torch.finfo(torch.float32).min
    got = run("f32", q, prefix, own, None, bits, bias=bias, max_distance=16)
    assert (got[:, :, 0] == 0).all()
    bias[:, 0] = 0.0
    bias[7] = -math.inf  # 16 and more away
    for t in prefix:
        t[:100] = 0.0  # (the definition adds the bias to what lies there)
    want = want_of(q, prefix, own, None, bits, bias=bias, max_distance=16)
    prefix[0][:100], prefix[1][:100] = math.nan, math.inf
    close(step(q, kept(prefix, bits), kept(own, bits), None, bits, bias=bias, max_distance=16), want, LIMIT["f32"])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
def test_large_tables(cuda_device, kind, bits):
    """The most buckets with many heads a key head, whose table and the widest
    rows' tiles do not fit one block together."""
    for B, H, D, P in ((3, 64, 128, 1500), (2, 128, 100, 1400), (3, 9, 128, 1500), (40, 4, 128, 1300)):
        q, prefix, own, bias = make(15, kind, B, 1, P, 9, H, 1, D, 256)
        run(kind, q, prefix, own, None, bits, bias=bias, max_distance=1000)


@pytest.mark.parametrize("kind", TYPES)
def test_strides_and_alignment(cuda_device, kind):
    """Heads before tokens, rows that start anywhere, one start broadcast over its
    heads, queries cut from a projection, a last dimension that is not contiguous."""
    q, prefix, own, _ = make(6, kind, 3, 2, 200, 70, 4, 2, 64)
    turned = [t.transpose(-3, -2).contiguous().transpose(-3, -2) for t in (*prefix, *own)]
    want = run(kind, q, prefix, own, None, 0, window=150)
    assert torch.equal(run(kind, q, turned[:2], turned[2:], None, 0, window=150), want)
    odd = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (*prefix, *own)]
    run(kind, q, odd[:2], odd[2:], None, 0, window=150)
    run(kind, q, prefix, odd[2:], None, 0)
    one = [t[:, :1].expand(-1, 2, -1) for t in prefix]
    run(kind, q, one, own, None, 0)
    wide = torch.randn(3, 2, 9, 64, device="cuda").to(TYPES[kind])[:, :, 3:7]
    for bits in FORMS:
        run(kind, wide, prefix, own, None, bits)
        run(kind, torch.cat([wide.flatten()[:1], wide.flatten()])[1:].view(wide.shape), prefix, own, None, bits)
    run(kind, q.transpose(2, 3).contiguous().transpose(2, 3), [t.transpose(1, 2).contiguous().transpose(1, 2) for t in prefix], own, None, 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", FORMS)
def test_agrees_with_the_step(cuda_device, kind, bits):
    """Over the same values, with the start copied before every cloud's cache, as
    window_attention_step, whose weights keep their bits too; and token by token over a
    growing cache."""
    from mps_pointops.attention import cache_read, window_attention_step

    q, prefix, own, bias = make(7, kind, 4, 1, 333, 50, 8, 2, 96, 10)
    a, b = kept(prefix, bits), kept(own, bits)
    if bits:
        whole_prefix, whole_own = cache_read(a, dtype=TYPES[kind]), cache_read(b, dtype=TYPES[kind])
    else:
        whole_prefix, whole_own = [t[None] for t in prefix], own
    k, v = (torch.cat([s.expand(4, -1, -1, -1), t], 1) for s, t in zip(whole_prefix, whole_own))
    for n in range(0, 51, 10):
        lengths = torch.full((4,), n, device="cuda")
        how = dict(window=200, sinks=2, bias=bias, max_distance=100)
        with torch.no_grad():
            want = window_attention_step(q, k, v, 333 + lengths, **how)
        close(step(q, a, b, lengths, bits, **how), want.cpu().double(), 2 * LIMIT[kind])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(cuda_device, kind, scale):
    """None, negative and large ones."""
    q, prefix, own, _ = make(8, kind, 2, 1, 100, 30, 4, 2, 40)
    for bits in FORMS:
        run(kind, q, prefix, own, None, bits, scale=scale)


@pytest.mark.parametrize("bits", [8, 4])
def test_queries_that_are_no_numbers(cuda_device, bits):
    """Give rows without numbers, and others' rows are as they were."""
    q, prefix, own, _ = make(9, "f32", 4, 1, 100, 30, 4, 2, 64)
    a, b = kept(prefix, bits), kept(own, bits)
    want = step(q, a, b, None, bits)
    q[1, 0, 2, 7], q[2, 0, 1, 3] = math.nan, math.inf
    got = step(q, a, b, None, bits)
    assert torch.isnan(got[1, 0, 2]).all() and torch.isnan(got[2, 0, 1]).all()
    got[1, 0, 2], got[2, 0, 1] = want[1, 0, 2], want[2, 0, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("bits", FORMS)
def test_offsets_beyond_32_bits(cuda_device, bits):
    """The last tokens of a cache of more than 2^32 values (4 bits: of bytes)."""
    N = (1 << 25) + 40 if bits != 4 else (1 << 26) + 40
    q, prefix, own, _ = make(10, "bf16", 1, 1, 64, 64, 2, 1, 128)
    from mps_pointops.attention import QuantizedCache, cache_write
    if bits:
        cache = QuantizedCache(1, N, 1, 128, bits=bits)
        cache_write(cache, *own)
    else:
        cache = [torch.zeros(1, N, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        for t, x in zip(cache, own):
            t[:, -64:] = x
    got = step(q, kept(prefix, bits), cache, None, bits, window=64)
    close(got, want_of(q, None, own, None, bits), LIMIT["bf16"])
    long = cache if bits else [t[0] for t in cache]
    tail = make(11, "bf16", 1, 1, 0, 1, 2, 1, 128)[2]
    got = step(q, long, kept(tail, bits), None, bits, window=65)
    close(got, want_of(q, [t[0] for t in own], tail, None, bits), LIMIT["bf16"])


@pytest.mark.parametrize("bits", FORMS)
def test_replays_in_a_graph(cuda_device, bits):
    """Captured once and replayed with other lengths, tokens and queries, with eager
    work between the replays."""
    q, prefix, own, _ = make(12, "bf16", 3, 1, 700, 300, 8, 2, 64)
    a, b = kept(prefix, bits), kept(own, bits)
    lengths = torch.tensor([1, 100, 300], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, a, b, lengths, bits)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # each with its own workspace
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(q, a, b, lengths, bits))
    for n in (0, 5, 299, 300):
        lengths.fill_(n)
        q.normal_()
        for graph in graphs:
            graph.replay()
        want = step(q, a, b, lengths, bits)
        for out in outs:
            assert torch.equal(out, want)
        torch.cuda.synchronize()


def test_two_streams(cuda_device):
    """Two calls at once do not share memory."""
    q, prefix, own, _ = make(13, "bf16", 8, 1, 5000, 100, 8, 2, 128)
    want = step(q, prefix, own, None, 0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step(q, prefix, own, None, 0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("bits", FORMS)
def test_empty_calls(cuda_device, bits):
    q, prefix, own, _ = make(14, "f32", 2, 1, 5, 4, 2, 1, 8)
    a = kept(prefix, bits)
    none = kept([t[:, :0] for t in own], bits)
    close(step(q, a, none, None, bits), want_of(q, prefix, [t[:, :0] for t in own], None, bits), LIMIT["f32"])
    if bits:
        assert (step(q, None, none, None, bits) == 0).all()
    nothing = kept([t[:0] for t in prefix], bits)
    assert (step(q, nothing, none, None, bits) == 0).all()
    empty = kept([t[:0] for t in own], bits)
    assert step(q[:0], a, empty, None, bits).shape == (0, 1, 2, 8)
    assert step(q[:, :0], a, kept(own, bits), None, bits).shape == (2, 0, 2, 8)
