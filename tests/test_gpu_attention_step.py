"""window_attention_step against window_attention's definition in 64 bits, one
cloud at a time at its own length.

Tolerances as in test_gpu_attention.py: 64 u for float32 and 3 u for the
16-bit types (here the weights' and the result's rounding only)."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import LIMIT, TYPES, close, definition

pytestmark = pytest.mark.gpu


def step_definition(q, k, v, lengths, **how):
    """Each cloud cut to its length; queries before its first position are zeros."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(q.shape[0]):
        n = k.shape[1] if lengths is None else min(max(int(lengths[b]), 0), k.shape[1])
        if n:
            out[b] = definition(q[b:b + 1], k[b:b + 1, :n], v[b:b + 1, :n], None, causal=True, **how)[0][0]
    return out


def run(kind, q, k, v, lengths, **how):
    from mps_pointops.attention import window_attention_step

    print(tuple(q.shape), tuple(k.shape), kind, {n: x for n, x in how.items() if n != "bias"}, flush=True)
    with torch.no_grad():
        out = window_attention_step(q, k, v, lengths, **how)
        assert out.dtype == q.dtype and out.shape == q.shape
        close(out, step_definition(q, k, v, lengths, **how), LIMIT[kind])
        assert torch.equal(out, window_attention_step(q, k, v, lengths, **how))


def make(seed, B, Q, N, H, G, D, dtype, buckets=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    return new(B, Q, H, D), new(B, N, G, D), new(B, N, G, D), new(buckets, H) if buckets else None


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B,Q,N,H,G,D,window,sinks", [
    (2, 1, 1, 1, 1, 1, None, 0), (3, 1, 33, 4, 2, 64, None, 0), (1, 1, 5000, 8, 2, 128, None, 0),
    (2, 1, 3000, 4, 4, 40, 500, 4), (2, 1, 3000, 4, 1, 33, 64, 70), (1, 5, 700, 6, 3, 96, None, 0),
    (2, 3, 1000, 40, 1, 32, 100, 2), (1, 40, 30, 2, 2, 16, None, 0), (1, 7, 2500, 2, 1, 80, 1, 0),
    (5, 1, 300, 33, 33, 24, 17, 1),
])
@pytest.mark.parametrize("biased", [False, True])
def test_step(cuda_device, kind, B, Q, N, H, G, D, window, sinks, biased):
    q, k, v, bias = make(1, B, Q, N, H, G, D, TYPES[kind], 16 if biased else 0)
    how = dict(window=window, sinks=sinks, **(dict(bias=bias, max_distance=50) if biased else {}))
    run(kind, q, k, v, None, **how)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
def test_lengths(cuda_device, kind, bits):
    """Caches of no, one and any number of tokens, fewer than the queries,
    lengths out of range, and no numbers behind them."""
    lengths = torch.tensor([0, 1, 2, 64, 65, 400, 777, -3, 10 ** 6], dtype=bits, device="cuda")
    q, k, v, bias = make(2, 9, 3, 777, 4, 2, 48, TYPES[kind], 12)
    for b, n in enumerate(lengths.clamp(0, 777).tolist()):
        k[b, n:] = math.nan
        v[b, n:] = math.inf
    for how in (dict(), dict(window=40, sinks=5), dict(bias=bias, max_distance=300)):
        run(kind, q, k, v, lengths, **how)


@pytest.mark.parametrize("kind", TYPES)
def test_strides_and_masked_places(cuda_device, kind):
    """A cache with heads before tokens, an unaligned one, and a token that is
    no number outside the window, within the tile of those that are seen."""
    q, k, v, bias = make(3, 2, 1, 600, 4, 2, 64, TYPES[kind], 8)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    run(kind, q, *turned, None, window=100, sinks=3)
    odd = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (k, v)]
    run(kind, q, *odd, None, window=100, sinks=3)
    for value in (math.nan, math.inf, -math.inf):
        for t in (k, v):
            t[:, 480:499, :, 5] = value
            t[:, 7] = value
        run(kind, q, k, v, None, window=100, sinks=3)  # sees 0 .. 2 and 500 ..
        run(kind, q, k, v, None, window=100, sinks=3, bias=bias, max_distance=64)
        two = torch.cat([q, q], 1)
        k[:, 499, 0, 0] = 1.0
        v[:, 499, 1, 1] = value  # seen by the first of two queries alone
        from mps_pointops.attention import window_attention_step
        with torch.no_grad():
            out = window_attention_step(two, k, v, None, window=100, sinks=3)
        want = step_definition(two, k, v, None, window=100, sinks=3)
        close(out[:, 1], want[:, 1], LIMIT[kind])
        assert not torch.isfinite(out[:, 0, 2:, 1]).any()


def test_bias_masks(cuda_device):
    """A bias of -inf for all that is seen leaves zeros; for some, leaves them out."""
    from mps_pointops.attention import window_attention_step

    q, k, v, bias = make(4, 2, 1, 200, 2, 1, 32, torch.float32, 8)
    bias[:, 0] = -math.inf
    bias[4:, 1] = -math.inf
    run("f32", q, k, v, None, bias=bias, max_distance=16)
    with torch.no_grad():
        assert (window_attention_step(q, k, v, None, bias=bias, max_distance=16)[:, :, 0] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
def test_continues_the_whole_pass(cuda_device, kind):
    """Token by token over a growing cache gives the rows of one causal pass,
    each within the tolerance of the definition, so within twice of it."""
    from mps_pointops.attention import window_attention, window_attention_step

    q, k, v, bias = make(5, 2, 60, 60, 4, 2, 32, TYPES[kind], 8)
    how = dict(window=25, sinks=2, bias=bias, max_distance=20)
    with torch.no_grad():
        want = window_attention(q, k, v, causal=True, **how)
        for n in range(1, 61):
            lengths = torch.full((2,), n, device="cuda")
            close(window_attention_step(q[:, n - 1:n], k, v, lengths, **how), want[:, n - 1:n].cpu().double(),
                  2 * LIMIT[kind])


def test_offsets_beyond_32_bits(cuda_device):
    """The last tokens of a cache of more than 2^32 values."""
    N, G, D = (1 << 25) + 40, 1, 128
    k = torch.zeros(1, N, G, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, N, G, D, dtype=torch.bfloat16, device="cuda")
    q, kk, vv, _ = make(6, 1, 1, 64, 2, 1, D, torch.bfloat16)
    k[:, -64:], v[:, -64:] = kk, vv
    from mps_pointops.attention import window_attention_step
    with torch.no_grad():
        out = window_attention_step(q, k, v, None, window=64)
    close(out, step_definition(q, kk, vv, None), LIMIT["bf16"])


def test_replays_in_a_graph(cuda_device):
    """Captured once and replayed with other lengths and tokens, with eager work
    between the replays."""
    from mps_pointops.attention import window_attention_step

    q, k, v, _ = make(7, 2, 1, 2000, 4, 2, 64, torch.bfloat16)
    lengths = torch.tensor([100, 2000], device="cuda")
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            window_attention_step(q, k, v, lengths)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = window_attention_step(q, k, v, lengths)
        for n in (5, 700, 1999, 2000):
            lengths.fill_(n)
            q.normal_()
            graph.replay()
            assert torch.equal(out, window_attention_step(q, k, v, lengths))
            torch.cuda.synchronize()


def test_gradients_are_refused_and_empty_calls(cuda_device):
    from mps_pointops.attention import window_attention_step

    q, k, v, _ = make(8, 1, 1, 8, 2, 1, 8, torch.float32)
    with pytest.raises(ValueError, match="gradients"):
        window_attention_step(q.requires_grad_(), k, v)
    with torch.no_grad():
        assert (window_attention_step(q, k[:, :0], v[:, :0]) == 0).all()
        assert window_attention_step(q[:0], k[:0], v[:0]).shape == (0, 1, 2, 8)
