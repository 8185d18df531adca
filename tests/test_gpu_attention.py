"""window_attention against its definition in 64 bits: outputs and gradients
over types, head layouts, lengths, windows, first keys, biases and strides,
with rows that see nothing and masked places that hold no numbers.

Tolerances, as the 2-norm of the difference over that of the result.  u is half
the spacing of the type's values at 1 (2^-24, 2^-11, 2^-8 is the spacing of
bfloat16, 2^-9 its half): float32 results carry the roundings of sums of up to a
few hundred terms and of an exponent of magnitude below 2^4, well below 64 u;
16-bit ones the rounding of the weights, of ds, of the output that delta is
formed from and of the result, each at most u and not all at once: 3 u.  A sum
over offsets that cancels (the bias's gradient) is allowed as much of the sum
of its terms' magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = {"f32": 64 * 2.0 ** -24, "f16": 3 * 2.0 ** -11, "bf16": 3 * 2.0 ** -8}


def bucket_matrix(offset, buckets, max_distance, causal):
    from mps_pointops.attention import bucket_edges

    side = buckets if causal else buckets // 2
    edges = torch.tensor(bucket_edges(side, max_distance))
    d = offset.clamp(min=0) if causal else offset.abs()
    bucket = (d[..., None] >= edges).sum(-1)
    return bucket if causal else bucket + side * (offset < 0)


def visible(Q, N, window, sinks, causal, length):
    p = torch.arange(N - Q, N)[:, None]
    j = torch.arange(N)
    seen = (j < length) & (p >= 0) & (p < length)
    if window is not None:
        seen = seen & (((p - j).abs() < window) | (j < sinks))
    return seen & (j <= p) if causal else seen


def definition(q, k, v, grad, window=None, sinks=0, causal=False, bias=None, max_distance=None, lengths=None,
               scale=None):
    """Outputs, gradients and the magnitudes of the bias's gradient, in 64
    bits on the CPU; masked places take no part at all."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, Q, H, D = q.shape
    N, G = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    table = None if bias is None else bias.detach().cpu().double()
    dbias = None if bias is None else torch.zeros_like(table)
    size = None if bias is None else torch.zeros_like(table)
    g = None if grad is None else grad.detach().cpu().double()
    for b in range(B):
        length = N if lengths is None else min(max(int(lengths[b]), 0), N)
        seen = visible(Q, N, window, sinks, causal, length)
        offset = torch.arange(N - Q, N)[:, None] - torch.arange(N)
        bucket = None if table is None else bucket_matrix(offset, table.shape[0], max_distance, causal)
        for h in range(H):
            kk, vv = k[b, :, h * G // H], v[b, :, h * G // H]
            for i in range(Q):
                at = seen[i].nonzero()[:, 0]
                if not len(at):
                    continue
                s = kk[at] @ q[b, i, h] * scale
                if table is not None:
                    s = s + table[bucket[i, at], h]
                    at, s = at[s != -math.inf], s[s != -math.inf]
                    if not len(at):
                        continue
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ vv[at]
                if g is None:
                    continue
                dp = vv[at] @ g[b, i, h]
                ds = p * (dp - (p * dp).sum())
                dv[b, at, h * G // H] += p[:, None] * g[b, i, h]
                dq[b, i, h] = scale * ds @ kk[at]
                dk[b, at, h * G // H] += scale * ds[:, None] * q[b, i, h]
                if table is not None:
                    dbias[:, h].index_add_(0, bucket[i, at], ds)
                    size[:, h].index_add_(0, bucket[i, at], ds.abs())
    return out, dq, dk, dv, dbias, size


def close(got, want, limit, size=None):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    norm = (want if size is None else size).norm()
    assert (got - want).norm() <= limit * norm, ((got - want).norm() / norm).item()


def tensors(seed, B, Q, N, H, G, D, dtype, buckets=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    return make(B, Q, H, D), make(B, N, G, D), make(B, N, G, D), make(B, Q, H, D), make(buckets, H) if buckets else None


def check(kind, q, k, v, grad, **how):
    from mps_pointops.attention import window_attention

    bias = how.get("bias")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([] if bias is None else [bias.detach().requires_grad_()])
    print(tuple(q.shape), tuple(k.shape), kind, {n: x for n, x in how.items() if n not in ("bias", "lengths")}, flush=True)
    out = window_attention(*leaves[:3], **{**how, **({} if bias is None else {"bias": leaves[3]})})
    assert out.dtype == q.dtype and out.shape == q.shape
    got = torch.autograd.grad(out, leaves, grad)
    for t, x in zip(leaves, got):
        assert x.dtype == t.dtype
    want = definition(q, k, v, grad, **how)
    close(out, want[0], LIMIT[kind])
    for x, y in zip(got[:3], want[1:4]):
        close(x, y, LIMIT[kind])
    if bias is not None:
        close(got[3], want[4], LIMIT[kind], want[5])
    again = torch.autograd.grad(window_attention(*leaves[:3], **{**how, **({} if bias is None else {"bias": leaves[3]})}),
                                leaves, grad)
    assert all(torch.equal(x, y) for x, y in zip(got, again))  # no sum depends on chance


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B,Q,N,H,G,D", [
    (1, 1, 1, 1, 1, 1), (2, 5, 5, 2, 1, 20), (1, 64, 64, 1, 1, 32), (2, 129, 129, 2, 2, 33), (1, 200, 200, 3, 1, 64),
    (1, 70, 333, 2, 1, 80), (1, 257, 257, 1, 1, 128), (1, 100, 100, 4, 2, 96), (1, 40, 9, 1, 1, 16), (1, 1, 300, 2, 2, 40),
])
@pytest.mark.parametrize("causal", [False, True])
def test_every_key(cuda_device, kind, B, Q, N, H, G, D, causal):
    q, k, v, g, _ = tensors(1, B, Q, N, H, G, D, TYPES[kind])
    if N == 1 or (causal and Q == 1 and N == 1):
        pytest.skip("one key: every gradient but v's is zero")
    check(kind, q, k, v, g, causal=causal)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("Q,N,window,sinks,causal", [
    (300, 300, 1, 1, True), (300, 300, 40, 0, True), (300, 300, 40, 3, True), (300, 300, 33, 0, False),
    (300, 300, 33, 70, False), (300, 300, 64, 64, True), (300, 300, 500, 5, False), (50, 300, 20, 4, True),
    (50, 300, 20, 150, False), (300, 120, 30, 2, True), (2000, 2000, 17, 130, True), (1500, 1500, 60, 2, False),
])
def test_windows_and_first_keys(cuda_device, kind, Q, N, window, sinks, causal):
    q, k, v, g, _ = tensors(2, 1, Q, N, 2, 1, 24, TYPES[kind])
    check(kind, q, k, v, g, window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("Q,N,D,window,sinks,causal,buckets,reach", [
    (200, 200, 32, None, 0, True, 16, 60), (200, 200, 32, None, 0, False, 16, 60), (300, 300, 40, 50, 2, True, 8, 30),
    (300, 300, 33, 50, 70, False, 12, 90), (40, 260, 64, None, 0, True, 32, 1024), (260, 260, 128, 90, 1, False, 64, 700),
    (2, 2, 16, None, 0, True, 2, 5), (150, 150, 16, None, 0, False, 256, 1000),
])
def test_bias(cuda_device, kind, Q, N, D, window, sinks, causal, buckets, reach):
    q, k, v, g, bias = tensors(3, 2, Q, N, 4, 2, D, TYPES[kind], buckets)
    check(kind, q, k, v, g, window=window, sinks=sinks, causal=causal, bias=bias, max_distance=reach)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
def test_lengths(cuda_device, kind, causal, bits):
    """Clouds of no, one and any number of points, and lengths out of range;
    what lies behind a cloud's length is not even a number."""
    lengths = torch.tensor([0, 1, 150, 77, 64, -5, 10 ** 6, 128], dtype=bits)
    q, k, v, g, bias = tensors(4, 8, 150, 150, 2, 1, 24, TYPES[kind], 8)
    for b, n in enumerate(lengths.clamp(0, 150).tolist()):
        for t in (q, k, v, g):
            t[b, n:] = math.nan
    from mps_pointops.attention import window_attention

    how = dict(window=30, sinks=2, causal=causal, bias=bias, max_distance=20, lengths=lengths.cuda())
    check(kind, q, k, v, g, **how)
    out = window_attention(q, k, v, **how)
    assert all((out[b, n:] == 0).all() for b, n in enumerate(lengths.clamp(0, 150).tolist()))


@pytest.mark.parametrize("kind", TYPES)
def test_strides(cuda_device, kind):
    """Views of one packed projection, swapped dimensions, one head for the
    whole batch, rows that are not aligned, and a gradient that is one value."""
    from mps_pointops.attention import window_attention

    gen = torch.Generator(device="cuda").manual_seed(5)
    packed = torch.randn(2, 90, 8, 32, generator=gen, device="cuda").to(TYPES[kind])
    g = torch.randn(2, 90, 4, 32, generator=gen, device="cuda").to(TYPES[kind])
    check(kind, packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:], g, window=20)
    odd = torch.randn(2 * 90 * 8 * 32 + 1, generator=gen, device="cuda").to(TYPES[kind])[1:].view(2, 90, 8, 32)
    check(kind, odd[:, :, :4], odd[:, :, 4:6], odd[:, :, 6:], g, window=20)
    swapped = packed.transpose(1, 2).contiguous().transpose(1, 2)
    check(kind, swapped[:, :, :4], swapped[:, :, 4:6], swapped[:, :, 6:], g, window=20)
    shared = packed[:1, :, 4:6].expand(2, -1, -1, -1)
    check(kind, packed[:, :, :4], shared, packed[:, :, 6:], g, window=20)
    last = packed.transpose(2, 3).contiguous().transpose(2, 3)
    check(kind, last[:, :, :4], last[:, :, 4:6], last[:, :, 6:], g.transpose(1, 3).contiguous().transpose(1, 3), window=20)
    q = packed[:, :, :4].clone().requires_grad_()
    window_attention(q, packed[:, :, 4:6], packed[:, :, 6:]).sum().backward()
    one = torch.ones_like(q)
    q2 = q.detach().clone().requires_grad_()
    window_attention(q2, packed[:, :, 4:6], packed[:, :, 6:]).backward(one)
    assert torch.equal(q.grad, q2.grad)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_masked_places_reach_no_output(cuda_device, kind, value):
    """A key and a value that are no numbers, in the middle of the tiles of
    rows that do not see them."""
    from mps_pointops.attention import window_attention

    q, k, v, _, bias = tensors(6, 1, 200, 200, 2, 1, 40, TYPES[kind], 8)
    for window, sinks, causal in ((30, 2, True), (11, 0, False)):
        how = dict(window=window, sinks=sinks, causal=causal, bias=bias, max_distance=16)
        for where in (k, v):
            bad = where.clone()
            bad[0, 100, 0, 3] = value
            args = (q, bad, v) if where is k else (q, k, bad)
            out = window_attention(*args, **how).cpu().double()
            seen = visible(200, 200, window, sinks, causal, 200)[:, 100]
            want = definition(*args, None, **how)[0]
            close(out[:, ~seen], want[:, ~seen], LIMIT[kind])
            if where is v:
                assert not torch.isfinite(out[:, seen, :, 3]).any()
            assert torch.equal(torch.isfinite(out[:, seen]), torch.isfinite(want[:, seen])) or where is k


@pytest.mark.parametrize("kind", TYPES)
def test_bias_masks(cuda_device, kind):
    """Buckets of -inf (some, and all that a row sees) and of the type's lowest
    value (which every key of a row may have: then they share it)."""
    from mps_pointops.attention import window_attention

    q, k, v, g, bias = tensors(7, 1, 90, 90, 2, 2, 32, TYPES[kind], 8)
    bias[3:, 0] = -math.inf
    check(kind, q, k, v, g, causal=True, bias=bias, max_distance=16)
    bias[:, 1] = -math.inf
    out = window_attention(q, k, v, causal=True, bias=bias, max_distance=16)
    assert (out[:, :, 1] == 0).all()
    bias[:, 1] = torch.finfo(TYPES[kind]).min
    q[:, :, 1] = 0
    out = window_attention(q, k, v, causal=True, bias=bias, max_distance=16)
    mean = v[0, :, 1].double().cumsum(0) / torch.arange(1, 91, device="cuda")[:, None]
    close(out[0, :, 1], mean.cpu(), LIMIT[kind])


def test_gradients_against_differences(cuda_device):
    """Central differences of a weighted sum of the 32-bit outputs: with steps
    of 2^-6 their own error is about 2^-12 of the third derivative, and
    rounding 2^-24 times the sum over 2^-6."""
    from mps_pointops.attention import window_attention

    q, k, v, g, bias = tensors(8, 1, 40, 40, 2, 1, 8, torch.float32, 8)
    how = dict(window=12, sinks=2, causal=False, max_distance=9)
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    grads = torch.autograd.grad(window_attention(q, k, v, bias=bias, **how), leaves, g)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for n, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        way /= way.norm()
        values = []
        for sign in (1, -1):
            args = [t.detach() + (sign * 2.0 ** -6 * way if t is leaf else 0) for t in leaves]
            out = window_attention(*args[:3], bias=args[3], **how)
            values.append((out.double() * g.double()).sum().item())
        slope = (values[0] - values[1]) * 2.0 ** 5
        along = (grad.double() * way.double()).sum().item()
        assert abs(slope - along) <= 2e-3 * grad.norm().item(), (n, slope, along)


def test_streams(cuda_device):
    """The call is ordered on the current stream, forward and backward."""
    from mps_pointops.attention import window_attention

    q, k, v, g, _ = tensors(10, 2, 500, 500, 4, 2, 64, torch.bfloat16)
    want = window_attention(q, k, v, window=100)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-2
        late = q + 0 * big[0, 0].nan_to_num(0, 0, 0).to(q.dtype)
        leaf = late.requires_grad_()
        out = window_attention(leaf, k, v, window=100)
        grad, = torch.autograd.grad(out, [leaf], g)
    side.synchronize()
    assert torch.equal(out, want) and torch.isfinite(grad).all()


def test_empty(cuda_device):
    from mps_pointops.attention import window_attention

    for shape, keys in (((0, 4, 2, 8), (0, 4, 2, 8)), ((2, 0, 2, 8), (2, 5, 2, 8)), ((2, 3, 2, 8), (2, 0, 2, 8)),
                        ((2, 3, 0, 8), (2, 3, 0, 8))):
        q = torch.ones(shape, device="cuda", requires_grad=True)
        k = torch.ones(keys, device="cuda", requires_grad=True)
        v = torch.ones(keys, device="cuda", requires_grad=True)
        out = window_attention(q, k, v)
        assert out.shape == q.shape and (out == 0).all()
        for x in torch.autograd.grad(out.sum(), (q, k, v)):
            assert (x == 0).all()
