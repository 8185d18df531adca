"""A cache in 8 and 4 bits, written and read back, against its definition in 64
bits: a search among the type's values.  Quotients by powers of two and the
values themselves are exact, so all comparisons are of equal values."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def values_of(bits):
    if bits == 4:
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    below = [m * 2.0 ** -9 for m in range(8)]
    return torch.tensor(below + [2.0 ** e * (1 + m / 8) for e in range(-6, 9) for m in range(8)][:-1], dtype=torch.float64)


def held(x, bits):
    """(..., D) values as the cache holds them, and the scales' exponents (128: a
    group with an infinity or NaN)."""
    x = x.detach().cpu().double()
    table = values_of(bits)
    middle = (table[1:] + table[:-1]) / 2
    out, scales = torch.empty_like(x), []
    for first in range(0, x.shape[-1], 32):
        group = x[..., first:first + 32]
        most = group.abs().amax(-1)
        good = torch.isfinite(group).all(-1)
        power = torch.full(most.shape, -127, dtype=torch.int64)
        for p in range(-127, 128):  # the smallest that holds the largest
            power = torch.where((power == p) & (most > table[-1] * 2.0 ** p), p + 1, power)
        part = (group / torch.pow(2.0, power.double())[..., None]).abs().contiguous()
        code = torch.searchsorted(middle, part)
        tie = part == middle[code.clamp(max=len(middle) - 1)]
        code = (code + (tie & (code % 2 == 1))).clamp(max=len(table) - 1)
        y = torch.copysign(table[code], group) * torch.pow(2.0, power.double())[..., None]
        out[..., first:first + 32] = torch.where(good[..., None], y, math.nan)
        scales.append(torch.where(good, power, 128))
    return out, torch.stack(scales, -1)


def same(got, want):
    got, want = got.cpu().double(), want.cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def make(seed, *shape, dtype=torch.float32, spread=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda")
    return (x * torch.exp(spread * torch.randn(shape[-2:], generator=gen, device="cuda"))).to(dtype)


def new_cache(B, N, G, D, bits):
    from mps_pointops.attention import QuantizedCache

    return QuantizedCache(B, N, G, D, bits=bits)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("B,N,G,D", [(1, 1, 1, 1), (2, 5, 3, 20), (3, 70, 2, 32), (1, 300, 1, 33), (2, 33, 4, 64),
                                     (2, 65, 1, 96), (2, 40, 3, 100), (1, 1000, 2, 128), (70, 1, 8, 40)])
def test_write_and_read(cuda_device, kind, bits, B, N, G, D):
    from mps_pointops.attention import cache_read, cache_write

    print(kind, bits, B, N, G, D, flush=True)
    k, v = make(1, B, N, G, D, dtype=TYPES[kind]), make(2, B, N, G, D, dtype=TYPES[kind])
    cache = new_cache(B, N, G, D, bits)
    cache_write(cache, k, v)
    for out in TYPES.values():
        got = cache_read(cache, dtype=out)
        for t, x, scales in zip(got, (k, v), (cache.k_scales, cache.v_scales)):
            want, power = held(x, bits)
            assert t.dtype == out and t.is_contiguous()
            same(t, want.to(out))
            assert torch.equal(scales.cpu().transpose(1, 2).long() - 127, power)


@pytest.mark.parametrize("bits", [8, 4])
def test_every_code_boundary(cuda_device, bits):
    """Each value of the type, the midpoints and their neighbours, under scales
    from the smallest to the largest, with the group's largest value beside them."""
    from mps_pointops.attention import cache_read, cache_write

    table = values_of(bits).float()
    middle = (table[1:] + table[:-1]) / 2
    points = torch.cat([table, middle, torch.nextafter(middle, middle + 1), torch.nextafter(middle, middle - 1)])
    points = torch.cat([points, -points])
    points = torch.nn.functional.pad(points, (0, -len(points) % 31)).view(-1, 31)
    points = torch.cat([points, torch.full((len(points), 1), float(table[-1]))], 1)
    rows = torch.stack([points * 2.0 ** p for p in (0, -126, -100, -3, 1, 60, 119)]).view(1, -1, 1, 32).cuda()
    cache = new_cache(1, rows.shape[1], 1, 32, bits)
    cache_write(cache, rows, -rows)
    want, _ = held(rows, bits)
    k, v = cache_read(cache, dtype=torch.float32)
    same(k, want.float())
    same(v, -want.float())


@pytest.mark.parametrize("bits", [8, 4])
def test_scales_at_their_borders(cuda_device, bits):
    """Largest magnitudes of M 2^x and their neighbours, zeros, subnormal numbers,
    the largest number, infinities and NaN of either sign."""
    from mps_pointops.attention import cache_read, cache_write

    top = 448.0 if bits == 8 else 6.0
    rows = []
    for p in range(-127, 120, 13):
        edge = torch.tensor(top * 2.0 ** p)
        rows += [edge, torch.nextafter(edge, edge * 2), torch.nextafter(edge, edge / 2)]
    rows += [torch.tensor(x) for x in (0.0, -0.0, 1e-45, -3e-42, 1.1754942e-38, 1.17549435e-38, 3.4028235e38, -3.4028235e38,
                                       math.inf, -math.inf, math.nan, -math.nan)]
    x = torch.zeros(1, len(rows), 2, 40)
    x[0, :, 0, 3] = torch.stack(rows)
    x[0, :, 0, 4] = torch.stack(rows) / 3
    x[0, :, 1, 39] = torch.stack(rows)  # the short group
    x = x.cuda()
    cache = new_cache(1, len(rows), 2, 40, bits)
    cache_write(cache, x, x)
    want, power = held(x, bits)
    k, v = cache_read(cache, dtype=torch.float32)
    same(k, want.float())
    same(v, want.float())
    assert torch.equal(cache.v_scales.cpu().transpose(1, 2).long() - 127, power)


@pytest.mark.parametrize("kind", TYPES)
def test_strides(cuda_device, kind):
    """Slices of one projection's output, heads before tokens, unaligned rows and a
    last dimension that is not contiguous."""
    from mps_pointops.attention import cache_read, cache_write

    packed = make(3, 2, 50, 9, 48, dtype=TYPES[kind])
    flat = make(4, 1, 1, 1, 2 * 50 * 3 * 48 + 1, dtype=TYPES[kind]).flatten()
    for k, v in [(packed[:, :, 1:4], packed[:, :, 5:8]), (packed.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :3], packed[:, :, :3]),
                 (flat[1:].view(2, 50, 3, 48), flat[:-1].view(2, 50, 3, 48)), (packed.transpose(2, 3).contiguous().transpose(2, 3)[:, :, :3], packed[:, :, :3]),
                 (packed[:1, :, :3].expand(2, -1, -1, -1), packed[:, :1, :3].expand(-1, 50, -1, -1))]:
        cache = new_cache(2, 50, 3, 48, 8)
        cache_write(cache, k, v)
        got = cache_read(cache, dtype=torch.float32)
        same(got[0], held(k, 8)[0].float())
        same(got[1], held(v, 8)[0].float())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lengths_type,starts_type", [(torch.int32, torch.int64), (torch.int64, torch.int32)])
def test_places(cuda_device, bits, lengths_type, starts_type):
    """Tokens at the end of lengths and from starts on, out of range on either
    side; what is not written stays, also behind a padded prompt."""
    from mps_pointops.attention import cache_read, cache_write

    B, N, T, G, D = 8, 30, 7, 2, 36
    lengths = torch.tensor([0, 1, 7, 8, 30, 29, -5, 10 ** 6], dtype=lengths_type, device="cuda")
    starts = torch.tensor([0, 0, 3, -4, 25, 40, -(2 ** 31), 2 ** 31 - 1], dtype=starts_type, device="cuda")
    old, new = make(5, B, N, G, D), make(6, B, T, G, D)
    for where in (None, starts):
        cache = new_cache(B, N, G, D, bits)
        cache_write(cache, old, -old)
        cache_write(cache, new, -new, lengths, starts=where)
        want = held(old, bits)[0]
        fresh = held(new, bits)[0]
        for b in range(B):
            end = min(max(int(lengths[b]), 0), N)
            start = end - T if where is None else int(starts[b])
            for t in range(T):
                if 0 <= start + t < end:
                    want[b, start + t] = fresh[b, t]
        k, v = cache_read(cache, dtype=torch.float32)
        same(k, want.float())
        same(v, -want.float())


def test_far_starts(cuda_device):
    from mps_pointops.attention import cache_read, cache_write

    cache = new_cache(2, 4, 1, 8, 8)
    x = torch.ones(2, 3, 1, 8, device="cuda")
    cache_write(cache, x, x, starts=torch.tensor([-2 ** 63, 2 ** 63 - 1], device="cuda"))
    assert not cache_read(cache)[0].any()


def test_views(cuda_device):
    """The first positions and one cloud share the cache's memory."""
    from mps_pointops.attention import cache_read, cache_write

    x = make(7, 3, 20, 2, 72)
    cache = new_cache(3, 20, 2, 72, 4)
    cache_write(cache.positions(0, 5), x[:, :5], x[:, 5:10])
    cache_write(cache.cloud(1).positions(0, 9), x[1:2, 11:], x[1:2, 2:11])
    want = torch.zeros(2, 3, 20, 2, 72, dtype=torch.float64)
    want[0, :, :5], want[1, :, :5] = held(x[:, :5], 4)[0], held(x[:, 5:10], 4)[0]
    want[0, 1, :9], want[1, 1, :9] = held(x[1, 11:], 4)[0], held(x[1, 2:11], 4)[0]
    for part, cut in ((cache, want), (cache.positions(3, 7), want[:, :, 3:7]), (cache.cloud(2), want[:, 2:3]), (cache.positions(20, 20), want[:, :, :0]),
                      (cache.cloud(1).positions(0, 9), want[:, 1:2, :9])):
        k, v = cache_read(part, dtype=torch.float32)
        same(k, cut[0].float())
        same(v, cut[1].float())


def test_offsets_beyond_32_bits(cuda_device):
    from mps_pointops.attention import cache_read, cache_write

    N = (1 << 25) + 9
    cache = new_cache(1, N, 1, 128, 8)  # 2^32 bytes of codes and more
    x = make(8, 1, 70, 1, 128, dtype=torch.bfloat16)
    cache_write(cache, x, x)
    tail = cache.positions(N - 70, N)
    k, v = cache_read(tail, dtype=torch.float32)
    same(k, held(x, 8)[0].float())
    same(v, held(x, 8)[0].float())
    k, _ = cache_read(cache, dtype=torch.bfloat16)  # 2^33 bytes
    same(k[:, -70:], held(x, 8)[0])
    assert not k[:, :-70].any()


def test_replays_in_a_graph(cuda_device):
    """A write and a read, captured once and replayed with other tokens and places."""
    from mps_pointops.attention import cache_read, cache_write

    x, lengths = make(9, 2, 1, 2, 64, dtype=torch.bfloat16), torch.tensor([4, 9], device="cuda")
    cache, eager = new_cache(2, 12, 2, 64, 8), new_cache(2, 12, 2, 64, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_write(cache, x, x, lengths)
        cache_read(cache)
    torch.cuda.current_stream().wait_stream(side)
    cache_write(eager, x, x, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_write(cache, x, x, lengths)
        out = cache_read(cache)
    for n in (1, 5, 12, 3):
        lengths.fill_(n)
        x.normal_()
        graph.replay()
        cache_write(eager, x, x, lengths)
        for a, b in zip(out, cache_read(eager)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
