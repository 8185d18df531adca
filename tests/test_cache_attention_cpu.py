"""Host-side checks of the quantised cache and the steps over kept keys that need
no GPU: refusals of the public calls, the C ABI's before any launch, layouts."""

from __future__ import annotations

import copy
import ctypes
import pickle
import struct

import pytest
import torch
from torch.autograd import forward_ad

from mps_pointops import _native, attention
from mps_pointops.attention import QuantizedCache


def rows(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def cache(batch=2, tokens=7, heads=2, width=8, bits=8):
    return QuantizedCache(batch, tokens, heads, width, bits=bits, device="cpu")


@pytest.mark.parametrize("width,bits,row,groups", [(1, 8, 32, 1), (32, 8, 32, 1), (33, 8, 64, 2), (128, 8, 128, 4), (8, 4, 16, 1), (96, 4, 48, 3), (100, 4, 64, 4)])
def test_layout(width, bits, row, groups):
    c = cache(3, 5, 2, width, bits)
    assert c.k_codes.shape == c.v_codes.shape == (3, 2, 5, row)
    assert c.k_scales.shape == c.v_scales.shape == (3, 2, 5, groups)
    assert not c.k_codes.any() and not c.v_scales.any()
    assert (c.batch, c.tokens, c.heads, c.width, c.bits, c.device.type) == (3, 5, 2, width, bits, "cpu")
    part = c.cloud(2).positions(0, 4)
    assert (part.batch, part.tokens, part.heads, part.width, part.bits) == (1, 4, 2, width, bits)
    part.k_codes.fill_(9)
    assert (c.k_codes[2, :, :4] == 9).all() and not c.k_codes[:2].any() and not c.k_codes[2, :, 4].any()
    assert c.positions(2, 5).k_codes.data_ptr() == c.k_codes.data_ptr() + 2 * row and c.positions(5, 5).tokens == 0
    assert "bits=%d" % bits in repr(part)


@pytest.mark.parametrize("bits", [8, 4])
def test_copies(bits):
    """Of a cache and of a part, by copy and by pickle, in memory of their own."""
    c = cache(3, 5, 2, 40, bits)
    c.k_codes.random_(0, 100)
    c.v_scales.random_(0, 100)
    for part in (c, c.cloud(1), c.positions(2, 4)):
        for new in (copy.deepcopy(part), pickle.loads(pickle.dumps(part))):
            assert (new.batch, new.tokens, new.heads, new.width, new.bits) == (part.batch, part.tokens, part.heads, 40, bits)
            for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
                assert torch.equal(getattr(new, name), getattr(part, name))
                assert getattr(new, name).data_ptr() != getattr(part, name).data_ptr()
            with pytest.raises(ValueError, match="ROCm"):  # the next check
                attention.cache_read(new)


def test_cache_refusals():
    for args, how, text in [((1, 1, 1, 0), {}, "128"), ((1, 1, 1, 129), {}, "128"), ((-1, 1, 1, 8), {}, "sizes"), ((1, 1 << 30, 0, 8), {}, "sizes"),
                            ((1, 1, 1, 8), dict(bits=5), "bits")]:
        with pytest.raises(ValueError, match=text):
            QuantizedCache(*args, device="cpu", **how)
    for wrong in (lambda c: c.positions(0, 8), lambda c: c.positions(-1, 2), lambda c: c.positions(3, 2), lambda c: c.cloud(2), lambda c: c.cloud(-1)):
        with pytest.raises(ValueError, match="there are"):
            wrong(cache())
    c = cache()
    for name in ("k_codes", "v_scales", "width", "other"):
        with pytest.raises(AttributeError, match="stays"):
            setattr(c, name, 3)
    c.v_codes.set_(torch.zeros(1, dtype=torch.uint8))  # memory that a call would read past
    for call in (lambda: attention.cache_write(c, rows(2, 3, 2, 8), rows(2, 3, 2, 8)), lambda: attention.cache_read(c),
                 lambda: attention.quantized_attention_step(rows(2, 1, 4, 8), c)):
        with pytest.raises(ValueError, match="memory"):
            call()


def test_write_refusals():
    k = rows(2, 3, 2, 8)
    call = attention.cache_write
    for args, how, error, text in [
        ((3, k, k), {}, TypeError, "QuantizedCache"), ((cache(), k, k[:, :2]), {}, ValueError, "same shape"), ((cache(), k[0], k[0]), {}, ValueError, "shape"),
        ((cache(), k, k.half()), {}, TypeError, "same type"), ((cache(), k.double(), k.double()), {}, TypeError, "float32"), ((cache(), [1], k), {}, TypeError, "tensors"),
        ((cache(3), k, k), {}, ValueError, "batch"), ((cache(heads=1), k, k), {}, ValueError, "heads"), ((cache(width=9), k, k), {}, ValueError, "width"),
        ((cache(), k, k, torch.zeros(2)), {}, TypeError, "lengths must be int32"), ((cache(), k, k, torch.zeros(3, dtype=torch.int64)), {}, ValueError, "lengths"),
        ((cache(), k, k, 5), {}, TypeError, "lengths"), ((cache(), k, k), dict(starts=[0, 0]), TypeError, "starts"), ((cache(), k, k), dict(starts=torch.zeros(2)), TypeError, "starts"),
        ((cache(), k, k), {}, ValueError, "ROCm"),  # CPU tensors are not computed
    ]:
        with pytest.raises(error, match=text):
            call(*args, **how)


def test_read_refusals():
    for args, how, error, text in [((rows(2),), {}, TypeError, "QuantizedCache"), ((cache(),), dict(dtype=torch.float64), TypeError, "float32"), ((cache(),), {}, ValueError, "ROCm")]:
        with pytest.raises(error, match=text):
            attention.cache_read(*args, **how)


def test_quantized_step_refusals(monkeypatch):
    monkeypatch.setattr(_native, "require_device", lambda device: 0)
    q = rows(2, 1, 4, 8)
    call = attention.quantized_attention_step
    for args, how, error, text in [
        ((q[0], cache()), {}, ValueError, "shape"), ((q, rows(2)), {}, TypeError, "QuantizedCache"), ((q.double(), cache()), {}, TypeError, "float32"),
        ((q, cache(3)), {}, ValueError, "batch"), ((q, cache(width=9)), {}, ValueError, "width"), ((q, cache(heads=3)), {}, ValueError, "multiple"),
        ((q, cache(heads=0)), {}, ValueError, "multiple"), ((q, cache()), dict(window=0), ValueError, "window"), ((q, cache()), dict(sinks=-1), ValueError, "sinks"),
        ((q, cache(), torch.zeros(2)), {}, TypeError, "lengths"), ((q, cache(), torch.zeros(1, dtype=torch.int32)), {}, ValueError, "lengths"),
        ((q, cache()), dict(bias=rows(8, 4)), ValueError, "max_distance"), ((q, cache()), dict(bias=rows(8, 3), max_distance=9), ValueError, "heads"),
        ((q, cache()), dict(bias=rows(8, 4).half(), max_distance=9), TypeError, "type"), ((q, cache()), dict(bias=rows(8, 4), max_distance=1025), ValueError, "1024"),
        ((q, cache()), dict(bias=3, max_distance=9), TypeError, "tensor"),
    ]:
        with pytest.raises(error, match=text):
            call(*args, **how)
    with pytest.raises(ValueError, match="gradients"):
        call(q.requires_grad_(), cache())
    with pytest.raises(ValueError, match="gradients"):
        call(rows(2, 1, 4, 8), cache(), bias=rows(8, 4).requires_grad_(), max_distance=9)


def test_prefix_step_refusals(monkeypatch):
    monkeypatch.setattr(_native, "require_device", lambda device: 0)
    q, p, k = rows(2, 1, 4, 8), rows(5, 2, 8), rows(2, 7, 2, 8)
    call = attention.prefix_attention_step
    for args, error, text in [
        ((q, (p, p), cache()), TypeError, "both"), ((q, cache(1), (k, k)), TypeError, "both"), ((q, cache(2), cache(2)), ValueError, "batch of 1"),
        ((q, cache(1, bits=4), cache(2)), ValueError, "bits"), ((q, cache(1, heads=4), cache(2)), ValueError, "heads"), ((q, cache(1, width=9), cache(2)), ValueError, "width"),
        ((q, p, (k, k)), TypeError, "pair"), ((q, (p, p), k), TypeError, "pair"), ((q, (p, 3), (k, k)), TypeError, "pair"), ((q, (p, p), (k, k, k)), TypeError, "pair"),
        ((q, (k, k), (k, k)), ValueError, "tokens, heads, width"), ((q, (p, p[:4]), (k, k)), ValueError, "same shape"), ((q, (p, p), (k, k[:, :4])), ValueError, "same shape"),
        ((q, (p.half(), p.half()), (k, k)), TypeError, "same type"), ((q, (p, p), (k[:1], k[:1])), ValueError, "batch"), ((q, (p[:, :1], p[:, :1]), (k, k)), ValueError, "heads"),
        ((q, (p[..., :7], p[..., :7]), (k, k)), ValueError, "width"), ((rows(2, 1, 4, 129), (rows(5, 2, 129),) * 2, (rows(2, 7, 2, 129),) * 2), ValueError, "128"),
        ((rows(2, 1, 5, 8), (p, p), (k, k)), ValueError, "multiple"),
    ]:
        with pytest.raises(error, match=text):
            call(*args)
    for which in range(5):
        tensors = [q.clone(), p.clone(), p.clone(), k.clone(), k.clone()]
        tensors[which].requires_grad_()
        with pytest.raises(ValueError, match="gradients"):
            call(tensors[0], tensors[1:3], tensors[3:])


CALLS = {
    "cache_write": lambda k: attention.cache_write(cache(tokens=3), k, k),
    "quantized_attention_step": lambda q: attention.quantized_attention_step(q, cache()),
    "prefix_attention_step": lambda q: attention.prefix_attention_step(q, (q[0], q[0]), (q, q)),
}


@pytest.mark.parametrize("name", CALLS)
def test_what_does_not_see_memory_is_refused(monkeypatch, name):
    """Traces, tangents and function transforms, before anything is launched."""
    monkeypatch.setattr(_native, "require_device", lambda device: 0)
    monkeypatch.setattr(_native, "call", None)
    x = rows(2, 3, 2, 8)
    with pytest.raises(RuntimeError, match=name):
        torch.jit.trace(CALLS[name], (x,), check_trace=False)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match=name):
        CALLS[name](forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError):
        torch.vmap(CALLS[name])(x[None])


# pointops_cache, pointops_keys and pointops_cache_attention
def packed_cache(k=16, v=16, ks=16, vs=16, strides=(14, 7), B=2, N=7, G=2, D=8, bits=8):
    return struct.pack("@4Q6qi4x", k, v, ks, vs, *strides, B, N, G, D, bits)


def packed_keys(k=16, v=16, ks=0, vs=0, strides=(112, 16, 8), N=7):
    return struct.pack("@4Q7q", k, v, ks, vs, *strides, *strides, N)


def packed(q=16, start=None, own=None, bias=0, lengths=0, edges=0, B=2, Q=1, H=4, G=2, D=8, window=9, sinks=0, n_edges=0, buckets=0, length_bits=0, type=0, bits=0):
    start = packed_keys(N=0) if start is None else start
    own = packed_keys() if own is None else own
    return struct.pack("@Q88s88s3Q3q5q2q5if", q, start, own, bias, lengths, edges, 32, 32, 8, B, Q, H, G, D, window, sinks, n_edges, buckets, length_bits, type, bits, 1.0)


def test_c_cache_refusals():
    lib = _native.library()
    three = (ctypes.c_int64 * 3)(48, 16, 8)

    def write(c=packed_cache(), k=16, tokens=3, lengths=None, length_bits=0, starts=None, start_bits=0, type=0, stride=three):
        return lib.pointops_cache_write(c, k, stride, k, stride, tokens, lengths, length_bits, starts, start_bits, type, None)

    for status in (write(None), write(packed_cache(bits=3)), write(packed_cache(D=0)), write(packed_cache(D=129)), write(packed_cache(N=-1)), write(packed_cache(k=0)),
                   write(packed_cache(vs=0)), write(packed_cache(v=24)), write(k=None), write(tokens=-1), write(type=3), write(lengths=16, length_bits=16), write(starts=16), write(stride=None),
                   write(packed_cache(D=128, ks=18)), write(packed_cache(D=64, vs=17)), write(packed_cache(B=1 << 29, G=1 << 29)), write(packed_cache(N=1 << 30))):
        assert status == 1
    for status in (write(tokens=0), write(packed_cache(B=0)), write(packed_cache(N=0, k=0, v=0, ks=0, vs=0)), write(packed_cache(G=0))):
        assert status == 0  # nothing to do

    def read(c=packed_cache(), k=16, v=16, type=0):
        return lib.pointops_cache_read(c, k, v, type, None)

    for status in (read(None), read(k=None), read(v=None), read(type=-1), read(packed_cache(bits=16)), read(packed_cache(k=8))):
        assert status == 1
    assert read(packed_cache(B=0), None, None) == read(packed_cache(N=0), None, None) == 0


def test_c_step_refusals():
    lib = _native.library()

    def step(args=packed(), out=16, workspace=16):
        return lib.pointops_cache_attention_step(args, out, workspace, None)

    coded = packed_keys(ks=16, vs=16)
    edges = (ctypes.c_int32 * 2)(1, 2)
    for args in (None, packed(D=0), packed(D=129), packed(H=5), packed(G=0), packed(window=0), packed(sinks=-1), packed(lengths=16, length_bits=8), packed(type=3),
                 packed(bits=5), packed(B=-1), packed(q=0), packed(own=packed_keys(k=0)), packed(own=packed_keys(v=0)), packed(start=packed_keys(N=-1)),
                 packed(start=packed_keys(k=0)), packed(bits=8), packed(bits=8, own=packed_keys(k=24, ks=16, vs=16)), packed(bits=8, own=packed_keys(ks=16)),
                 packed(bits=8, start=packed_keys(v=8, ks=16, vs=16), own=coded), packed(bias=16, edges=0), packed(bias=16, edges=ctypes.addressof(edges), n_edges=2, buckets=6),
                 packed(bits=4, D=128, own=packed_keys(ks=18, vs=16)), packed(bits=4, D=64, own=packed_keys(ks=16, vs=17)),
                 packed(own=packed_keys(N=1 << 30)), packed(own=packed_keys(N=1 << 29), start=packed_keys(N=1 << 29)), packed(B=1 << 28, Q=8)):
        assert step(args) == 1, args
    assert lib.pointops_cache_attention_step_workspace_bytes(None) == 0
    assert step(out=None) == 1
    parts = packed(start=packed_keys(N=100000), window=1 << 20)
    assert lib.pointops_cache_attention_step_workspace_bytes(parts) > 0 and step(parts, workspace=None) == 1
    long = packed(bits=8, window=1 << 20, own=packed_keys(ks=16, vs=16, N=100000))
    assert lib.pointops_cache_attention_step_workspace_bytes(long) > 0 and step(long, workspace=None) == 1
    for args in (packed(B=0), packed(Q=0), packed(H=0, G=0)):
        assert step(args) == 0 and lib.pointops_cache_attention_step_workspace_bytes(args) == 0
