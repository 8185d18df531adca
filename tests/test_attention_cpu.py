"""Host-side checks of the attention operators that need no GPU: the buckets'
edges, refusals of the public calls, and the C ABI's before any launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from mps_pointops import _native, attention


def bucket(d: int, buckets: int, max_distance: int) -> int:
    """The definition, with exact comparisons: the largest t for which
    (d / e) ** (buckets - e) >= (max_distance / e) ** t."""
    e = buckets // 2
    if d < e:
        return d
    n, t = buckets - e, 0
    while t + 1 < n and d ** n >= max_distance ** (t + 1) * e ** (n - t - 1):
        t += 1
    return e + t


@pytest.mark.parametrize("buckets,max_distance", [(2, 2), (2, 1000), (3, 5), (16, 128), (32, 128), (20, 500), (7, 9), (64, 1024),
                                                  (256, 1024), (33, 40)])
def test_edges_are_the_buckets_first_distances(buckets, max_distance):
    edges = attention.bucket_edges(buckets, max_distance)
    assert len(edges) == buckets - 1 and list(edges) == sorted(edges)
    for d in list(range(0, max_distance + 3)) + [10 ** 6]:
        assert sum(e <= d for e in edges) == bucket(d, buckets, max_distance)


def test_edges_agree_with_the_logarithm():
    """Away from the steps themselves the formula in floating point gives the
    same buckets."""
    edges = attention.bucket_edges(32, 128)
    for d in range(16, 128):
        x = math.log(d / 16) / math.log(128 / 16) * 16
        if abs(x - round(x)) > 1e-9:
            assert sum(e <= d for e in edges) == 16 + int(x)


def test_edges_refusals():
    with pytest.raises(ValueError, match="at least 2"):
        attention.bucket_edges(1, 10)
    with pytest.raises(ValueError, match="max_distance"):
        attention.bucket_edges(16, 8)


def heads(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_window_attention_refusals():
    q, k = heads(2, 5, 4, 8), heads(2, 7, 2, 8)
    call = attention.window_attention
    for wrong, error, text in [
        ((q[0], k, k), ValueError, "shape"), ((q, k, k[:, :3]), ValueError, "same shape"),
        ((q, heads(1, 7, 2, 8), heads(1, 7, 2, 8)), ValueError, "batch"), ((q, heads(2, 7, 2, 9), heads(2, 7, 2, 9)), ValueError, "width"),
        ((q, heads(2, 7, 3, 8), heads(2, 7, 3, 8)), ValueError, "multiple"), ((q, heads(2, 7, 0, 8), heads(2, 7, 0, 8)), ValueError, "multiple"),
        ((q.double(), k.double(), k.double()), TypeError, "float32"), ((q, k.half(), k.half()), TypeError, "same type"),
        ((q, [1], k), TypeError, "tensors"), ((heads(1, 2, 1, 129),) * 3, ValueError, "128"), ((heads(1, 2, 1, 0),) * 3, ValueError, "128"),
    ]:
        with pytest.raises(error, match=text):
            call(*wrong)
    for how, error, text in [
        (dict(window=0), ValueError, "window"), (dict(sinks=-1), ValueError, "sinks"),
        (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError, "lengths"), (dict(lengths=torch.zeros(2)), TypeError, "lengths"),
        (dict(lengths=[1, 2]), TypeError, "lengths"), (dict(bias=torch.zeros(8, 4)), ValueError, "max_distance"),
        (dict(bias=torch.zeros(8, 3), max_distance=9), ValueError, "heads"), (dict(bias=torch.zeros(7, 4), max_distance=9), ValueError, "even"),
        (dict(bias=torch.zeros(8, 4).half(), max_distance=9), TypeError, "type"), (dict(bias=torch.zeros(8, 4), max_distance=1025), ValueError, "1024"),
        (dict(bias=torch.zeros(8, 4), max_distance=2), ValueError, "more than 2"), (dict(bias=torch.zeros(1, 4), max_distance=9, causal=True), ValueError, "at least 2"),
        (dict(bias=torch.zeros(514, 4), max_distance=900), ValueError, "256"), (dict(bias=3, max_distance=9), TypeError, "tensor"),
        (dict(), ValueError, "ROCm"),  # CPU tensors are not computed
    ]:
        with pytest.raises(error, match=text):
            call(q, k, k, **how)


def test_step_refusals():
    q, k = heads(2, 1, 4, 8), heads(2, 7, 2, 8)
    with pytest.raises(ValueError, match="lengths"):
        attention.window_attention_step(q, k, k, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="window"):
        attention.window_attention_step(q, k, k, window=0)
    with pytest.raises(ValueError, match="ROCm"):
        attention.window_attention_step(q, k, k)


def test_norm_refusals():
    q, k, angle, w = heads(2, 5, 4, 8), heads(2, 5, 2, 8), torch.zeros(5, 4), torch.ones(8)
    call = attention.qk_norm_rotate
    for args, error, text in [
        ((q, k[:, :4], w, w, angle, angle), ValueError, "tokens"), ((q, k, w[:7], w, angle, angle), ValueError, "q_weight"),
        ((q, k, w, w.double(), angle, angle), TypeError, "k_weight"), ((q, k.half(), w, w, angle, angle), TypeError, "same type"),
        ((q, k, w, w, angle.half(), angle.half()), TypeError, "float32"), ((q, k, w, w, angle, angle[:4]), ValueError, "cos and sin"),
        ((q, k, w, w, angle[:4], angle[:4]), ValueError, "cos and sin"), ((q, k, w, w, torch.zeros(5, 5), torch.zeros(5, 5)), ValueError, "half"),
        ((q, k, w, w, None, angle), TypeError, "tensors"), ((q, k, 1.0, w, angle, angle), TypeError, "q_weight"),
        ((q.half(), k.half(), w, w.half(), angle, angle), TypeError, "same type"),
        ((q, k, w, w, angle.clone().requires_grad_(), angle), ValueError, "detach"), ((q, k, w, w, angle, angle), ValueError, "ROCm"),
    ]:
        with pytest.raises(error, match=text):
            call(*args)


def test_relative_bias_refusals():
    call = attention.relative_bias
    for args, how, error, text in [
        ((torch.zeros(8), 3, 3), dict(max_distance=9), ValueError, "shape"), ((torch.zeros(8, 2).double(), 3, 3), dict(max_distance=9), TypeError, "float32"),
        ((torch.zeros(8, 2), -1, 3), dict(max_distance=9), ValueError, "non-negative"), ((torch.zeros(8, 2), 3, 1 << 22), dict(max_distance=9), ValueError, "at most"),
        ((torch.zeros(9, 2), 3, 3), dict(max_distance=9), ValueError, "even"), ((3, 3, 3), dict(max_distance=9), TypeError, "tensor"),
        ((torch.zeros(8, 2), 3, 3), dict(max_distance=9), ValueError, "ROCm"),
    ]:
        with pytest.raises(error, match=text):
            call(*args, **how)


def packed(**change):
    """A pointops_attention with no tensors, changed field by field."""
    fields = dict(q=0, k=0, v=0, bias=0, lengths=0, edges=0, s0=0, s1=0, s2=0, s3=0, s4=0, s5=0, s6=0, s7=0, s8=0,
                  B=1, Q=4, N=4, H=2, G=1, D=8, window=2, sinks=0, n_edges=0, buckets=0, bits=0, causal=1, type=0, scale=1.0)
    assert set(change) <= set(fields)
    return attention._ARGS.pack(*{**fields, **change}.values())


def test_capi_rejects_bad_attention_arguments_before_any_launch():
    lib = _native.library()
    edges = (ctypes.c_int32 * 2)(1, 2)
    falling = (ctypes.c_int32 * 2)(2, 1)
    far = (ctypes.c_int32 * 2)(1, 2000)
    address = ctypes.addressof
    forward, step = lib.pointops_attention_forward, lib.pointops_attention_step
    for bad in (dict(B=-1), dict(D=0), dict(D=129), dict(H=3, G=2), dict(G=0), dict(window=0), dict(sinks=-1), dict(type=3),
                dict(Q=1 << 30), dict(lengths=8, bits=16), dict(bias=8, n_edges=2, buckets=3),
                dict(bias=8, edges=address(edges), n_edges=0, buckets=1), dict(bias=8, edges=address(edges), n_edges=2, buckets=4),
                dict(bias=8, edges=address(falling), n_edges=2, buckets=3), dict(bias=8, edges=address(far), n_edges=2, buckets=3)):
        assert forward(packed(**bad), 8, None, None) == 1, bad
        assert step(packed(**bad), 8, None, None) == 1, bad
    assert forward(packed(), 8, None, None) == 1  # tensors that are not there
    assert forward(None, 8, None, None) == 1
    assert step(packed(q=8, k=8, v=8, causal=0), 8, None, None) == 1
    for none in (dict(B=0), dict(H=0, G=0), dict(Q=0)):
        assert forward(packed(**none), None, None, None) == 0, none
        assert step(packed(**none), None, None, None) == 0, none
    backward = lib.pointops_attention_backward
    assert backward(packed(), *[None] * 10) == 1
    assert backward(packed(B=0), *[None] * 10) == 0
    assert lib.pointops_attention_backward_workspace_bytes(packed(D=0)) == 0
    assert lib.pointops_attention_backward_workspace_bytes(packed()) >= 4 * 2 * 4


def test_capi_rejects_bad_norm_and_bias_arguments_before_any_launch():
    lib = _native.library()

    def norm(**change):
        fields = dict(q=0, k=0, wq=0, wk=0, cos=0, sin=0, s0=0, s1=0, s2=0, s3=0, s4=0, s5=0, a0=0, a1=0,
                      B=1, N=4, H=2, G=1, D=8, R=4, type=0, weight=0, eps=1e-6)
        return attention._NORM_ARGS.pack(*{**fields, **change}.values())

    call = lib.pointops_qk_norm_rotate
    for bad in (dict(D=0), dict(D=129), dict(R=3), dict(R=10), dict(R=-2), dict(type=5), dict(type=1, weight=2), dict(B=-1), dict()):
        assert call(norm(**bad), 8, 8, None) == 1, bad
    assert call(norm(B=0), None, None, None) == 0
    edges = (ctypes.c_int32 * 1)(1)
    bias = lib.pointops_relative_bias
    assert bias(8, None, 1, 2, 0, 8, 1, 4, 4, None) == 1
    assert bias(8, edges, 1, 3, 0, 8, 1, 4, 4, None) == 1
    assert bias(8, edges, 1, 2, 7, 8, 1, 4, 4, None) == 1
    assert bias(8, edges, 1, 2, 0, 8, 1, 1 << 22, 4, None) == 1
    assert bias(None, edges, 1, 2, 0, None, 1, 4, 4, None) == 1
    assert bias(None, edges, 1, 2, 0, None, 1, 0, 4, None) == 0
