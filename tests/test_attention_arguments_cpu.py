"""More host-side checks of the attention operators that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mps_pointops import _native, attention

from test_attention_cpu import packed


def test_backward_needs_its_workspace_where_queries_are_none():
    """The bias's parts lie in it for keys that no query meets."""
    edges = (ctypes.c_int32 * 2)(1, 2)
    args = packed(Q=0, k=8, v=8, bias=8, edges=ctypes.addressof(edges), n_edges=2, buckets=3)
    lib = _native.library()
    assert lib.pointops_attention_backward_workspace_bytes(args) > 0
    assert lib.pointops_attention_backward(args, None, None, None, None, None, 8, 8, 8, None, None) == 1


@pytest.mark.timeout(60)
@pytest.mark.parametrize("buckets,max_distance", [(256, 1 << 30), (128, 1 << 30), (255, 1 << 20), (2, 1 << 30), (3, 2), (256, 129),
                                                  (17, 10 ** 9 + 7), (64, 33)])
def test_edges_of_large_distances(buckets, max_distance):
    """Each edge against its definition in whole numbers: the least d with
    (d / e) ** (buckets - e) >= (max_distance / e) ** t."""
    edges = attention.bucket_edges(buckets, max_distance)
    e = buckets // 2
    steps = buckets - e
    assert edges[:e] == tuple(range(1, e + 1)) and len(edges) == buckets - 1
    for t, d in enumerate(edges[e:], 1):
        assert d ** steps >= max_distance ** t * e ** (steps - t) > (d - 1) ** steps


def test_largest_dense_bias():
    """The sizes that the launches hold, and one more of each."""
    table = torch.zeros(8, 2)
    for queries, keys in ((4194240, 3), (3, 4194303)):
        with pytest.raises(ValueError, match="ROCm"):  # the next check
            attention.relative_bias(table, queries, keys, max_distance=9)
    for queries, keys in ((4194241, 3), (4194303, 3), (3, 4194304)):
        with pytest.raises(ValueError, match="at most"):
            attention.relative_bias(table, queries, keys, max_distance=9)
    lib = _native.library()
    edges = (ctypes.c_int32 * 1)(1)
    for Q, N in ((4194241, 4), (4, 1 << 22)):
        assert lib.pointops_relative_bias(8, edges, 1, 2, 0, 8, 0, Q, N, None) == 1
        assert lib.pointops_relative_bias_backward(8, 1, 1, edges, 1, 2, 0, 8, 8, 0, Q, N, None) == 1
        assert lib.pointops_relative_bias_backward_workspace_bytes(1, Q, N, 2) == 0
    assert lib.pointops_relative_bias(8, edges, 1, 2, 0, 8, 0, 4194240, 4, None) == 0  # without heads: nothing to do
