"""More host-side checks of the attention operators that need no GPU."""

from __future__ import annotations

import ctypes

from mps_pointops import _native

from test_attention_cpu import packed


def test_backward_needs_its_workspace_where_queries_are_none():
    """The bias's parts lie in it for keys that no query meets."""
    edges = (ctypes.c_int32 * 2)(1, 2)
    args = packed(Q=0, k=8, v=8, bias=8, edges=ctypes.addressof(edges), n_edges=2, buckets=3)
    lib = _native.library()
    assert lib.pointops_attention_backward_workspace_bytes(args) > 0
    assert lib.pointops_attention_backward(args, None, None, None, None, None, 8, 8, 8, None, None) == 1
