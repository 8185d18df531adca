"""What a step over kept keys asks for as its workspace, by the C ABI, without a GPU."""

from __future__ import annotations

import pytest

from mps_pointops import _native
from test_cache_attention_cpu import packed, packed_keys


@pytest.mark.parametrize("bits,type", [(0, 0), (0, 2), (8, 2), (4, 1)])
@pytest.mark.parametrize("B,H,G", [(512, 32, 32), (700, 8, 4), (64, 64, 2), (3, 2, 2)])
def test_parts_hold_the_rows_that_there_are(bits, type, B, H, G):
    """Rows behind a start have a part of it and one of their own each, of D values and four more (a
    sequence of one row took room for 16); the start's, and of few rows the caches', are cut to fill the card."""
    D, start, own = 128, 5000, 40
    scales = dict(ks=16, vs=16) if bits else {}
    call = packed(B=B, Q=1, H=H, G=G, D=D, type=type, bits=bits, window=1 << 20, start=packed_keys(N=start, **scales), own=packed_keys(N=own, **scales))
    size = _native.library().pointops_cache_attention_step_workspace_bytes(call)
    part = 4 * (D + 4)
    per, heads = H // G, G
    blocks = heads * -(-B * per // 64)  # of the start's rows, where they are many
    splits = max(2, -(-512 // blocks))
    assert B * H * 2 * part <= size <= (B * H + (heads * (B * per + 63)) * splits) * part
