"""Sizes that the 4-bit attention's entry point refuses before it launches."""

from __future__ import annotations

import pytest

from cacheslide_b200 import _native as N


@pytest.mark.parametrize("tokens,q_heads", [(2 ** 31 - 2, 2), (2 ** 31 - 130, 2),
                                            ((2 ** 31 - 2) // 8, 16), (2 ** 40, 2)])
def test_rows_that_a_tile_more_carries_past_31_bits(tokens, q_heads):
    """Row tiles are counted with the last one whole."""
    p = N.KV4AttnParams()
    p.pool = N.KV4Pool(None, 0, 2, 16, 128, 64, N.CS_BF16)
    p.tokens, p.q_heads, p.scale, p.requests = tokens, q_heads, 1.0, 0
    p.q = p.out = p.starts = 4096  # not looked at
    assert N.load().cs_kv4_attn_workspace(p) == 0
    assert N.load().cs_kv4_attn(p, 4096, None) == N.CS_ERR_INVALID
