"""Sizes past the frame cache's 32-bit offsets are refused (no GPU needed: the calls return before any device)."""

from __future__ import annotations

import pytest

from .test_frame_cache_host import ATTENTION, refused


@pytest.mark.parametrize("heads,kv", [(1 << 25, 1 << 19), (1 << 25, 1 << 25), (2**31 - 64, 2**25 - 1)])
def test_attention_refuses_rows_past_31_bits(heads, kv):
    """A row of 2^31 elements (4 GB) or more: offsets within a row are 32-bit."""
    change = dict(rows=1, heads=heads, kv_heads=kv, n_pages=1)
    refused("trc_cache_attention", tuple({**ATTENTION, **change}.values()), "2^31 elements")
