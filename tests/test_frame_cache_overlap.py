"""Buffers of the frame-cache calls that share memory are refused before any device is asked for (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest

from .test_frame_cache_host import PLAN, refused


def at(address):
    return ctypes.c_void_p(address)  # none that a refused call follows


# 2 sequences, 3 table columns, 5 rows, 4 free pages, a buffer every 4,096 bytes
SPREAD = {**PLAN, **{name: at(4096 * (i + 1)) for i, name in enumerate(
    ("cached", "new", "free", "table", "cu", "total", "slots", "positions", "counts"))}}


@pytest.mark.parametrize("written,size", [("table", 24), ("cu", 12), ("total", 8), ("slots", 20), ("positions", 20),
                                          ("counts", 8)])
@pytest.mark.parametrize("other,other_size", [("cached", 8), ("new", 8), ("free", 16), ("table", 24), ("cu", 12),
                                              ("total", 8), ("slots", 20), ("positions", 20), ("counts", 8)])
def test_plan_refuses_overlap(written, size, other, other_size):
    """The same buffer, and one that begins or ends inside the other by one element."""
    if written == other:
        return
    base = SPREAD[other].value
    for address in (base, base + other_size - 4, base - size + 4):
        refused("trc_cache_plan", tuple({**SPREAD, written: at(address)}.values()), "overlap")
