"""Buffers of the frame-cache calls that share memory are refused before any device is asked for (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest

from .test_frame_cache_host import APPEND, ATTENTION, PLAN, refused


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


# 6 rows of one band with 2 heads and a cache head, 768 bytes apart; q rows 256 bytes, 768 apart; pools of 4 pages
ROWS = {**APPEND, **dict(rows=6, heads=2, row_stride=384, q_stride=384),
        **{name: at(65536 * (i + 1)) for i, name in enumerate(("qkv", "positions", "slots", "freqs", "q", "k", "v"))}}


@pytest.mark.parametrize("change", [
    dict(v=ROWS["k"]), dict(v=at(ROWS["k"].value + 4 * 2048 - 16)), dict(k=ROWS["qkv"]), dict(q=ROWS["k"]), dict(q=ROWS["slots"]),
    dict(gates=ROWS["q"]), dict(gates=ROWS["positions"]), dict(freqs=at(ROWS["v"].value + 16)),
    dict(q=at(ROWS["qkv"].value + 16)), dict(q=at(ROWS["qkv"].value + 496)), dict(q=at(ROWS["qkv"].value + 528 + 768)),
    dict(q=at(ROWS["qkv"].value - 256 + 16)), dict(q=ROWS["qkv"], q_stride=392), dict(q=ROWS["qkv"], row_stride=0),
    dict(q=ROWS["qkv"], row_stride=200, q_stride=200), dict(q=at(ROWS["qkv"].value - 5 * 768), row_stride=-384),
    dict(q=ROWS["qkv"], bands=2, band_stride=256, row_stride=512, q_stride=512)])
def test_append_refuses_overlap(change):
    refused("trc_cache_append", tuple({**ROWS, **change}.values()), "overlap")


SEEN = {**ATTENTION, **dict(rows=6, heads=2, kv_heads=1, q_stride=384, out_stride=384, gates=at(4096), workspace=at(8192),
                            workspace_bytes=1024),
        **{name: at(65536 * (i + 1)) for i, name in enumerate(("q", "k", "v", "table", "cu", "total", "out"))}}


@pytest.mark.parametrize("change", [
    dict(out=SEEN["q"]), dict(out=at(SEEN["q"].value + 240)), dict(out=at(SEEN["q"].value - 240 + 768)),
    dict(out=at(SEEN["q"].value + 256), out_stride=392), dict(out=SEEN["k"]), dict(out=at(SEEN["v"].value + 4 * 2048 - 16)),
    dict(out=SEEN["table"]), dict(cu=SEEN["out"]), dict(total=at(SEEN["out"].value + 16)), dict(gates=SEEN["out"]),
    dict(workspace=SEEN["out"]), dict(workspace=SEEN["q"]), dict(workspace=SEEN["k"]), dict(workspace=SEEN["gates"])])
def test_attention_refuses_overlap(change):
    refused("trc_cache_attention", tuple({**SEEN, **change}.values()), "overlap")
