"""Refusals of the frame-cache entry points (no GPU needed) and the oracle's own small cases."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import cache_oracle as CO
from turbo_roformer_b200 import _lib, cache_append, cache_attention, cache_plan

P = ctypes.c_void_p(4096)  # a pointer that no refused call follows


def refused(fn, args, word):
    rc = getattr(_lib.load(), fn)(*args)
    assert rc == -1, rc
    assert word in _lib.load().trc_last_error().decode()


PLAN = dict(cached=P, new=P, n_seqs=2, page=16, free=P, n_free=4, table=P, stride=3, rows=5, cu=P, total=P, slots=P,
            positions=P, counts=P, stream=None)
APPEND = dict(precision=0, qkv=P, row_stride=192, band_stride=192, rows=2, bands=1, heads=1, kv_heads=1, positions=P,
              slots=P, freqs=P, page=16, n_pages=4, q=P, q_stride=64, k=P, v=P, gates=None, status=None, stream=None)
ATTENTION = dict(precision=1, q=P, q_stride=64, k=P, v=P, table=P, stride=2, cu=P, total=P, n_seqs=1, rows=2, max_new=2,
                 max_total=20, heads=1, kv_heads=1, page=16, n_pages=4, causal=1, window=0, scale=0.125, gates=None,
                 out=P, out_stride=64, workspace=None, workspace_bytes=0, status=None, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(cached=None), "null"), (dict(counts=None), "null"), (dict(free=None), "null"), (dict(slots=None), "null"),
    (dict(n_seqs=0), "sequences"), (dict(n_seqs=8193), "sequences"), (dict(page=48), "page"), (dict(page=0), "page"),
    (dict(n_free=-1), "sizes"), (dict(stride=0), "sizes"), (dict(rows=-1), "sizes")])
def test_plan_refuses(change, word):
    refused("trc_cache_plan", tuple({**PLAN, **change}.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(precision=2), "precision"), (dict(rows=-1), "sizes"), (dict(bands=0), "sizes"), (dict(heads=3, kv_heads=2), "sizes"),
    (dict(n_pages=0), "sizes"), (dict(page=256), "page"), (dict(qkv=None), "null"), (dict(slots=None), "null"),
    (dict(k=None), "null"), (dict(row_stride=196), "16-byte"), (dict(q=ctypes.c_void_p(4104)), "16-byte"),
    (dict(bands=2, band_stride=128, q_stride=128), "strides"), (dict(q_stride=56), "strides"),
    (dict(freqs=ctypes.c_void_p(4100)), "16-byte"),
    (dict(rows=1 << 21), "1,048,560"), (dict(rows=1048561), "1,048,560")])
def test_append_refuses(change, word):
    refused("trc_cache_append", tuple({**APPEND, **change}.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(precision=-1), "precision"), (dict(n_seqs=0), "sequences"), (dict(n_seqs=2049), "sequences"),
    (dict(rows=-1), "sizes"), (dict(max_new=-1), "sizes"), (dict(max_total=-1), "sizes"), (dict(window=-1), "sizes"),
    (dict(heads=3, kv_heads=2, q_stride=192, out_stride=192), "sizes"), (dict(stride=0), "sizes"),
    (dict(heads=65, q_stride=65 * 64, out_stride=65 * 64), "TRC_CACHE_MAX_GROUP"), (dict(page=8), "page"),
    (dict(n_pages=1 << 28), "2^31"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(q=None), "null"),
    (dict(cu=None), "null"), (dict(out=None), "null"), (dict(q_stride=68), "16-byte"),
    (dict(k=ctypes.c_void_p(4098)), "16-byte"), (dict(out_stride=56), "strides")])
def test_attention_refuses(change, word):
    refused("trc_cache_attention", tuple({**ATTENTION, **change}.values()), word)


def test_workspace_refuses():
    for args in ((-1, 8, 8), (1, 8, 3), (1, 0, 1), (1, 65, 1)):
        assert _lib.load().trc_cache_workspace(*args) == -1


def test_no_rows_is_no_work():
    """Nothing to do returns before any device is asked for."""
    assert _lib.load().trc_cache_append(*{**APPEND, "rows": 0}.values()) == 0
    assert _lib.load().trc_cache_attention(*{**ATTENTION, "rows": 0}.values()) == 0


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        cache_plan(i, i, i[:, None], i, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        cache_append(torch.zeros(2, 1, 192, dtype=torch.float16), i, i, pool, pool, 1, 1, freqs=None)
    with pytest.raises(ValueError, match="CUDA"):
        cache_attention(torch.zeros(2, 1, 64, dtype=torch.float16), pool, pool, i[:, None], i, i[:1], 1, 1)


def test_oracle_plan_by_hand():
    """Pages of 16: 15 + 3 frames cross into a new page, 16 + 0 need none, 0 + 20 take two."""
    table, cu, total, slots, pos, taken, flags = CO.plan([15, 16, 0], [3, 0, 20], 16, [9, 8, 7, 6],
                                                         [[1, -1], [2, -1], [-1, -1]], 25)
    assert table.tolist() == [[1, 9], [2, -1], [8, 7]] and cu == [0, 3, 3, 23] and total == [18, 16, 20]
    assert slots.tolist() == [31, 144, 145, *range(128, 144), 112, 113, 114, 115, -1, -1]
    assert pos.tolist() == [15, 16, 17, *range(20), 0, 0] and (taken, flags) == (3, 0)


def test_oracle_attention_is_softmax():
    """One sequence whose pages lie in order, against torch's softmax in 64 bits."""
    r = np.random.default_rng(0)
    q, k, v = r.standard_normal((5, 4, 64)), r.standard_normal((2, 2, 16, 64)), r.standard_normal((2, 2, 16, 64))
    out, _, keys = CO.attention(q, k, v, [[1, 0]], [0, 5], [23], 16, True, 7, 0.125)
    kk = torch.from_numpy(np.concatenate([k[1], k[0]], 1)[:, :23]).repeat_interleave(2, 0)
    vv = torch.from_numpy(np.concatenate([v[1], v[0]], 1)[:, :23]).repeat_interleave(2, 0)
    s = torch.from_numpy(q).transpose(0, 1) @ kk.transpose(1, 2) / 8
    back = torch.arange(18, 23)[:, None] - torch.arange(23)
    s = s.masked_fill((back < 0) | (back >= 7), -torch.inf)
    np.testing.assert_allclose(out, (s.softmax(-1) @ vv).transpose(0, 1).numpy(), rtol=1e-12, atol=1e-14)
    assert keys.tolist() == [7] * 5
