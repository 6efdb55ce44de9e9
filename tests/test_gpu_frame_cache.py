"""The frame cache on the GPU (trc_cache_plan / _append / _attention) against its 64-bit oracle, and a run of them
together against the whole-chunk stages.

Tolerances. Append: one rotation in fp32 (two products, a sum, cos and sin good to 2^-23 and an angle rounded to
2^-25 half turns: together below 2^-21 of |x0| + |x1|), one rounding of at most half a step u of the type
(2^-11 fp16, 2^-8 bf16) of the value. Attention, with A = sum p_j |v_j| (gated) from the oracle: rounding each
weight to 16 bits moves the result by at most u A; the weights' own relative error e comes from the score (70 fp32
roundings of sum |q_i k_i| scale) and the exponential (7.5e-5 at most) and counts twice, in the sum and in the
norm; fp32 sums over n keys add n 2^-24 A, twice; fp16 weights below 2^-25 flush, n 2^-25 max|v| at most; and the
result is rounded once, u |ref|."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import cache_oracle as CO
from turbo_roformer_b200 import CachePlan, cache_append, cache_attention, cache_plan

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def f64(t):
    return t.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ plan
def run_plan(cached, new, page, free, table, max_rows, **kw):
    t = ints(table)
    p = cache_plan(ints(cached), ints(new), t, ints(free), page, max_rows, **kw)
    return t, p


def check_plan(cached, new, page, free, table, max_rows):
    t, p = run_plan(cached, new, page, free, table, max_rows)
    rt, cu, total, slots, pos, taken, flags = CO.plan(cached, new, page, free, table, max_rows)
    assert p.counts.tolist() == [taken, flags]
    assert p.cu.tolist() == cu and p.total.tolist() == total
    assert np.array_equal(t.cpu().numpy(), rt)
    assert np.array_equal(p.slots.cpu().numpy(), slots)
    assert np.array_equal(p.positions.cpu().numpy(), pos)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n,cached_to,new_to,pad", [(1, 0, 1, 0), (1, 1000, 700, 5), (7, 40, 3, 1), (513, 90, 40, 17),
                                                    (1500, 300, 20, 1000), (8192, 50, 2, 3)])
def test_plan_matches_oracle(cuda_device, page, n, cached_to, new_to, pad):
    r = np.random.default_rng([page, n])
    cached, new = r.integers(0, cached_to + 1, n), r.integers(0, new_to + 1, n)
    need = -(-(cached + new) // page)
    width = int(need.max()) + 2
    pages = r.permutation(int(need.sum()) + 3)
    table = np.full((n, width), -1)
    held, at = -(-cached // page), 0
    for i, h in enumerate(held):
        table[i, :h] = pages[at:at + h]
        at += h
    check_plan(cached.tolist(), new.tolist(), page, pages[at:].tolist(), table, int(new.sum()) + pad)


def test_plan_page_edges(cuda_device):
    """Lengths at, one below and one above page borders; nothing cached, nothing new."""
    cached = [0, 0, 15, 16, 17, 31, 32, 0, 16, 15]
    new = [0, 16, 1, 1, 15, 2, 0, 17, 16, 18]
    table = np.arange(40).reshape(10, 4) + 100
    check_plan(cached, new, 16, list(range(50, 70)), table, sum(new))


@pytest.mark.parametrize("case", ["no_pages", "no_free_list", "table_full", "rows_full", "no_rows", "negative", "huge"])
def test_plan_flags(cuda_device, case):
    cached, new, free, table, rows = [5, 40, 0, 7], [30, 10, 20, 0], list(range(20)), np.full((4, 6), 77), 60
    if case == "no_pages":
        free = [3, 4]
    elif case == "no_free_list":
        free = []
    elif case == "table_full":
        table = np.full((4, 2), 77)
    elif case == "rows_full":
        rows = 33
    elif case == "no_rows":
        rows = 0
    elif case == "negative":
        cached, new = [5, -1, 0, 7], [30, 10, -20, 0]
    elif case == "huge":
        cached, new = [5, 2**31 - 1, 0, 2**30], [30, 2**31 - 1, 20, 1]
    check_plan(cached, new, 16, free, table, rows)


def test_plan_into_given_buffers_and_refusals(cuda_device):
    cached, new, table, free = ints([3, 4]), ints([2, 0]), ints([[0, -1], [1, -1]]), ints([5, 6])
    first = cache_plan(cached, new, table, free, 16, 4)
    given = CachePlan(*(torch.full_like(t, -9) for t in first))
    again = cache_plan(cached, new, table, free, 16, 4, out=given)
    assert again is given
    for a, b in zip(first, given):
        assert torch.equal(a, b)
    for args in [(cached, new[:1], table, free, 16, 4), (cached, new, table[:1], free, 16, 4),
                 (cached, new, table, free, 48, 4), (cached.long(), new, table, free, 16, 4),
                 (cached, new, table.t(), free, 16, 4), (cached, new.cpu(), table, free, 16, 4),
                 (cached, new, table, free, 16, -1)]:
        with pytest.raises(ValueError):
            cache_plan(*args)
    with pytest.raises(ValueError):
        cache_plan(cached, new, table, free, 16, 5, out=given)


# ------------------------------------------------------------------------------------------------ append
FREQS = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,bands,heads,kv,page,far,gates,rope", [
    (1, 1, 1, 1, 16, 0, True, True), (3, 2, 8, 8, 64, 1700, True, True), (37, 1, 7, 1, 32, 10**7, True, True),
    (200, 1, 12, 4, 16, 2**30, False, True), (5, 62, 8, 8, 128, 999, True, True), (70, 3, 5, 5, 16, 300, False, False),
    (1000, 1, 1, 1, 64, 5000, True, True)])
def test_append_matches_oracle(cuda_device, dtype, rows, bands, heads, kv, page, far, gates, rope):
    dt, r = DT[dtype], np.random.default_rng([rows, bands, heads])
    width = (heads + 2 * kv) * 64 + (-(-heads // 8) * 8 if gates else 0)
    # strided: rows and bands of a larger buffer
    big = torch.from_numpy(r.standard_normal((rows, bands + 1, width + 8)).astype(np.float32)).to(dt).cuda()
    qkv = big[:, :bands, 8:]
    n_pages = -(-rows // page) + 2
    slots = r.permutation(n_pages * page)[:rows]
    pos = np.maximum(0, far - np.arange(rows))
    skip = r.random(rows) < 0.2
    slots[skip] = -1
    k = torch.full((n_pages, bands * kv, page, 64), 7.0, dtype=dt, device="cuda")
    v = torch.full_like(k, 8.0)
    wide = torch.full((rows, bands * heads + 2, 64), 9.0, dtype=dt, device="cuda")
    q = wide[:, 1:-1]
    g = torch.full((rows, bands * heads), 5.0, device="cuda") if gates else None
    status = ints([0])
    cache_append(qkv, ints(pos), ints(slots), k, v, heads, kv, freqs=torch.from_numpy(FREQS).cuda() if rope else None,
                 q=q, gates=g, status=status)
    assert status.item() == 0
    x = f64(qkv)
    split = lambda a, b, h: x[..., a * 64: b * 64].reshape(rows, bands * h, 64)  # noqa: E731
    freqs = FREQS if rope else np.zeros(32)
    u, keep = half_step(dt), ~skip
    for name, src, got in (("q", split(0, heads, heads), f64(q)[keep]),
                           ("k", split(heads, heads + kv, kv), f64(k)[slots[keep] // page, :, slots[keep] % page])):
        ref, size = CO.rotate(src, pos, freqs)
        tol = (u * np.abs(ref) + 2.0**-21 * size + 2.0**-25) if rope else 0.0  # 2^-25: half a step of fp16 subnormals
        assert (np.abs(got - ref[keep]) <= (tol[keep] if rope else 0.0)).all(), name
    assert np.array_equal(f64(v)[slots[keep] // page, :, slots[keep] % page],
                          split(heads + kv, heads + 2 * kv, kv)[keep])
    if gates:
        at = (heads + 2 * kv) * 64
        ref = 1 / (1 + np.exp(-x[..., at:at + heads].reshape(rows, -1)))
        np.testing.assert_allclose(f64(g)[keep], ref[keep], rtol=2e-6)
        assert (g.cpu().numpy()[skip] == 5.0).all()
    # nothing else was written: rows without a slot, the other slots, the buffer around q
    assert (f64(q)[skip] == 9.0).all() and (wide[:, [0, -1]] == 9.0).all()
    untouched = np.ones(n_pages * page, bool)
    untouched[slots[keep]] = False
    free = np.flatnonzero(untouched)
    assert (f64(k)[free // page, :, free % page] == 7.0).all() and (f64(v)[free // page, :, free % page] == 8.0).all()


def test_append_bad_slot_and_refusals(cuda_device):
    dt = torch.float16
    qkv = torch.randn(3, 1, 192, device="cuda").to(dt)
    k = torch.zeros(2, 1, 16, 64, dtype=dt, device="cuda")
    v, status = torch.zeros_like(k), ints([0])
    q, g = cache_append(qkv, ints([0, 1, 2]), ints([31, 32, -5]), k, v, 1, 1, freqs=None, status=status)
    assert status.item() != 0 and g is None  # slot 32 lies behind the pool
    assert torch.equal(v[1, 0, 15], qkv[0, 0, 128:]) and torch.equal(q[0, 0], qkv[0, 0, :64])
    assert v.count_nonzero() == v[1, 0, 15].count_nonzero()
    i = ints([0, 1, 2])
    ok = dict(qkv=qkv, positions=i, slots=i, k_pages=k, v_pages=v, heads=1, kv_heads=1, freqs=None)
    for bad in [dict(qkv=qkv.float()), dict(qkv=qkv[:, 0]), dict(heads=2), dict(kv_heads=0), dict(gates=True),
                dict(positions=i[:2]), dict(slots=i.long()), dict(k_pages=k[:1]), dict(v_pages=v.bfloat16()),
                dict(freqs=torch.zeros(31, device="cuda")), dict(q=torch.zeros(3, 1, 64, device="cuda")),
                dict(gates=torch.zeros(3, 2, device="cuda"), heads=1), dict(k_pages=k[:, :, :8], v_pages=v[:, :, :8]),
                dict(status=torch.zeros(1, device="cuda")), dict(qkv=qkv.expand(3, 2, 192)[..., ::2])]:
        with pytest.raises(ValueError):
            cache_append(**{**ok, **bad})
    with pytest.raises(Exception, match="16-byte"):
        cache_append(**{**ok, "qkv": torch.zeros(3, 1, 200, dtype=dt, device="cuda")[..., 1:193]})


# ------------------------------------------------------------------------------------------------ attention
class Case:
    """A ragged batch over a pool in which everything that no sequence owns is NaN."""

    def __init__(self, dtype, new, total, heads, kv, page, pad=0, seed=0, scale=1.0, gates=False):
        r = np.random.default_rng([seed, heads, page, len(new)])
        dt = DT[dtype]
        self.new, self.total, self.page, self.dtype = list(new), list(total), page, dt
        need = [-(-t // page) for t in total]
        n_pages = sum(need) + 2
        pages = r.permutation(n_pages)
        self.table = np.full((len(new), max(need + [1])), -1)
        k = np.full((n_pages, kv, page, 64), np.nan, np.float32)
        v = k.copy()
        at = 0
        for i, (t, c) in enumerate(zip(total, need)):
            self.table[i, :c] = pages[at:at + c]
            at += c
            for j in range(c):
                live = min(page, t - j * page)
                k[self.table[i, j], :, :live] = r.standard_normal((kv, live, 64)) * scale
                v[self.table[i, j], :, :live] = r.standard_normal((kv, live, 64))
        self.cu = np.concatenate([[0], np.cumsum(new)])
        self.rows = int(self.cu[-1]) + pad
        self.k, self.v = (torch.from_numpy(x).to(dt).cuda() for x in (k, v))
        self.q = torch.from_numpy(r.standard_normal((self.rows, heads, 64)).astype(np.float32) * scale).to(dt).cuda()
        self.gates = torch.from_numpy(r.random((self.rows, heads)).astype(np.float32)).cuda() if gates else None
        self.max_new, self.max_total = max(new), max(total)

    def run(self, out=None, **kw):
        kw = {"max_new": self.max_new, "max_total": self.max_total, **kw}
        return cache_attention(self.q, self.k, self.v, ints(self.table), ints(self.cu), ints(self.total),
                               kw.pop("max_new"), kw.pop("max_total"), gates=self.gates, out=out, **kw)

    def check(self, causal=True, window=0, scale=0.125, **kw):
        heads = self.q.shape[1]
        out = torch.full_like(self.q, 3.0)
        status = ints([0])
        got = self.run(out, causal=causal, window=window, scale=scale, status=status, **kw)
        assert got is out and status.item() == 0
        live = int(self.cu[-1])
        assert (out[live:] == 3.0).all()  # rows behind the last sequence
        k, v = (np.nan_to_num(f64(x)) for x in (self.k, self.v))
        ref, size, keys = CO.attention(f64(self.q), k, v, self.table, self.cu, self.total, self.page, causal, window,
                                       scale, None if self.gates is None else f64(self.gates))
        got, ref, size, keys = f64(out)[:live], ref[:live], size[:live], keys[:live, None, None]
        u = half_step(self.dtype)
        # sum |q_i k_i| scale <= 64 max|q| max|k| scale is far too wide: by Cauchy-Schwarz from the rows' norms
        qk = np.sqrt((f64(self.q)[:live] ** 2).sum(-1)).max(initial=0) * np.sqrt((k**2).sum(-1)).max() * scale
        e = 7.5e-5 + 70 * 2.0**-24 * qk
        tol = 1.01 * (u * np.abs(ref) + size * (u + 2 * e + 2 * keys * 2.0**-24)) + 2.0**-24
        if self.dtype == torch.float16:
            tol = tol + np.minimum(keys, 2.0**11) * 2.0**-25 * np.abs(v).max()
        assert np.isfinite(got).all()
        off = np.abs(got - ref)
        assert (off <= tol).all(), (off / tol).max()
        return out


TINY_LENGTHS = [([1], [1]), ([1], [2]), ([0, 1, 0], [3, 17, 0]), ([2, 5], [2, 40]), ([1, 1, 1], [63, 64, 65]),
                ([16], [16]), ([3, 0, 4], [128, 5, 129])]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new,total", TINY_LENGTHS)
@pytest.mark.parametrize("page", [16, 128])
def test_attention_small(cuda_device, dtype, new, total, page):
    c = Case(dtype, new, total, 2, 2, page, pad=2, gates=True)
    c.check(causal=True)
    c.check(causal=False)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 100, 127, 128, 129, 200, 300, 385, 500])
def test_attention_row_counts(cuda_device, rows):
    """Every variant's row tiles, one row below and above their borders, with keys before and between them."""
    c = Case("fp16", [rows, 1, rows // 2], [rows + 77, 300, rows], 2, 1, 32, seed=rows)
    c.check(causal=True)
    c.check(causal=False, window=50)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (5, 1), (8, 8), (12, 4), (64, 1), (28, 4), (62, 62)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_heads(cuda_device, heads, kv, page):
    c = Case("bf16", [1, 9, 3], [200, 150, 3], heads, kv, page, gates=True)
    c.check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 10**9, 2**31 - 1])
@pytest.mark.parametrize("new", [1, 20, 150])
def test_attention_windows(cuda_device, causal, window, new):
    Case("fp16", [new, new], [new + 333, new], 4, 2, 16, seed=window % 97).check(causal=causal, window=window)


@pytest.mark.parametrize("new", [1, 30, 170])
def test_attention_rows_that_see_nothing(cuda_device, new):
    """Lengths that say fewer frames are cached than the push has: causal rows in front see no key and are zero."""
    c = Case("fp16", [new + 40, new], [new, 0], 2, 2, 16, gates=True)
    out = c.check(causal=True)
    assert not out[:40].any()
    assert not out[new + 40:].any()
    c.check(causal=False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new,total,heads,kv,page", [
    ([1], [20000], 1, 1, 64), ([1], [5003], 8, 8, 128), ([2, 1, 1], [9001, 1, 700], 8, 2, 16),
    ([40], [3000], 2, 1, 32), ([100], [6000], 2, 2, 64), ([130, 1], [2000, 7001], 4, 2, 64)])
def test_attention_long(cuda_device, dtype, new, total, heads, kv, page):
    """Few heads over long caches: runs divided among CTAs and joined."""
    c = Case(dtype, new, total, heads, kv, page, gates=True)
    c.check()
    c.check(causal=False, window=total[0] // 2 + 3)


def test_attention_many_sequences(cuda_device):
    r = np.random.default_rng(5)
    new = r.integers(0, 3, 700)
    total = new + r.integers(0, 90, 700)
    Case("fp16", new.tolist(), total.tolist(), 2, 1, 16).check()
    new = np.zeros(2048, int)
    new[[0, 5, 2047]] = 1, 3, 2
    Case("fp16", new.tolist(), np.where(new > 0, 30, 0).tolist(), 1, 1, 16).check()


def test_attention_many_items_per_cta(cuda_device):
    """More heads than CTAs: whole items, items cut at shares, and their joins in one call."""
    c = Case("fp16", [1, 2], [1000, 600], 496, 496, 64)
    c.check()
    Case("fp16", [40], [200], 496, 496, 64).check(causal=False)


@pytest.mark.parametrize("bounds", [dict(max_new=0), dict(max_new=5000), dict(max_total=0), dict(max_total=10**6)])
def test_attention_bounds_choose_only_the_variant(cuda_device, bounds):
    Case("fp16", [150, 2, 20], [900, 640, 20], 4, 2, 32).check(**bounds)


@pytest.mark.parametrize("new", [1, 20, 60, 110, 400])
def test_attention_rescales(cuda_device, new):
    """Scores that grow along the keys by far more than 2^8: the running maximum moves at every step."""
    c = Case("fp16", [new], [new + 500], 2, 2, 64, seed=3)
    ramp = torch.linspace(0, 6, new + 500, device="cuda")
    for j, page in enumerate(c.table[0]):
        if page >= 0:
            part = ramp[j * 64:(j + 1) * 64]
            c.k[page, :, :len(part), 0] = part.to(c.k.dtype)
    c.q[..., 0] = 8.0
    c.check(causal=False, scale=1.0)
    c.check(causal=True, scale=1.0)


def test_attention_strided_rows(cuda_device):
    c = Case("fp16", [3, 2], [30, 50], 4, 2, 16)
    ref = c.run()
    wide = torch.zeros(5, 6, 64, dtype=c.dtype, device="cuda")
    wide[:, 1:5] = c.q
    c.q = wide[:, 1:5]
    out = torch.full((5, 7, 64), 2.0, dtype=c.dtype, device="cuda")
    c.run(out[:, 2:6])
    assert torch.equal(out[:, 2:6], ref) and (out[:, [0, 1, 6]] == 2.0).all()


def test_attention_nan_stays_in_its_row(cuda_device):
    """A NaN query makes its own row NaN and no other; NaN behind the lengths makes none (every case's pool)."""
    for new in (3, 140):
        c = Case("fp16", [new], [new + 100], 2, 2, 16)
        want = c.run().clone()
        c.q[1, 0, 5] = float("nan")
        got = c.run()
        assert got[1, 0].isnan().all()
        got[1, 0] = want[1, 0]
        assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 140])
def test_attention_pages_before_the_window_are_not_read(cuda_device, new):
    """Pages that fell out of the window may be given back: their table entries are not followed."""
    c = Case("fp16", [new], [1500], 2, 2, 16)
    want = c.run(window=64).clone()
    gone = (1500 - new - 63) // 16
    c.table[0, :gone] = -1
    status = ints([0])
    assert torch.equal(c.run(window=64, status=status), want) and status.item() == 0


@pytest.mark.parametrize("new", [1, 140])
def test_attention_bad_lengths_and_pages(cuda_device, new):
    """Pages outside the pool set the status, and the other sequence's rows are right; lengths beyond the table
    and offsets beyond the rows read nothing outside the buffers."""
    c = Case("fp16", [new, 2], [600, 90], 2, 2, 16)
    want = c.run().clone()
    good = c.table.copy()
    for bad in (-1, 10**6, 2**31 - 1, c.k.shape[0]):
        c.table = good.copy()
        c.table[0, 3] = bad
        status = ints([0])
        got = c.run(status=status)
        assert status.item() != 0
        assert torch.equal(got[new:], want[new:])
    c.table = good
    c.total = [10**9, 90]  # clamped to the table; entries behind the first sequence's pages are -1
    got = c.run()
    assert torch.equal(got[new:], want[new:])
    c.total = [600, 90]
    cu = c.cu.copy()
    for cu_bad in ([0, new, 10**9], [-5, new, new + 2], [0, new + 2, new]):
        c.cu = np.array(cu_bad)
        c.run()
    c.cu = cu
    assert torch.equal(c.run(), want)


def test_attention_refusals(cuda_device):
    c = Case("fp16", [2], [20], 2, 2, 16)
    t, cu, total = ints(c.table), ints(c.cu), ints(c.total)
    ok = dict(q=c.q, k_pages=c.k, v_pages=c.v, table=t, cu=cu, total=total, max_new=2, max_total=20)
    for bad in [dict(q=c.q.float()), dict(q=c.q[:, :, :32]), dict(q=c.q[:, :1].expand(2, 3, 64)), dict(k_pages=c.k.bfloat16()),
                dict(k_pages=c.k.cpu()), dict(table=t.long()), dict(cu=cu[:1]), dict(total=ints([20, 20])),
                dict(gates=torch.zeros(2, 2, device="cuda", dtype=torch.float16)), dict(out=torch.zeros(2, 2, 64, device="cuda")),
                dict(v_pages=c.v.transpose(0, 1)), dict(q=c.q[:, :, ::2])]:
        with pytest.raises(ValueError):
            cache_attention(**{**ok, **bad})
    for bad in [dict(window=-1), dict(scale=0.0), dict(max_new=-1), dict(max_total=-1)]:
        with pytest.raises(Exception, match="cache attention"):
            cache_attention(**{**ok, **bad})
    # the C entry needs its workspace where a run may be divided
    from turbo_roformer_b200 import _lib

    p = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
    rc = _lib.load().trc_cache_attention(0, p(c.q), 128, p(c.k), p(c.v), p(t), t.shape[1], p(cu), p(total), 1, 2, 2, 5000,
                                         2, 2, 16, c.k.shape[0], 1, 0, 0.125, None, p(c.q.clone()), 128, None, 0, None, None)
    assert rc == -1 and b"workspace" in _lib.load().trc_last_error()


@pytest.mark.parametrize("new", [1, 30, 200])
def test_attention_on_another_stream_and_repeated(cuda_device, new):
    c = Case("fp16", [new, 3], [new + 1500, 700], 8, 8, 64)
    want = c.run().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [c.run() for _ in range(3)]
    s.synchronize()
    for g in got:  # the joins go by the order of the keys: bit for bit
        assert torch.equal(g, want)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new,total,heads,kv,page", [
    ([200], [455], 12, 4, 16), ([60, 77, 3], [60, 700, 90], 10, 2, 128), ([26, 25, 51], [300, 26, 1000], 5, 1, 32),
    ([7], [200], 64, 1, 64), ([3, 2, 9], [700, 20, 9], 99, 3, 16), ([129, 128, 127, 64, 33, 32], [700] * 6, 2, 2, 64)])
def test_attention_tiles(cuda_device, dtype, new, total, heads, kv, page):
    """Groups that do not divide a tile's 128 rows, tiles that end inside a sequence, batches that take both kernels."""
    c = Case(dtype, new, total, heads, kv, page, pad=5, gates=True, seed=len(new))
    c.check(causal=True)
    c.check(causal=False, window=70)
    c.check(causal=True, window=300)


@pytest.mark.parametrize("new", [40, 150, 400])
def test_attention_many_divided_items(cuda_device, new):
    """Many cache heads, several items and parts of items to each worker of the tensor-core kernel, and the joins."""
    c = Case("fp16", [new, new // 3], [900, 640], 200, 200, 64, gates=True)
    c.check(causal=False)
    c.check(causal=True)


def test_attention_shared_pages(cuda_device):
    """Two sequences whose tables name the same pages (a common beginning): both read them."""
    c = Case("fp16", [1, 40], [300, 300], 2, 2, 32)
    c.table[1, :6] = c.table[0, :6]
    c.check()


@pytest.mark.parametrize("rows", [250, 255, 256, 257, 260, 512, 513])
def test_attention_row_counts_around_shared_tiles(cuda_device, rows):
    """The border between separate and shared tiles, with a sequence of every other variant in the same batch."""
    c = Case("bf16", [rows, 3, 0, rows // 2, 40], [rows + 130, 200, 90, rows, 41], 2, 2, 64, gates=True, seed=rows)
    c.check(causal=True)
    c.check(causal=False, window=90)


@pytest.mark.parametrize("new", [300, 700])
def test_attention_shared_tiles_keep_the_rules(cuda_device, new):
    """Rows that see nothing, NaN queries, pages given back and bad pages in pushes whose tiles share their keys."""
    test_attention_rows_that_see_nothing(cuda_device, new)
    test_attention_pages_before_the_window_are_not_read(cuda_device, new)
    test_attention_bad_lengths_and_pages(cuda_device, new)
    c = Case("fp16", [new], [new + 100], 2, 2, 16)
    want = c.run().clone()
    c.q[1, 0, 5] = float("nan")
    got = c.run()
    assert got[1, 0].isnan().all()
    want[1, 0] = got[1, 0] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [400])
def test_shared_tiles_on_streams_and_divided(cuda_device, new):
    test_attention_on_another_stream_and_repeated(cuda_device, new)
    test_pool_offsets_past_32_bits(cuda_device, new)
    cases = [Case("fp16", n, t, 8, 4, 64, seed=i) for i, (n, t) in enumerate([([200, 20], [1500, 900]), ([1], [3000])])]
    want = [c.run().clone() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(4):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(c.run())
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert torch.equal(out, want[k % 2])


@pytest.mark.parametrize("new", [2, 60, 200])
def test_pool_offsets_past_32_bits(cuda_device, new):
    """Pages whose elements lie more than 2^31 (and bytes more than 2^32) into the pool, written and read."""
    kv, page, n_pages, dt = 8, 128, 36000, torch.float16  # 2.4e9 elements per pool
    k = torch.empty(n_pages, kv, page, 64, dtype=dt, device="cuda")
    v = torch.empty_like(k)
    c = Case("fp16", [new], [new + 300], kv, kv, page, seed=1)
    at = [n_pages - 1 - 7 * i for i in range(c.table.shape[1])]
    for j, p in enumerate(at):
        k[p], v[p] = c.k[c.table[0, j]], c.v[c.table[0, j]]
    c.table[0, :], c.k, c.v = at, k, v
    # the last rows once more, by append
    last = torch.cat([c.q.reshape(new, -1), torch.randn(new, 2 * kv * 64, device="cuda").to(dt)], 1)[:, None]
    pos = np.arange(300, new + 300)
    slots = np.array(at)[pos // page] * page + pos % page
    cache_append(last, ints(pos), ints(slots), k, v, kv, kv, freqs=None, q=c.q)
    assert torch.equal(k[int(slots[-1]) // page, :, int(slots[-1]) % page].reshape(-1), last[-1, 0, kv * 64:2 * kv * 64])
    out = c.run()
    c.k, c.v, c.table = k[at], v[at], np.arange(len(at))[None]
    del k, v
    c.check()
    assert torch.equal(c.run(), out)


def test_two_streams_at_once(cuda_device):
    """Calls that overlap on two streams, of every kernel, each with its own workspace: the same bits as alone."""
    cases = [Case("fp16", n, t, 8, 4, 64, seed=i) for i, (n, t) in enumerate(
        [([1, 2], [3000, 700]), ([40, 1], [2000, 2000]), ([200, 20], [1500, 900])])]
    want = [c.run().clone() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(6):
        for i, c in enumerate(cases):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append((i, c.run()))
    torch.cuda.synchronize()
    for i, g in got:
        assert torch.equal(g, want[i])


@pytest.mark.parametrize("new", [1, 50, 300])
def test_captured_attention_follows_the_lengths(cuda_device, new):
    """A captured call reads lengths and tables at replay: shorter, longer and empty pushes within its capacity."""
    c = Case("fp16", [new, new], [new + 800, new + 500], 4, 2, 32, gates=True)
    table, cu, total = ints(c.table), ints(c.cu), ints(c.total)
    out, status = torch.zeros_like(c.q), ints([0])
    call = lambda: cache_attention(c.q, c.k, c.v, table, cu, total, c.max_new, c.max_total, gates=c.gates, out=out,  # noqa: E731
                                   status=status)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for a, b in ([new, new], [0, new], [new, 0], [0, 0], [(new + 1) // 2, 1]):
        c.new, c.cu = [a, b], np.array([0, a, a + b])
        cu.copy_(ints(c.cu))
        out.fill_(3.0)
        graph.replay()
        assert status.item() == 0 and (out[a + b:] == 3.0).all()
        want = torch.full_like(out, 3.0)
        c.run(want)
        assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ together
def test_whole_chunk_equals_the_chunk_stages(tiny_cuda, tiny_cfg):
    """A whole chunk pushed into an empty cache: the same attention as trc_rope_pack + trc_attention (time mode)."""
    from turbo_roformer_b200 import _lib

    T, Fb = 130, tiny_cfg.n_bands
    g = torch.Generator().manual_seed(11)
    qkvg = (torch.randn(T * Fb, 1544, generator=g) * 0.5).half().cuda()
    p = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
    st = ctypes.c_void_p(tiny_cuda.stream_ptr())
    Q = torch.empty(T * Fb * 512, device="cuda", dtype=torch.float16)
    K, V, O = torch.empty_like(Q), torch.empty_like(Q), torch.empty_like(Q)
    G = torch.empty(T * Fb, 8, device="cuda")
    _lib.check(tiny_cuda.lib.trc_rope_pack(tiny_cuda.handle, 0, p(qkvg), 1, T, p(Q), p(K), p(V), p(G), st))
    _lib.check(tiny_cuda.lib.trc_attention(tiny_cuda.handle, 0, p(Q), p(K), p(V), p(G), p(O), 1, T, st))
    tiny_cuda.check()
    page = 32
    k = torch.full((6, Fb * 8, page, 64), float("nan"), device="cuda", dtype=torch.float16)
    v, table = k.clone(), ints(np.full((1, 5), -1))
    plan = cache_plan(ints([0]), ints([T]), table, ints([4, 2, 0, 5, 1, 3]), page, T)
    q, gates = cache_append(qkvg.view(T, Fb, 1544), plan.positions, plan.slots, k, v, 8, 8,
                            freqs=torch.from_numpy(FREQS).cuda(), gates=True)
    out = cache_attention(q, k, v, table, plan.cu, plan.total, T, T, causal=False, scale=1.0, gates=gates)
    assert torch.equal(gates.view_as(G), G) and plan.counts.tolist() == [5, 0]
    ref, got = O.view(T, Fb * 8, 64).double(), out.double()
    # two kernels of the same arithmetic: weights and result rounded once each on either side, and q and k rounded to
    # neighbouring values where the angles' last bits differ
    assert 20 * torch.log10(ref.norm() / (got - ref).norm()) >= 60


@pytest.mark.parametrize("graph", [False, True])
def test_pushes_of_live_streams(cuda_device, graph):
    """Streams that come, grow push by push and are cut to a window: plan, append and attention of every push, in a
    captured graph or not, against the oracle on the whole history; padded rows stay as they were."""
    heads, kv, page, bands, window, cap = 4, 2, 16, 3, 40, 24
    r, dt = np.random.default_rng(3), torch.float16
    n, cols, n_pages = 3, 12, 40
    k = torch.full((n_pages, bands * kv, page, 64), float("nan"), dtype=dt, device="cuda")
    v, table = torch.full_like(k, float("nan")), ints(np.full((n, cols), -1))
    cached, new, status = ints([0] * n), ints([0] * n), ints([0])
    free = ints(r.permutation(n_pages))
    qkv = torch.zeros(cap, bands, (heads + 2 * kv) * 64 + 8, dtype=dt, device="cuda")
    q = torch.full((cap, bands * heads, 64), 6.0, dtype=dt, device="cuda")
    out, gates = q.clone(), torch.full((cap, bands * heads), 6.0, device="cuda")
    freqs = torch.from_numpy(FREQS).cuda()
    bound_new, bound_total = cap, cols * page

    def push():
        plan = cache_plan(cached, new, table, free, page, cap)
        cache_append(qkv, plan.positions, plan.slots, k, v, heads, kv, freqs=freqs, q=q, gates=gates, status=status)
        cache_attention(q, k, v, table, plan.cu, plan.total, bound_new, bound_total, window=window, gates=gates,
                        out=out, status=status)
        return plan

    captured = None
    if graph:
        push()  # loads and attributes outside the capture
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            plan = push()
    history = [[] for _ in range(n)]
    for lengths in ([5, 0, 1], [1, 1, 1], [10, 3, 11], [0, 0, 0], [1, 20, 2], [13, 1, 1]):
        out.fill_(6.0)
        new.copy_(ints(lengths))
        x = torch.from_numpy(r.standard_normal(tuple(qkv.shape)).astype(np.float32)).to(dt)
        qkv.copy_(x)
        if graph:
            captured.replay()
        else:
            plan = push()
        taken, flags = plan.counts.tolist()
        assert flags == 0 and status.item() == 0
        at = 0
        for i, m in enumerate(lengths):
            history[i] += [f64(x[at + j]) for j in range(m)]
            if m:
                rows = np.stack(history[i])[:, :, : (heads + 2 * kv) * 64]
                split = lambda a, b, h: rows[..., a * 64: b * 64].reshape(len(rows), bands * h, 64)  # noqa: E731
                # the oracle's own rotation, rounded once to the type as the cache holds it
                half = lambda y: y.astype(np.float16).astype(np.float64)  # noqa: E731
                qs = half(CO.rotate(split(0, heads, heads), np.arange(len(rows)), FREQS)[0])
                ks = half(CO.rotate(split(heads, heads + kv, kv), np.arange(len(rows)), FREQS)[0])
                vs = split(heads + kv, heads + 2 * kv, kv)
                pad = -(-len(rows) // page) * page - len(rows)
                pool = lambda y: np.pad(y, ((0, pad), (0, 0), (0, 0))).reshape(-1, page, bands * kv, 64).transpose(  # noqa: E731
                    0, 2, 1, 3)
                g = 1 / (1 + np.exp(-f64(x[at:at + m])[..., (heads + 2 * kv) * 64:][..., :heads].reshape(m, -1)))
                ref, size, _ = CO.attention(qs[-m:], pool(ks), pool(vs), [list(range(len(rows)))], [0, m],
                                            [len(rows)], page, True, window, 0.125, g)
                # as in Case.check; q and k may be rounded to the neighbouring value where the rotation's fp32 error
                # crosses a border: each such element moves a score by at most a step of one product
                e = 7.5e-5 + (70 * 2.0**-24 + 2 * 2.0**-10 / 8) * 15 * 15 * 0.125
                tol = 1.01 * (2.0**-11 * np.abs(ref) + size * (2.0**-11 + 2 * e)) + 40 * 2.0**-25 * 5
                assert (np.abs(f64(out[at:at + m]) - ref) <= tol).all()
            at += m
        assert (out[at:] == 6.0).all()
        # what a program keeps between pushes: lengths and the rest of the free list
        cached.add_(new)
        free.copy_(torch.cat([free[taken:], free[:taken]]))
