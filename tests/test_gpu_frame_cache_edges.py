"""The frame cache on the GPU where it can go wrong: blocks of several frames, keys and values that are not finite,
lengths that do not fit, buffers that overlap. Tolerances are those derived in test_gpu_frame_cache.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import cache_oracle as CO
from turbo_roformer_b200 import cache_append, cache_attention, cache_plan

from .test_gpu_frame_cache import FREQS, Case, f64, ints, test_append_matches_oracle as check_append

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ append
# Frames of a block: the most of 16, 8, 4, 2, 1 that leave eight blocks per SM (1,184 on 148 SMs). A thread then takes
# every 32 / frames-th head row, four in flight: 8, 16, 32, 64 or 128 head rows at a time.
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("frames,rows,bands,heads,kv,page,gates,rope", [
    (16, 18961, 1, 11, 1, 16, False, True), (16, 333, 62, 11, 1, 64, True, True), (16, 329, 62, 8, 8, 128, True, True),
    (8, 161, 62, 18, 2, 32, True, True), (8, 9601, 1, 7, 7, 64, True, False), (4, 83, 62, 33, 3, 16, True, True),
    (4, 5003, 1, 40, 8, 128, False, True), (2, 41, 60, 65, 5, 32, True, True), (1, 3, 2, 130, 10, 16, True, True)])
def test_append_frames_of_a_block(cuda_device, dtype, frames, rows, bands, heads, kv, page, gates, rope):
    """Every number of frames to a block, last blocks that are not full, rows without a slot beside live ones, and head
    rows that take several passes with a ragged end."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    most = [f for f in (16, 8, 4, 2) if -(-rows // f) * bands >= 8 * sms]
    assert sms != 148 or (most or [1])[0] == frames
    assert rows % frames or frames == 1
    check_append(cuda_device, dtype, rows, bands, heads, kv, page, 123456, gates, rope)


def test_append_bad_slots_beside_good_ones(cuda_device):
    """Blocks of 16 frames in which some slots lie behind the pool: those rows' k and v go nowhere, all others arrive."""
    rows, bands, heads, kv, page, dt = 333, 62, 3, 1, 16, torch.float16
    r = np.random.default_rng(8)
    n_pages = -(-rows // page)
    slots = r.permutation(n_pages * page)[:rows]
    bad = r.random(rows) < 0.1
    slots[bad] += n_pages * page
    qkv = torch.randn(rows, bands, (heads + 2 * kv) * 64, device="cuda").to(dt)
    k = torch.full((n_pages, bands * kv, page, 64), 7.0, dtype=dt, device="cuda")
    v, status = torch.full_like(k, 8.0), ints([0])
    q, _ = cache_append(qkv, ints(np.arange(rows)), ints(slots), k, v, heads, kv, freqs=None, status=status)
    assert status.item() != 0
    assert torch.equal(q, qkv[:, :, :heads * 64].reshape(rows, bands * heads, 64))
    want_k, want_v = torch.full_like(k, 7.0), torch.full_like(v, 8.0)
    good = torch.from_numpy(slots[~bad]).cuda()
    rest = qkv[torch.from_numpy(~bad).cuda()]
    want_k[good // page, :, good % page] = rest[:, :, heads * 64:(heads + kv) * 64]
    want_v[good // page, :, good % page] = rest[:, :, (heads + kv) * 64:]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


# ------------------------------------------------------------------------------------------------ not finite
VARIANTS = [1, 20, 60, 140, 400]  # new frames of one query head: every kernel form


def put(c, pool, frame, value, dims=slice(None)):
    """`value` into a frame of the first sequence, all cache heads."""
    pool[int(c.table[0, frame // c.page]), :, frame % c.page, dims] = value


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", VARIANTS)
def test_nan_key_makes_the_rows_that_see_it_nan(cuda_device, dtype, new):
    """A NaN in one key, at every place of 16: rows that see it are NaN, the others as if it were not there."""
    c = Case(dtype, [new], [new + 70], 2, 2, 32)
    want = c.run().clone()
    keep = c.k.clone()
    for at in [*range(16, 32), 70 + new // 2, 70 + new - 1]:
        c.k.copy_(keep)
        put(c, c.k, at, float("nan"), slice(5, 6))
        got = c.run()
        sees = torch.arange(70, 70 + new, device="cuda") >= at
        assert got[sees].isnan().all(), at
        assert torch.equal(got[~sees], want[~sees]), at


@pytest.mark.parametrize("new", VARIANTS)
def test_nan_key_alone_in_the_window(cuda_device, new):
    """Rows that see one key only: NaN where that key is NaN, the value itself elsewhere."""
    c = Case("fp16", [new], [new + 33], 2, 2, 16)
    want = c.run(window=1).clone()
    for frame in range(33, 33 + new, 3):
        put(c, c.k, frame, float("nan"))
    got = c.run(window=1)
    gone = torch.arange(new, device="cuda") % 3 == 0
    assert got[gone].isnan().all() and torch.equal(got[~gone], want[~gone])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", VARIANTS)
def test_infinite_keys(cuda_device, dtype, new):
    """A key element of +inf: scores of +inf make the row NaN, scores of -inf are weights of zero."""
    for at in (3, 14, 15, 65, 78, 79):
        c = Case(dtype, [new], [new + 100], 1, 1, 64)
        put(c, c.k, at, float("inf"), slice(9, 10))
        got = f64(c.run(causal=False))
        up = f64(c.q)[:, 0, 9] > 0
        assert np.isnan(got[up]).all(), at
        k, v = np.nan_to_num(f64(c.k), posinf=1e30), np.nan_to_num(f64(c.v))
        ref, size, keys = CO.attention(f64(c.q), k, v, c.table, c.cu, c.total, c.page, False, 0, 0.125)
        u = torch.finfo(c.dtype).eps / 2
        norms = np.linalg.norm(f64(c.q)[:, 0], axis=-1).max() * np.linalg.norm(np.where(k < 1e30, k, 0), axis=-1).max()
        e = 7.5e-5 + 70 * 2.0**-24 * norms * 0.125
        tol = 1.01 * (u * np.abs(ref) + size * (u + 2 * e + 2 * (new + 100) * 2.0**-24)) + 2.0**-24
        tol = tol + (new + 100) * 2.0**-25 * np.abs(v).max() * (c.dtype == torch.float16)
        assert (np.abs(got - ref)[~up] <= tol[~up]).all(), at


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("new", [1, 3, 20, 100, 300])
def test_keys_not_finite_in_divided_items(cuda_device, new, value):
    """Long caches whose keys are divided among workers: a key that is not finite in the first, a middle or the last
    part makes the rows of its head NaN that score NaN or +inf there, and no others."""
    total = new + 6000
    for at in (14, 2999, total - new):
        c = Case("fp16", [new, 2], [total, 900], 4, 4, 64, seed=1)
        want = f64(c.run(causal=False))
        c.k[int(c.table[0, at // 64]), 2, at % 64, 7] = value
        got, q = f64(c.run(causal=False)), f64(c.q)
        gone = np.zeros_like(got, bool)
        gone[:new, 2] = True if value != value else (q[:new, 2, 7] > 0)[:, None]
        assert np.isnan(got[gone]).all(), at
        assert np.isfinite(got[~gone]).all(), at
        other = [0, 1, 3]
        assert np.array_equal(got[:, other], want[:, other]) and np.array_equal(got[new:], want[new:]), at


@pytest.mark.parametrize("dtype,big", [("bf16", 3e38), ("fp16", 65504.0)])
@pytest.mark.parametrize("new", VARIANTS)
def test_hidden_values_of_any_finite_size(cuda_device, dtype, big, new):
    """Values of frames that a row's masks hide do not reach it, the type's largest among them."""
    c = Case(dtype, [new], [new + 40], 2, 2, 16)
    c.v.nan_to_num_(0.0)
    c.v.mul_(2.0**-40 if dtype == "bf16" else 1.0)
    first = 40 + new // 2 + 1  # seen by the rows from here on, where there are any
    for frame in range(first, 40 + new):
        put(c, c.v, frame, 0.0)
    want = c.run().clone()
    for frame in range(first, 40 + new):
        put(c, c.v, frame, big if frame % 2 else -big)
    got = c.run()
    assert torch.equal(got[:first - 40], want[:first - 40])


# ------------------------------------------------------------------------------------------------ lengths
@pytest.mark.parametrize("new", [1, 40, 300])
def test_lengths_that_do_not_fit_set_the_status(cuda_device, new):
    """Totals outside the table and offsets outside the rows are reported; the other sequence's rows are right."""
    c = Case("fp16", [new, 2], [600, 90], 2, 2, 16)
    c.table = np.pad(c.table, ((0, 0), (0, 2)), constant_values=0)  # valid pages behind: nothing else to stumble on
    want = c.run().clone()
    for total in (601 + 16 * c.table.shape[1], 2**31 - 1, 2**30 + 1, -1, -2**31):
        c.total, status = [total, 90], ints([0])
        got = c.run(status=status)
        assert status.item() != 0, total
        assert torch.equal(got[new:], want[new:])
    c.total = [600, 90]
    good = c.cu.copy()
    for cu in ([-1, new, new + 2], [0, new, new + 3], [0, new, new - 1], [0, new, 2**31 - 1], [0, -2**31, 2]):
        c.cu, status = np.array(cu), ints([0])
        c.run(status=status)
        assert status.item() != 0, cu
    c.cu, status = good, ints([0])
    assert torch.equal(c.run(status=status), want) and status.item() == 0
    # fewer frames cached than pushed, and a sequence without new frames, are no errors
    c.total = [new // 2, 90]
    c.run(status=status)
    c.cu, c.total = np.array([0, 0, 2]), [-7, 90]
    c.run(status=status)
    assert status.item() == 0


def test_a_full_table_reaches_the_status(cuda_device):
    """A stream that outgrows its table: the plan's flag, and the status of the attention that follows."""
    table, dt = ints([[3, -1]]), torch.float16
    k = torch.randn(6, 1, 16, 64, device="cuda").to(dt)
    plan = cache_plan(ints([16]), ints([20]), table, ints([4, 5, 2]), 16, 20)
    assert plan.counts.tolist() == [2, 2] and plan.total.tolist() == [36]
    status = ints([0])
    cache_attention(torch.randn(20, 1, 64, device="cuda").to(dt), k, k.clone(), table, plan.cu, plan.total, 20, 36,
                    status=status)
    assert status.item() != 0


def test_plan_of_absurd_lengths_ends_soon(cuda_device):
    """Lengths of up to 2^30 frames in every sequence name 2^39 pages: the work stays that of the table and the rows."""
    n, page, rows, free = 8192, 16, 50, [11, 12, 13]
    cached, new = np.full(n, 0), np.full(n, 2**30)
    cached[0], new[0] = 5, 30  # two pages of its own first
    table = ints(np.full((n, 3), 77))
    args = ints(cached), ints(new)
    p = cache_plan(*args, table, ints(free), page, rows)
    torch.cuda.synchronize()
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    t0.record()
    p = cache_plan(*args, table, ints(free), page, rows, out=p)
    t1.record()
    torch.cuda.synchronize()
    want = np.full((n, 3), -1)
    want[0] = 77, 11, 12
    want[1, 0] = 13
    assert np.array_equal(table.cpu().numpy(), want)
    assert p.counts.tolist() == [3, CO.NO_PAGES | CO.TABLE_FULL | CO.ROWS_FULL]
    assert p.cu[:3].tolist() == [0, 30, 30 + 2**30] and p.cu[-1].item() == 2**31 - 1
    slots = [77 * 16 + x for x in range(5, 16)] + [11 * 16 + x for x in range(16)] + [12 * 16 + x for x in range(3)]
    assert p.slots.tolist() == slots + [13 * 16 + x for x in range(16)] + [-1] * 4
    assert p.positions.tolist() == [*range(5, 35), *range(20)]
    # 8,192 sequences in 32 warps are some thousand steps of well under a microsecond; 2^31 pages in 1,024 threads would
    # be two million steps each
    assert t0.elapsed_time(t1) < 50, t0.elapsed_time(t1)


# ------------------------------------------------------------------------------------------------ many sequences
def test_one_plan_for_several_attention_calls(cuda_device):
    """A plan of more sequences than one attention call takes: calls over slices of its table, offsets and totals."""
    r, page, n = np.random.default_rng(4), 16, 3000
    new, total = r.integers(0, 3, n), r.integers(3, 40, n)
    c = Case("bf16", new.tolist(), total.tolist(), 2, 1, page, pad=3)
    table, cu, totals = ints(c.table), ints(c.cu), ints(c.total)
    out, status = torch.full_like(c.q, 3.0), ints([0])
    with pytest.raises(Exception, match="TRC_CACHE_MAX_SEQS"):
        cache_attention(c.q, c.k, c.v, table, cu, totals, 2, 40)
    for a, b in ((0, 2048), (2048, n)):
        cache_attention(c.q, c.k, c.v, table[a:b], cu[a:b + 1], totals[a:b], 2, 40, out=out, status=status)
    assert status.item() == 0 and (out[int(c.cu[-1]):] == 3.0).all()
    for a in (0, 1500, 2040, 2900):  # the same rows from a call of their own
        b = min(a + 100, n)
        alone = cache_attention(c.q, c.k, c.v, table[a:b], cu[a:b + 1], totals[a:b], 2, 40)
        x, y = int(c.cu[a]), int(c.cu[b])
        assert torch.equal(alone[x:y], out[x:y])


# ------------------------------------------------------------------------------------------------ overlapping buffers
def test_plan_refuses_buffers_that_overlap(cuda_device):
    cached, new, table, free = ints([3, 4]), ints([2, 0]), ints([[0, -1], [1, -1]]), ints([5, 6])
    p = cache_plan(cached, new, table, free, 16, 4)
    for bad in (p._replace(total=cached), p._replace(total=new), p._replace(slots=p.positions),
                p._replace(slots=table.view(-1)), p._replace(counts=free)):
        with pytest.raises(Exception, match="overlap"):
            cache_plan(cached, new, table, free, 16, 4, out=bad)
    with pytest.raises(Exception, match="overlap"):
        cache_plan(p.total, new, table, free, 16, 4, out=p)
    with pytest.raises(Exception, match="overlap"):
        cache_plan(cached, cached, table, table.view(-1)[2:], 16, 4)
    cache_plan(cached, cached, table, free, 16, 4)  # inputs may be the same
    one = ints(np.zeros(3 + 2 + 4 + 4 + 2))  # results side by side in one buffer
    q = type(p)(*torch.split(one, [3, 2, 4, 4, 2]))
    assert torch.equal(cache_plan(cached, new, table, free, 16, 4, out=q).positions, p.positions)


def test_append_refuses_buffers_that_overlap(cuda_device):
    dt, i = torch.float16, ints([0, 1, 2])
    qkv = torch.randn(3, 1, 256, device="cuda").to(dt)
    k = torch.zeros(2, 1, 16, 64, dtype=dt, device="cuda")
    v = torch.zeros_like(k)
    call = lambda **kw: cache_append(**{**dict(qkv=qkv, positions=i, slots=i, k_pages=k, v_pages=v, heads=2, kv_heads=1,  # noqa: E731
                                               freqs=None), **kw})
    for bad in (dict(v_pages=k), dict(q=qkv[:, 0, 64:192].view(3, 2, 64)), dict(q=k.view(-1)[:384].view(3, 2, 64)),
                dict(q=qkv.view(-1)[:384].view(3, 2, 64))):
        with pytest.raises(Exception, match="overlap"):
            call(**bad)
    # q of a row over the row's own q, and beside it
    freqs = torch.from_numpy(FREQS).cuda()
    want = call(freqs=freqs)[0].clone()
    kept_k, kept_v = k.clone(), v.clone()
    wide = torch.zeros(3, 1, 384, dtype=dt, device="cuda")
    wide[..., :256] = qkv
    call(qkv=wide[..., :256], q=wide[:, 0, 256:].view(3, 2, 64), freqs=freqs)
    assert torch.equal(wide[:, 0, 256:].reshape(3, 2, 64), want) and torch.equal(wide[..., :256], qkv)
    call(q=qkv[:, 0, :128].view(3, 2, 64), freqs=freqs)
    assert torch.equal(qkv[:, 0, :128].reshape(3, 2, 64), want)
    assert torch.equal(k, kept_k) and torch.equal(v, kept_v) and torch.equal(wide[..., 128:256], qkv[..., 128:])


def test_attention_refuses_buffers_that_overlap(cuda_device):
    c = Case("fp16", [3], [20], 2, 2, 16)
    wide = torch.zeros(3, 6, 64, dtype=c.dtype, device="cuda")
    wide[:, 1:3] = c.q
    want = c.run().clone()
    flat = wide.view(-1)
    c.q = wide[:, 1:3]
    for bad in (c.q, wide[:, 2:4], wide[:, 0:2], flat[64:64 + 384].view(3, 2, 64), c.k.view(-1)[:384].view(3, 2, 64),
                c.v.view(-1)[-384:].view(3, 2, 64)):
        with pytest.raises(Exception, match="overlap"):
            c.run(bad)
    assert torch.equal(c.run(wide[:, 3:5]), want)  # beside q in the same rows
