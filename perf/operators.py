"""Cases and plain forms of the frame-cache operators: the K/V cache of live input, in pages.

A live stream's time attention keeps the keys and values of the frames it has already heard in fixed-size pages
of a common pool; each push brings a few new frames per stream. Three operators serve a push:

* ``plan``: from each stream's cached and new length, the pages it still needs (taken from a free list, entered in
  its block table), and for every new frame its position and its slot in the pool;
* ``append``: rotary q, and rotary k and plain v written to the frames' slots, from the rows of the qkv product;
* ``attention``: the new frames over everything their stream has cached, softmax exact, gated per head.

A token of the cache is one frame; its heads are all bands' heads (62 bands x 8 heads = 496 in the shipped model),
head dim 64. ``run`` computes the plain forms from elementary torch operations, or makes the package's calls where
``own`` is set.
"""

import math

import numpy as np
import torch

own = False

DIM = 64  # head dimension
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
FREE_SPARE = 7  # pages of the free list that a plan leaves over


def listed():
    plan = {"op": "plan"}
    app = {"op": "append"}
    att = {"op": "attention"}
    return [
        # eight live streams push 0.1 s (10 frames) each, 17 s cached: a call's latency
        {"name": "plan_push", **plan, "seqs": 8, "new": 10, "cached": 1700, "page": 64, "pad": 0},
        # a service's songs admitted together: thousands of ragged sequences, small pages, padded to a capacity
        {"name": "plan_service", **plan, "seqs": 4001, "new": 511, "cached": 1700, "page": 16, "pad": 4099},
        # one stream, one frame of the shipped model (62 bands x 8 heads with gates): a call's latency
        {"name": "append_frame", **app, "dtype": "fp16", "tokens": 1, "bands": 62, "heads": 8, "kv_heads": 8,
         "page": 64, "far": 1700, "gates": True, "pad": 0},
        # grouped heads without gates at far positions (a stream that has run for hours), padded rows
        {"name": "append_grouped_far", **app, "dtype": "bf16", "tokens": 4097, "bands": 1, "heads": 32, "kv_heads": 8,
         "page": 16, "far": 5000000, "gates": False, "pad": 95},
        # a whole 17 s chunk enters the cache
        {"name": "append_chunk", **app, "dtype": "fp16", "tokens": 1700, "bands": 62, "heads": 8, "kv_heads": 8,
         "page": 64, "far": 1700, "gates": True, "pad": 0},
        # the first frames of two streams, one band's heads: a call's latency
        {"name": "attn_start", **att, "dtype": "fp16", "seqs": 2, "heads": 8, "kv_heads": 8, "new": 1, "cached": 40,
         "ragged": True, "page": 16, "causal": True, "window": 0, "gates": False, "pad": 0},
        # one stream, one new frame over 17 s, all bands
        {"name": "attn_frame", **att, "dtype": "fp16", "seqs": 1, "heads": 496, "kv_heads": 496, "new": 1,
         "cached": 1700, "ragged": False, "page": 64, "causal": True, "window": 0, "gates": True, "pad": 0},
        # five streams push up to 0.1 s each, the model's 17 s window, ragged
        {"name": "attn_push", **att, "dtype": "fp16", "seqs": 5, "heads": 496, "kv_heads": 496, "new": 10,
         "cached": 1999, "ragged": True, "page": 32, "causal": False, "window": 1700, "gates": True, "pad": 3},
        # one frame over a very long cache and few heads: the work is along the keys
        {"name": "attn_long", **att, "dtype": "bf16", "seqs": 1, "heads": 8, "kv_heads": 8, "new": 1,
         "cached": 300000, "ragged": False, "page": 128, "causal": True, "window": 0, "gates": False, "pad": 0},
        # pushes of a second (100 frames) over 17 s, all bands
        {"name": "attn_second", **att, "dtype": "fp16", "seqs": 2, "heads": 496, "kv_heads": 496, "new": 100,
         "cached": 1600, "ragged": False, "page": 64, "causal": False, "window": 0, "gates": True, "pad": 0},
        # single frames and long chunks in one batch, grouped heads, causal, small pages
        {"name": "attn_mixed", **att, "dtype": "bf16", "seqs": 13, "heads": 32, "kv_heads": 8, "new": 700,
         "cached": 2500, "ragged": True, "page": 16, "causal": True, "window": 0, "gates": False, "pad": 61},
        # a whole chunk with nothing cached: the time attention of one 17 s chunk
        {"name": "attn_chunk", **att, "dtype": "fp16", "seqs": 1, "heads": 496, "kv_heads": 496, "new": 1701,
         "cached": 0, "ragged": False, "page": 64, "causal": False, "window": 0, "gates": True, "pad": 0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    pad = rng.choice([0, 0, rng.randint(1, 200)])
    while op == "plan":
        case = {"op": op, "seqs": _spread(rng, 1, 4096), "new": _spread(rng, 1, 2000), "cached": _spread(rng, 1, 20000),
                "page": page, "pad": pad}
        if case["seqs"] * case["new"] <= 2000000 and case["seqs"] * (case["cached"] + case["new"]) // page <= 2000000:
            return case
    dtype = rng.choice(["fp16", "bf16"])
    while op == "append":
        bands, group = rng.choice([(1, 1), (1, 4), (62, 1), (60, 1), (1, 7)])
        kv = rng.choice([1, 2, 8, 8])
        case = {"op": op, "dtype": dtype, "tokens": _spread(rng, 1, 8000), "bands": bands, "heads": kv * group,
                "kv_heads": kv, "page": page, "far": _spread(rng, 1, 10000000), "gates": rng.random() < 0.5, "pad": pad}
        if case["tokens"] * bands * (case["heads"] + 2 * kv) <= 1700 * 62 * 24:
            return case
    while True:
        kv = rng.choice([1, 2, 8, 8, 60, 62, 496])
        group = rng.choice([1, 1, 1, 2, 4, 5, 8]) if kv <= 8 else 1
        case = {"op": op, "dtype": dtype, "seqs": _spread(rng, 1, 64), "heads": kv * group, "kv_heads": kv,
                "new": _spread(rng, 1, 2000), "cached": rng.choice([0, 1, 1, 1, 1]) * _spread(rng, 1, 200000),
                "ragged": rng.random() < 0.6, "page": page, "causal": rng.random() < 0.6,
                "window": rng.choice([0, 0, 0, _spread(rng, 1, 4000)]), "gates": rng.random() < 0.5, "pad": pad}
        longest = case["cached"] + case["new"]
        if (case["seqs"] * case["heads"] * case["new"] * longest <= 700000000
                and case["seqs"] * longest * kv <= 5000000):
            return case


def _lengths(case):
    """(cached, new) of each sequence as int64 arrays: they go with the case, whatever the seed. Ragged ones hold
    lengths down to none; the first sequence has the longest of both."""
    n, new, cached = case["seqs"], case["new"], case["cached"]
    if case["op"] == "attention" and not case["ragged"]:
        return np.full(n, cached, np.int64), np.full(n, new, np.int64)
    r = np.random.default_rng([n, new, cached, case["page"]])
    c, q = r.integers(0, cached + 1, n), r.integers(0, new + 1, n)
    if case["op"] == "attention":
        q = np.where(r.random(n) < 0.4, np.minimum(q, 1), q)  # single frames among the chunks
    c[0], q[0] = cached, new
    return c.astype(np.int64), q.astype(np.int64)


def _tables(total, page, pages):
    """Block tables of `total` lengths from a list of page numbers, -1 where a sequence has no page."""
    need = -(-total // page)
    table = np.full((len(total), max(1, int(need.max()))), -1, np.int32)
    start = np.cumsum(need) - need
    k = np.arange(table.shape[1])
    live = k[None, :] < need[:, None]
    table[live] = pages[(start[:, None] + k[None, :])[live]]
    return table


def _normal(shape, dtype, generator):
    return torch.randn(shape, device="cuda", dtype=torch.float32, generator=generator).to(dtype)


def _on_gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    page, s = case["page"], {"case": case}
    if case["op"] == "plan":
        cached, new = _lengths(case)
        held, need = -(-cached // page), -(-(cached + new) // page)
        pages = r.permutation(int(need.sum()) + FREE_SPARE).astype(np.int32)
        table = _tables(cached, page, pages)
        wide = np.full((len(cached), max(1, int(need.max()))), -1, np.int32)
        wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
        s.update(cached=_on_gpu(cached.astype(np.int32)), new=_on_gpu(new.astype(np.int32)), table=_on_gpu(wide),
                 free=_on_gpu(pages[int(held.sum()):]), capacity=int(new.sum()) + case["pad"])
        return s
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "append":
        n, bands, heads, kv = case["tokens"] + case["pad"], case["bands"], case["heads"], case["kv_heads"]
        width = (heads + 2 * kv) * DIM + (-(-heads // 8) * 8 if case["gates"] else 0)
        n_pages = -(-n // page) + 1
        # consecutive frames of one stream that ends at frame `far`, in pages anywhere in the pool
        pos = np.maximum(0, case["far"] - case["tokens"]) + np.arange(n)
        slots = r.permutation(n_pages)[np.arange(n) // page] * page + np.arange(n) % page
        slots[case["tokens"]:], pos[case["tokens"]:] = -1, 0
        s.update(qkv=_normal((n, bands, width), dtype, g), positions=_on_gpu(pos.astype(np.int32)),
                 slots=_on_gpu(slots.astype(np.int32)), k=_normal((n_pages, bands * kv, page, DIM), dtype, g),
                 v=_normal((n_pages, bands * kv, page, DIM), dtype, g),
                 q=torch.zeros(n, bands * heads, DIM, device="cuda", dtype=dtype),
                 gates=torch.zeros(n, bands * heads, device="cuda") if case["gates"] else None,
                 freqs=_on_gpu((10000.0 ** (-np.arange(0, DIM, 2) / DIM)).astype(np.float32)))
        return s
    cached, new = _lengths(case)
    total = cached + new
    n, heads, kv = int(new.sum()) + case["pad"], case["heads"], case["kv_heads"]
    n_pages = int((-(-total // page)).sum()) + 3
    s.update(q=_normal((n, heads, DIM), dtype, g), k=_normal((n_pages, kv, page, DIM), dtype, g),
             v=_normal((n_pages, kv, page, DIM), dtype, g),
             table=_on_gpu(_tables(total, page, r.permutation(n_pages).astype(np.int32))),
             cu=_on_gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), total=_on_gpu(total.astype(np.int32)),
             max_new=int(new.max()), max_total=int(total.max()),
             gates=torch.sigmoid(torch.randn(n, heads, device="cuda", generator=g)) if case["gates"] else None,
             out=torch.zeros(n, heads, DIM, device="cuda", dtype=dtype))
    return s


def run(state):
    return {"plan": _plan, "append": _append, "attention": _attention}[state["case"]["op"]](state)


def _plan(s):
    page, cached, new, table, free, n = s["case"]["page"], s["cached"], s["new"], s["table"], s["free"], s["capacity"]
    if own:
        from turbo_roformer_b200 import cache_plan

        p = cache_plan(cached, new, table, free, page, n)
        return {"table": table, "cu": p.cu, "total": p.total, "slots": p.slots, "positions": p.positions,
                "taken": p.counts[0]}
    total = cached + new
    held, need = (cached + page - 1) // page, (total + page - 1) // page
    extra = need - held
    before = torch.cumsum(extra, 0) - extra
    column = torch.arange(table.shape[1], device="cuda")
    k = column[None, :] - held[:, None]
    fresh = (k >= 0) & (column[None, :] < need[:, None])
    table = torch.where(fresh, free[(before[:, None] + k).clamp(0, len(free) - 1)], table)
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0, dtype=torch.int32)])
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], row, right=True).clamp(max=len(new) - 1)
    live = row < cu[-1]
    pos = torch.where(live, cached[seq] + row - cu[seq], 0)
    slots = torch.where(live, table[seq, pos // page] * page + pos % page, -1)
    return {"table": table, "cu": cu, "total": total, "slots": slots, "positions": pos,
            "taken": extra.sum(dtype=torch.int32)}


def _append(s):
    c, qkv, k_pages, v_pages, gates = s["case"], s["qkv"], s["k"], s["v"], s["gates"]
    bands, heads, kv, page = c["bands"], c["heads"], c["kv_heads"], c["page"]
    if own:
        from turbo_roformer_b200 import cache_append

        cache_append(qkv, s["positions"], s["slots"], k_pages, v_pages, heads, kv, freqs=s["freqs"], q=s["q"],
                     gates=gates)
        return {"q": s["q"], "k": k_pages, "v": v_pages, "gates": gates}
    n, dtype = len(qkv), qkv.dtype
    x = qkv.float()
    angle = s["positions"].double()[:, None] * s["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, None, None], torch.sin(angle).float()[:, None, None]
    rows = x[..., : (heads + kv) * DIM].reshape(n, bands, heads + kv, DIM // 2, 2)
    a, b = rows[..., 0], rows[..., 1]
    rotated = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).reshape(n, bands, heads + kv, DIM).to(dtype)
    live = s["slots"] >= 0
    slot = s["slots"][live].long()
    s["q"][live] = rotated[:, :, :heads].reshape(n, bands * heads, DIM)[live]
    k_pages[slot // page, :, slot % page] = rotated[:, :, heads:].reshape(n, bands * kv, DIM)[live]
    value = qkv[..., (heads + kv) * DIM: (heads + 2 * kv) * DIM].reshape(n, bands * kv, DIM)
    v_pages[slot // page, :, slot % page] = value[live]
    if gates is not None:
        at = (heads + 2 * kv) * DIM
        gates[live] = (1 / (1 + torch.exp(-x[..., at: at + heads]))).reshape(n, bands * heads)[live]
    return {"q": s["q"], "k": k_pages, "v": v_pages, "gates": gates}


def _attention(s):
    c, q, table, cu, total, gates, out = s["case"], s["q"], s["table"], s["cu"], s["total"], s["gates"], s["out"]
    page, heads, kv, causal, window = c["page"], c["heads"], c["kv_heads"], c["causal"], c["window"]
    if own:
        from turbo_roformer_b200 import cache_attention

        return cache_attention(q, s["k"], s["v"], table, cu, total, s["max_new"], s["max_total"], causal=causal,
                               window=window, gates=gates, out=out)
    cu, total = cu.long(), total.long()
    new = cu[1:] - cu[:-1]
    i, j = torch.arange(s["max_new"], device="cuda"), torch.arange(s["max_total"], device="cuda")
    # queries padded to (sequence, new frame), keys to (sequence, frame)
    row = (cu[:-1, None] + i).clamp(max=len(q) - 1)
    query = q[row].float().permute(0, 2, 1, 3)  # (sequence, head, new frame, 64)
    at = table[:, j // page].long().clamp(min=0)
    known = j < total[:, None]
    key = s["k"][at, :, j % page].float().permute(0, 2, 1, 3)
    value = torch.where(known[:, :, None, None], s["v"][at, :, j % page].float(), 0).permute(0, 2, 1, 3)
    n, g = len(new), heads // kv
    score = query.reshape(n, kv, g * len(i), DIM) @ key.transpose(2, 3) * 0.125
    score = score.reshape(n, heads, len(i), len(j))
    pos = (total - new)[:, None] + i
    seen = known[:, None, :].expand(-1, len(i), -1)
    if causal:
        seen = seen & (j <= pos[:, :, None])
    if window:
        seen = seen & (j > pos[:, :, None] - window)
    score = score.masked_fill(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    norm = p.sum(-1, keepdim=True)
    answer = p.reshape(n, kv, g * len(i), len(j)) @ value
    answer = answer.reshape(n, heads, len(i), DIM) / torch.where(norm == 0, 1, norm)
    live = i < new[:, None]
    answer = answer.permute(0, 2, 1, 3)[live]  # the rows in their order
    if gates is not None:
        answer = answer * gates[: len(answer), :, None]
    out[: len(answer)] = answer.to(out.dtype)
    return out


def _visible(case):
    """Per sequence: (query, key) pairs that the masks leave, and keys that some query sees."""
    pairs = keys = 0
    for cached, new in zip(*_lengths(case)):
        total = cached + new
        pos = cached + np.arange(new)
        hi = np.minimum(total, pos + 1) if case["causal"] else np.full(new, total)
        lo = np.maximum(0, pos - case["window"] + 1) if case["window"] else np.zeros(new, np.int64)
        pairs += int(np.maximum(0, hi - lo).sum())
        keys += int(hi.max() - lo.min()) if new else 0
    return pairs, keys


def work(case):
    page = case["page"]
    if case["op"] == "plan":
        cached, new = _lengths(case)
        taken = int((-(-(cached + new) // page) + cached // -page).sum())
        n = len(cached)
        # lengths in and out, offsets, the last held page's entry, each fresh page read and entered, slot and position
        return {"bytes": 4 * (2 * n + 2 * n + 1 + n + 2 * taken) + 8 * (int(new.sum()) + case["pad"]), "flops": 0}
    if case["op"] == "append":
        n, bands, heads, kv = case["tokens"], case["bands"], case["heads"], case["kv_heads"]
        gates = n * bands * heads * 6 if case["gates"] else 0
        return {"bytes": 2 * 2 * n * bands * (heads + 2 * kv) * DIM + gates + 8 * (n + case["pad"]),
                "flops": 3 * n * bands * (heads + kv) * DIM}
    pairs, keys = _visible(case)
    rows, heads = int(_lengths(case)[1].sum()), case["heads"]
    return {"bytes": 2 * 2 * rows * heads * DIM + 2 * 2 * keys * case["kv_heads"] * DIM + 4 * keys // page
            + (4 * rows * heads if case["gates"] else 0), "flops": 4 * DIM * pairs * heads}


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention}[case["op"]](s)


def _exact_plan(s):
    page, table = s["case"]["page"], s["table"].cpu().numpy()
    cached, new, free = (s[k].cpu().tolist() for k in ("cached", "new", "free"))
    slots, positions, cu, taken = [], [], [0], 0
    for i, (c, n) in enumerate(zip(cached, new)):
        for column in range(-(-c // page), -(-(c + n) // page)):
            table[i, column] = free[taken]
            taken += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(int(table[i, p // page]) * page + p % page)
        cu.append(cu[-1] + n)
    spare = s["capacity"] - len(slots)
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"table": torch.from_numpy(table), "cu": ints(cu), "total": ints([c + n for c, n in zip(cached, new)]),
            "slots": ints(slots + [-1] * spare), "positions": ints(positions + [0] * spare), "taken": ints(taken)}


def _exact_append(s):
    c = s["case"]
    n, bands, heads, kv = c["tokens"], c["bands"], c["heads"], c["kv_heads"]
    x = s["qkv"][:n].double()
    turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64),
                       s["positions"][:n].double()[:, None] * s["freqs"].double())[:, None, None, :]
    rotate = lambda y: torch.view_as_real(torch.view_as_complex(  # noqa: E731
        y.reshape(n, bands, -1, DIM // 2, 2).contiguous()) * turn).reshape(n, -1, DIM)
    parts = torch.split(x, [heads * DIM, kv * DIM, kv * DIM, x.shape[-1] - (heads + 2 * kv) * DIM], -1)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    q[:n] = rotate(parts[0])
    slot = s["slots"][:n].long()
    block = torch.arange(bands * kv, device="cuda")
    k[slot[:, None] // c["page"], block, slot[:, None] % c["page"]] = rotate(parts[1])
    v[slot[:, None] // c["page"], block, slot[:, None] % c["page"]] = parts[2].reshape(n, -1, DIM)
    gates = None
    if s["gates"] is not None:
        gates = s["gates"].double()
        gates[:n] = torch.special.expit(parts[3][..., :heads]).reshape(n, -1)
    return {"q": q, "k": k, "v": v, "gates": gates}


def _exact_attention(s):
    c, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    cu, totals = s["cu"].tolist(), s["total"].tolist()
    out = s["out"].double()
    for i, total in enumerate(totals):
        a, b = cu[i], cu[i + 1]
        if a == b or not total:
            continue
        pages = s["table"][i, : -(-total // c["page"])].long()
        for h in range(0, c["kv_heads"], 31):
            h1 = min(h + 31, c["kv_heads"])
            k, v = (s[x][pages, h:h1].double().transpose(0, 1).reshape(h1 - h, -1, DIM)[:, :total] for x in "kv")
            for r0 in range(a, b, 512):
                r1 = min(r0 + 512, b)
                q = s["q"][r0:r1, h * group: h1 * group].double().transpose(0, 1)
                score = torch.einsum("hqd,hkd->hqk", q, k.repeat_interleave(group, 0)) / 8
                back = (total - b + torch.arange(r0, r1, device="cuda"))[:, None] - torch.arange(total, device="cuda")
                hidden = torch.zeros_like(back, dtype=torch.bool)
                if c["causal"]:
                    hidden |= back < 0
                if c["window"]:
                    hidden |= back >= c["window"]
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                p = p.masked_fill(hidden.all(-1, keepdim=True), 0)  # a row that sees nothing
                y = torch.einsum("hqk,hkd->qhd", p, v.repeat_interleave(group, 0))
                if s["gates"] is not None:
                    y *= s["gates"][r0:r1, h * group: h1 * group, None].double()
                out[r0:r1, h * group: h1 * group] = y
    return out
