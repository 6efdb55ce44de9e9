"""The frame cache of live input: keys and values of heard frames in pages, and attention over them.

The reference recomputes a whole chunk for every forward (turbo_roformer/fast.py:269-341: qkv, rope_pack,
attention); it has no cache. For streams whose new frames look back over what was heard, a push of a few frames
per stream takes three calls, all on the tensors' device and its current stream, without host synchronisation:

* ``cache_plan`` (``trc_cache_plan``): block tables, slots and positions from the streams' lengths;
* ``cache_append`` (``trc_cache_append``): ``rope_pack`` into the pages;
* ``cache_attention`` (``trc_cache_attention``): ``attention`` of the new frames over the pages.

Layouts are those of ``include/trcuda.h``: pools (pages, cache heads, page, 64), a frame's heads being all bands'
heads; rows of all streams packed one behind the other; rows behind the last one are left as they were. Each call
can be captured in a CUDA graph. ``status`` (an int32 tensor of one element, zeroed by the caller) receives a
nonzero code when a kernel met a bad page or slot number; the plan's flags are in ``counts[1]``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

HEAD_DIM = 64
PAGES = (16, 32, 64, 128)
_PRECISION = {torch.float16: _lib.TRC_PREC_FP16, torch.bfloat16: _lib.TRC_PREC_BF16}
_INT32_MAX = 2**31 - 1


class CachePlan(NamedTuple):
    """What ``cache_plan`` writes, int32 on the device (``include/trcuda.h``, trc_cache_plan)."""

    cu: torch.Tensor         # (sequences + 1,) first row of each sequence
    total: torch.Tensor      # (sequences,) frames in the cache once the new ones are appended
    slots: torch.Tensor      # (max_rows,) slot of each row, -1 for none
    positions: torch.Tensor  # (max_rows,) frame number of each row
    counts: torch.Tensor     # (2,) pages taken from the free list; TRC_CACHE_* flags, 0 for none


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t: torch.Tensor, device: torch.device, ndim: int, name: str) -> None:
    if t.dtype != torch.int32 or t.device != device or t.ndim != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {ndim}-d int32 tensor on {device}")


def _status_ptr(status: torch.Tensor | None, device: torch.device) -> int:
    if status is None:
        return 0
    if status.dtype != torch.int32 or status.device != device or status.numel() != 1:
        raise ValueError(f"status must be an int32 tensor of one element on {device}")
    return status.data_ptr()


def _call(device: torch.device, fn: str, *args) -> None:
    """fn(*args, stream) with `device` current (it is set and put back only where another one is)."""
    lib = _lib.load()
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = getattr(lib, fn)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, fn)(*args, stream)
    if rc:
        _lib.check(rc)


def _pools(k: torch.Tensor, v: torch.Tensor, device: torch.device, dtype: torch.dtype) -> tuple[int, int, int]:
    """(pages, cache heads, frames per page) of a pool pair."""
    if k.ndim != 4 or k.shape != v.shape or k.shape[3] != HEAD_DIM or k.shape[2] not in PAGES:
        raise ValueError("pools must be (pages, cache heads, 16 | 32 | 64 | 128, 64), k and v alike")
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
        raise ValueError(f"pools must be {dtype} on {device}")
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("pools must be contiguous")
    return k.shape[0], k.shape[1], k.shape[2]


def _row_stride(t: torch.Tensor, shape: tuple[int, int, int], device: torch.device, dtype: torch.dtype,
                name: str) -> int:
    """Elements between rows of a (rows, heads, 64) tensor whose rows are contiguous."""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {shape} {dtype} on {device}")
    st = t.stride()
    if st[2] != 1 or (shape[1] > 1 and st[1] != HEAD_DIM):
        raise ValueError(f"{name}: a row's heads must be contiguous")
    return st[0] if shape[0] > 1 else shape[1] * HEAD_DIM


def cache_plan(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page: int,
               max_rows: int, out: CachePlan | None = None) -> CachePlan:
    """Pages, slots and positions of a push: ``cached`` and ``new`` (sequences,) int32 frames each sequence has and
    gets. Sequences take the pages they lack from the front of ``free_pages`` into ``table`` (sequences, columns),
    in place; ``max_rows`` is the capacity of the per-row outputs. ``out``: a plan to write into."""
    device = cached.device
    _need(cached.is_cuda, "cached must be a CUDA tensor")
    _ints(cached, device, 1, "cached")
    _ints(new, device, 1, "new")
    _ints(table, device, 2, "table")
    _ints(free_pages, device, 1, "free_pages")
    n = cached.shape[0]
    _need(new.shape[0] == n and table.shape[0] == n, "cached, new and table must agree in the number of sequences")
    _need(page in PAGES, f"page must be one of {PAGES}")
    _need(0 <= max_rows <= _INT32_MAX, "max_rows out of range")
    if out is None:
        # one allocation, the arrays on 16-byte boundaries
        sizes = (n + 1, n, max_rows, max_rows, 2)
        up = [(x + 3) & ~3 for x in sizes]
        out = CachePlan(*(p[:x] for p, x in zip(torch.empty(sum(up), dtype=torch.int32, device=device).split(up),
                                                sizes)))
    else:
        for t, size, name in zip(out, (n + 1, n, max_rows, max_rows, 2), CachePlan._fields):
            _ints(t, device, 1, name)
            _need(t.shape[0] == size, f"{name} must have {size} elements")
    _call(device, "trc_cache_plan", cached.data_ptr(), new.data_ptr(), n, page, free_pages.data_ptr(),
          free_pages.shape[0], table.data_ptr(), table.shape[1], max_rows, out.cu.data_ptr(), out.total.data_ptr(),
          out.slots.data_ptr(), out.positions.data_ptr(), out.counts.data_ptr())
    return out


def cache_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, heads: int, kv_heads: int, *, freqs: torch.Tensor | None,
                 q: torch.Tensor | None = None, gates: torch.Tensor | bool | None = None,
                 status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary q, and rotary k and plain v into the pages, from rows of the qkv product.

    ``qkv`` (rows, bands, width), fp16 or bf16, a band's elements contiguous: heads * 64 of q, kv_heads * 64 of k,
    kv_heads * 64 of v, then ``heads`` gate logits where gates are wanted. ``freqs`` (32,) fp32: the rotary
    frequencies (the checkpoint's ``rotary_embed.freqs``), None for no rotation. Returns q (rows, bands * heads,
    64) and the sigmoid gates (rows, bands * heads) fp32, or None; ``q`` and ``gates`` may be tensors to write into
    (``gates=True``: a new one). Rows whose slot is -1 are skipped: where q and gates are new, their values there
    are undefined."""
    device, dtype = qkv.device, qkv.dtype
    _need(qkv.is_cuda and qkv.ndim == 3 and dtype in _PRECISION, "qkv must be a (rows, bands, width) fp16 or bf16 CUDA tensor")
    rows, bands, width = qkv.shape
    _need(heads >= 1 and kv_heads >= 1 and heads % kv_heads == 0, "kv_heads must divide heads")
    n_pages, cache_heads, page = _pools(k_pages, v_pages, device, dtype)
    _need(bands >= 1 and cache_heads == bands * kv_heads, "the pools must have bands * kv_heads cache heads")
    wanted = gates is not None and gates is not False
    _need(width >= (heads + 2 * kv_heads) * HEAD_DIM + (heads if wanted else 0), "qkv rows too short")
    _need(qkv.stride(2) == 1, "qkv: a band's elements must be contiguous")
    _ints(positions, device, 1, "positions")
    _ints(slots, device, 1, "slots")
    _need(positions.shape[0] >= rows and slots.shape[0] >= rows, "positions and slots must cover the rows")
    if freqs is not None:
        _need(freqs.dtype == torch.float32 and freqs.device == device and freqs.shape == (HEAD_DIM // 2,)
              and freqs.is_contiguous(), f"freqs must be 32 float32 on {device}")
    shape = (rows, bands * heads, HEAD_DIM)
    if q is None:
        q = torch.empty(shape, dtype=dtype, device=device)
    if gates is True:
        gates = torch.empty(shape[:2], dtype=torch.float32, device=device)
    elif wanted:
        _need(gates.shape == shape[:2] and gates.dtype == torch.float32 and gates.device == device
              and gates.is_contiguous(), f"gates must be a contiguous {shape[:2]} float32 tensor on {device}")
    else:
        gates = None
    q_stride = _row_stride(q, shape, device, dtype, "q")
    status_ptr = _status_ptr(status, device)
    if rows:
        row_stride = qkv.stride(0) if rows > 1 else 0
        band_stride = qkv.stride(1) if bands > 1 else 0
        _call(device, "trc_cache_append", _PRECISION[dtype], qkv.data_ptr(), row_stride, band_stride, rows, bands,
              heads, kv_heads, positions.data_ptr(), slots.data_ptr(), freqs.data_ptr() if freqs is not None else 0,
              page, n_pages, q.data_ptr(), q_stride, k_pages.data_ptr(), v_pages.data_ptr(),
              gates.data_ptr() if gates is not None else 0, status_ptr)
    return q, gates


_workspace_bytes: dict[tuple[int, int, int, int], int] = {}  # per device and arguments of trc_cache_workspace


def cache_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    cu: torch.Tensor, total: torch.Tensor, max_new: int, max_total: int, *, causal: bool = True,
                    window: int = 0, scale: float = 0.125, gates: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new frames over their sequences' pages: ``q`` (rows, heads, 64) packed as ``cu`` says,
    against frames 0 .. total[i] - 1 of each sequence, the new ones being the last. ``causal``: a frame sees none
    after it; ``window`` > 0: only that many up to itself. ``gates`` (rows, heads) fp32 scale the result, which is
    zero for a frame that sees nothing. ``max_new`` / ``max_total``: the longest new part and total as far as the
    host knows; they choose the kernel variant only. ``out``: where to write; otherwise a new tensor, undefined in
    rows behind the last sequence's."""
    device, dtype = q.device, q.dtype
    _need(q.is_cuda and q.ndim == 3 and dtype in _PRECISION, "q must be a (rows, heads, 64) fp16 or bf16 CUDA tensor")
    rows, heads, _ = shape = tuple(q.shape)
    n_pages, kv_heads, page = _pools(k_pages, v_pages, device, dtype)
    _need(heads >= 1 and shape[2] == HEAD_DIM and heads % kv_heads == 0, "the cache heads must divide q's heads")
    _ints(table, device, 2, "table")
    _ints(cu, device, 1, "cu")
    _ints(total, device, 1, "total")
    n = total.shape[0]
    _need(table.shape[0] == n and cu.shape[0] == n + 1, "table, cu and total must agree in the number of sequences")
    q_stride = _row_stride(q, shape, device, dtype, "q")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
    out_stride = _row_stride(out, shape, device, dtype, "out")
    gates_ptr = 0
    if gates is not None:
        _need(gates.shape == shape[:2] and gates.dtype == torch.float32 and gates.device == device
              and gates.is_contiguous(), f"gates must be a contiguous {shape[:2]} float32 tensor on {device}")
        gates_ptr = gates.data_ptr()
    status_ptr = _status_ptr(status, device)
    if not rows:
        return out
    workspace, size = 0, 0
    if max_total > 512:  # as trc_cache_attention documents
        key = (device.index, max_new, heads, kv_heads)
        size = _workspace_bytes.get(key, 0)
        if not size:
            with torch.cuda.device(device):
                size = _lib.load().trc_cache_workspace(max_new, heads, kv_heads)
            if size < 0:
                _lib.check(size)
            _workspace_bytes[key] = size
        held = torch.empty(size, dtype=torch.uint8, device=device)  # from the current stream's pool
        workspace = held.data_ptr()
    _call(device, "trc_cache_attention", _PRECISION[dtype], q.data_ptr(), q_stride, k_pages.data_ptr(),
          v_pages.data_ptr(), table.data_ptr(), table.shape[1], cu.data_ptr(), total.data_ptr(), n, rows, max_new,
          max_total, heads, kv_heads, page, n_pages, int(causal), window, scale, gates_ptr, out.data_ptr(), out_stride,
          workspace, size, status_ptr)
    return out
