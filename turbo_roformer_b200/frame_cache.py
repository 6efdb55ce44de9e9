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
MAX_WHOLE = 512  # TRC_CACHE_MAX_WHOLE: up to this max_total trc_cache_attention takes no workspace
_INT32_MAX = 2**31 - 1


class CachePlan(NamedTuple):
    """What ``cache_plan`` writes, int32 on the device (``include/trcuda.h``, trc_cache_plan)."""

    cu: torch.Tensor         # (sequences + 1,) first row of each sequence
    total: torch.Tensor      # (sequences,) frames in the cache once the new ones are appended
    slots: torch.Tensor      # (max_rows,) slot of each row, -1 for none
    positions: torch.Tensor  # (max_rows,) frame number of each row
    counts: torch.Tensor     # (2,) pages taken from the free list; TRC_CACHE_* flags, 0 for none


def _ints(t: torch.Tensor, index: int, ndim: int, name: str) -> None:
    if t.dtype is not torch.int32 or t.get_device() != index or t.ndim != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {ndim}-d int32 tensor on cuda:{index}")


def _status_ptr(status: torch.Tensor | None, index: int) -> int:
    if status is None:
        return 0
    if status.dtype is not torch.int32 or status.get_device() != index or status.numel() != 1:
        raise ValueError(f"status must be an int32 tensor of one element on cuda:{index}")
    return status.data_ptr()


def _call(index: int, fn: str, *args) -> None:
    """fn(*args, stream) on device `index` and its current stream (made current only where another device is)."""
    lib = _lib.load()
    # the raw handle of torch.cuda.current_stream(index), without the Stream object around it (a pass's latency)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = getattr(lib, fn)(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = getattr(lib, fn)(*args, stream)
    if rc:
        _lib.check(rc)


def _pools(k: torch.Tensor, v: torch.Tensor, index: int, dtype: torch.dtype) -> tuple[int, int, int]:
    """(pages, cache heads, frames per page) of a pool pair."""
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[3] != HEAD_DIM or shape[2] not in PAGES:
        raise ValueError("pools must be (pages, cache heads, 16 | 32 | 64 | 128, 64), k and v alike")
    if k.dtype is not dtype or v.dtype is not dtype or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"pools must be {dtype} on cuda:{index}")
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("pools must be contiguous")
    return shape[0], shape[1], shape[2]


def _row_stride(t: torch.Tensor, rows: int, heads: int, index: int, dtype: torch.dtype, name: str) -> int:
    """Elements between rows of a (rows, heads, 64) tensor whose rows are contiguous."""
    if t.shape != (rows, heads, HEAD_DIM) or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be ({rows}, {heads}, {HEAD_DIM}) {dtype} on cuda:{index}")
    st = t.stride()
    if st[2] != 1 or (heads > 1 and st[1] != HEAD_DIM):
        raise ValueError(f"{name}: a row's heads must be contiguous")
    return st[0] if rows > 1 else heads * HEAD_DIM


def _gates_ptr(gates: torch.Tensor, rows: int, heads: int, index: int) -> int:
    if (gates.shape != (rows, heads) or gates.dtype is not torch.float32 or gates.get_device() != index
            or not gates.is_contiguous()):
        raise ValueError(f"gates must be a contiguous ({rows}, {heads}) float32 tensor on cuda:{index}")
    return gates.data_ptr()


def cache_plan(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page: int,
               max_rows: int, out: CachePlan | None = None) -> CachePlan:
    """Pages, slots and positions of a push: ``cached`` and ``new`` (sequences,) int32 frames each sequence has and
    gets. Sequences take the pages they lack from the front of ``free_pages`` into ``table`` (sequences, columns),
    in place; ``max_rows`` is the capacity of the per-row outputs. ``out``: a plan to write into."""
    if not cached.is_cuda:
        raise ValueError("cached must be a CUDA tensor")
    index = cached.get_device()
    _ints(cached, index, 1, "cached")
    _ints(new, index, 1, "new")
    _ints(table, index, 2, "table")
    _ints(free_pages, index, 1, "free_pages")
    n = cached.shape[0]
    rows, columns = table.shape
    if new.shape[0] != n or rows != n:
        raise ValueError("cached, new and table must agree in the number of sequences")
    if page not in PAGES:
        raise ValueError(f"page must be one of {PAGES}")
    if not 0 <= max_rows <= _INT32_MAX:
        raise ValueError("max_rows out of range")
    if out is None:
        # one allocation, the slots first: on a 16-byte boundary
        slots, positions, cu, total, counts = cached.new_empty(2 * (max_rows + n) + 3).split_with_sizes(
            (max_rows, max_rows, n + 1, n, 2))
        out = CachePlan(cu, total, slots, positions, counts)
    else:
        for t, size, name in zip(out, (n + 1, n, max_rows, max_rows, 2), CachePlan._fields):
            _ints(t, index, 1, name)
            if t.shape[0] != size:
                raise ValueError(f"{name} must have {size} elements")
        cu, total, slots, positions, counts = out
    _call(index, "trc_cache_plan", cached.data_ptr(), new.data_ptr(), n, page, free_pages.data_ptr(),
          free_pages.shape[0], table.data_ptr(), columns, max_rows, cu.data_ptr(), total.data_ptr(), slots.data_ptr(),
          positions.data_ptr(), counts.data_ptr())
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
    dtype = qkv.dtype
    if not qkv.is_cuda or qkv.ndim != 3 or dtype not in _PRECISION:
        raise ValueError("qkv must be a (rows, bands, width) fp16 or bf16 CUDA tensor")
    index = qkv.get_device()
    rows, bands, width = qkv.shape
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("kv_heads must divide heads")
    n_pages, cache_heads, page = _pools(k_pages, v_pages, index, dtype)
    if bands < 1 or cache_heads != bands * kv_heads:
        raise ValueError("the pools must have bands * kv_heads cache heads")
    wanted = gates is not None and gates is not False
    if width < (heads + 2 * kv_heads) * HEAD_DIM + (heads if wanted else 0):
        raise ValueError("qkv rows too short")
    row_stride, band_stride, one = qkv.stride()
    if one != 1:
        raise ValueError("qkv: a band's elements must be contiguous")
    _ints(positions, index, 1, "positions")
    _ints(slots, index, 1, "slots")
    if positions.shape[0] < rows or slots.shape[0] < rows:
        raise ValueError("positions and slots must cover the rows")
    freqs_ptr = gates_ptr = 0
    if freqs is not None:
        if (freqs.dtype is not torch.float32 or freqs.get_device() != index or freqs.shape != (HEAD_DIM // 2,)
                or not freqs.is_contiguous()):
            raise ValueError(f"freqs must be 32 float32 on cuda:{index}")
        freqs_ptr = freqs.data_ptr()
    if q is None:
        q = qkv.new_empty((rows, bands * heads, HEAD_DIM))
    q_stride = _row_stride(q, rows, bands * heads, index, dtype, "q")
    if wanted:
        if gates is True:
            gates = qkv.new_empty((rows, bands * heads), dtype=torch.float32)
        gates_ptr = _gates_ptr(gates, rows, bands * heads, index)
    else:
        gates = None
    status_ptr = _status_ptr(status, index)
    if rows:
        # strides of dimensions of one element say nothing
        _call(index, "trc_cache_append", _PRECISION[dtype], qkv.data_ptr(), row_stride if rows > 1 else 0,
              band_stride if bands > 1 else 0, rows, bands, heads, kv_heads, positions.data_ptr(), slots.data_ptr(),
              freqs_ptr, page, n_pages, q.data_ptr(), q_stride, k_pages.data_ptr(), v_pages.data_ptr(), gates_ptr,
              status_ptr)
    return q, gates


_workspace_bytes: dict[tuple[int, int, int, int], int] = {}  # by device and arguments of trc_cache_workspace


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
    dtype = q.dtype
    if not q.is_cuda or q.ndim != 3 or dtype not in _PRECISION:
        raise ValueError("q must be a (rows, heads, 64) fp16 or bf16 CUDA tensor")
    index = q.get_device()
    rows, heads, dim = q.shape
    n_pages, kv_heads, page = _pools(k_pages, v_pages, index, dtype)
    if dim != HEAD_DIM or heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("q must have 64 elements per head, and the cache heads must divide its heads")
    _ints(table, index, 2, "table")
    _ints(cu, index, 1, "cu")
    _ints(total, index, 1, "total")
    n, columns = table.shape
    if total.shape[0] != n or cu.shape[0] != n + 1:
        raise ValueError("table, cu and total must agree in the number of sequences")
    q_stride = _row_stride(q, rows, heads, index, dtype, "q")
    if out is None:
        out = q.new_empty((rows, heads, HEAD_DIM))
    out_stride = _row_stride(out, rows, heads, index, dtype, "out")
    gates_ptr = _gates_ptr(gates, rows, heads, index) if gates is not None else 0
    status_ptr = _status_ptr(status, index)
    if not rows:
        return out
    workspace = size = 0
    if max_total > MAX_WHOLE:
        key = (index, max_new, heads, kv_heads)
        size = _workspace_bytes.get(key, 0)
        if not size:
            with torch.cuda.device(index):
                size = _lib.load().trc_cache_workspace(max_new, heads, kv_heads)
            if size < 0:
                _lib.check(size)
            if len(_workspace_bytes) > 4096:
                _workspace_bytes.clear()
            _workspace_bytes[key] = size
        held = q.new_empty(size, dtype=torch.uint8)  # of the current stream's pool: free for later work on it
        workspace = held.data_ptr()
    _call(index, "trc_cache_attention", _PRECISION[dtype], q.data_ptr(), q_stride, k_pages.data_ptr(),
          v_pages.data_ptr(), table.data_ptr(), columns, cu.data_ptr(), total.data_ptr(), n, rows, max_new, max_total,
          heads, kv_heads, page, n_pages, 1 if causal else 0, window, scale, gates_ptr, out.data_ptr(), out_stride,
          workspace, size, status_ptr)
    return out
