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
nonzero code when a kernel met a bad page or slot number, or lengths that do not fit the rows or the table; the plan's
flags are in ``counts[1]``.

There is no backward pass: a tensor that requires grad is refused unless gradients are off (``torch.no_grad``).
Tensors are checked (``ValueError``), results allocated and the library called in the extension module
``_cache_binding`` (``csrc/cache_binding.cpp``), because a push's kernels are shorter than these take in Python.
"""

from __future__ import annotations

import ctypes
import importlib.util
import threading
from typing import NamedTuple

import torch

from . import _build, _lib


class CachePlan(NamedTuple):
    """What ``cache_plan`` writes, int32 on the device (``include/trcuda.h``, trc_cache_plan)."""

    cu: torch.Tensor         # (sequences + 1,) first row of each sequence
    total: torch.Tensor      # (sequences,) frames in the cache once the new ones are appended
    slots: torch.Tensor      # (max_rows,) slot of each row, -1 for none
    positions: torch.Tensor  # (max_rows,) frame number of each row
    counts: torch.Tensor     # (2,) pages taken from the free list; TRC_CACHE_* flags, 0 for none


_lock = threading.Lock()
_binding = None


def _load():
    """The extension module, built if it is missing, with the library's entry points."""
    global _binding
    lib = _lib.load()
    with _lock:
        if _binding is None:
            try:
                spec = importlib.util.spec_from_file_location("_cache_binding", _build.build_binding())
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
            except Exception as e:  # no compiler, or built for another torch
                raise _lib.KernelUnavailable(str(e)) from e
            at = lambda fn: ctypes.cast(fn, ctypes.c_void_p).value  # noqa: E731
            module.bind(at(lib.trc_cache_plan), at(lib.trc_cache_append), at(lib.trc_cache_workspace),
                        at(lib.trc_cache_attention), _lib.check)
            _binding = module
        return _binding


def cache_plan(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page: int,
               max_rows: int, out: CachePlan | None = None) -> CachePlan:
    """Pages, slots and positions of a push: ``cached`` and ``new`` (sequences,) int32 frames each sequence has and
    gets. Sequences take the pages they lack from the front of ``free_pages`` into ``table`` (sequences, columns),
    in place; ``max_rows`` is the capacity of the per-row outputs. ``out``: a plan to write into; its ``total`` is not
    ``cached`` (kept lengths are advanced by ``cached += new`` after the push)."""
    r = (_binding or _load()).plan(cached, new, table, free_pages, page, max_rows, out)
    return r if r is out else CachePlan._make(r)


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
    are undefined. Rows that name the same slot leave it undefined. What is written overlaps no other argument; only
    with one band may ``q`` be the q of ``qkv`` itself."""
    return (_binding or _load()).append(qkv, positions, slots, k_pages, v_pages, heads, kv_heads, freqs, q, gates,
                                        status)


def cache_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    cu: torch.Tensor, total: torch.Tensor, max_new: int, max_total: int, *, causal: bool = True,
                    window: int = 0, scale: float = 0.125, gates: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new frames over their sequences' pages: ``q`` (rows, heads, 64) packed as ``cu`` says,
    against frames 0 .. total[i] - 1 of each sequence, the new ones being the last. ``causal``: a frame sees none
    after it; ``window`` > 0: only that many up to itself. ``gates`` (rows, heads) fp32 scale the result, which is
    zero for a frame that sees nothing. ``max_new`` / ``max_total``: the longest new part and total as far as the
    host knows; they choose the kernel variant only. At most 2,048 sequences: of a longer plan, calls take slices
    ``table[a:b]``, ``cu[a:b + 1]``, ``total[a:b]`` with the same ``q`` and ``out``. ``out``: where to write (not over
    another argument); otherwise a new tensor, undefined in rows behind the last sequence's.

    Weights are rounded to the 16-bit type for the product with v; scores, sums and norms are fp32. A NaN or +inf
    score makes its row NaN. A v that is not finite may also make NaN of rows that a mask hides it from, where other
    rows of their push see it."""
    return (_binding or _load()).attention(q, k_pages, v_pages, table, cu, total, max_new, max_total, causal, window,
                                           scale, gates, out, status)
