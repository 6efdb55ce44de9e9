"""The frame cache and autograd: no backward pass, so no silent result without history, and writes that autograd sees."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from turbo_roformer_b200 import CachePlan, cache_append, cache_attention, cache_plan


def tensors(device):
    half = dict(dtype=torch.float16, device=device)
    i = torch.tensor([0, 1], dtype=torch.int32, device=device)
    append = dict(qkv=torch.zeros(2, 1, 200, **half), positions=i, slots=i, k_pages=torch.zeros(2, 1, 16, 64, **half),
                  v_pages=torch.zeros(2, 1, 16, 64, **half), heads=1, kv_heads=1,
                  freqs=torch.zeros(32, device=device), q=torch.zeros(2, 1, 64, **half),
                  gates=torch.zeros(2, 1, device=device))
    attention = dict(q=torch.zeros(2, 1, 64, **half), k_pages=append["k_pages"], v_pages=append["v_pages"],
                     table=i[:1, None], cu=torch.tensor([0, 2], dtype=torch.int32, device=device),
                     total=torch.tensor([2], dtype=torch.int32, device=device), max_new=2, max_total=2,
                     gates=torch.zeros(2, 1, device=device), out=torch.zeros(2, 1, 64, **half))
    return append, attention


def refused(fn, kw, names):
    for name in names:
        bad = {**kw, name: kw[name].clone().requires_grad_()}
        with pytest.raises(ValueError, match=f"{name} requires grad"):
            fn(**bad)


def test_grad_is_refused_before_the_device():
    append, attention = tensors("cpu")
    refused(cache_append, append, ["qkv"])
    refused(cache_attention, attention, ["q"])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        cache_append(**{**append, "qkv": append["qkv"].clone().requires_grad_()})


@pytest.mark.gpu
def test_grad_is_refused(cuda_device):
    append, attention = tensors("cuda")
    refused(cache_append, append, ["qkv", "k_pages", "v_pages", "freqs", "q", "gates"])
    refused(cache_attention, attention, ["q", "k_pages", "v_pages", "gates", "out"])
    with torch.no_grad():
        cache_append(**{**append, "qkv": append["qkv"].clone().requires_grad_()})
        cache_attention(**{**attention, "q": attention["q"].clone().requires_grad_()})


@pytest.mark.gpu
def test_writes_raise_versions(cuda_device):
    """Tensors written in place count a version more, the others none; inference tensors have no versions."""
    append, attention = tensors("cuda")
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    plan = dict(cached=ints([3]), new=ints([2]), table=ints([[0]]), free_pages=ints([1]))
    out = CachePlan(*(torch.zeros_like(t) for t in cache_plan(**plan, page=16, max_rows=2)))
    versions = lambda kw: {k: t._version for k, t in kw.items() if torch.is_tensor(t)}  # noqa: E731
    for call, kw, changed in (
            (lambda: cache_plan(**plan, page=16, max_rows=2, out=out), {**plan, **out._asdict()},
             {"table", *CachePlan._fields}),
            (lambda: cache_append(**append), append, {"k_pages", "v_pages", "q", "gates"}),
            (lambda: cache_attention(**attention), attention, {"out"})):
        before = versions(kw)
        call()
        after = versions(kw)
        assert {k for k in after if after[k] != before[k]} == changed
    with torch.inference_mode():
        append, attention = tensors("cuda")
        cache_append(**append)
        cache_attention(**attention)
