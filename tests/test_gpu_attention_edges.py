"""Whole-chunk attention (trc_attention) with keys that are not finite: the formula's NaN, at every key position."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_stages import call, from_sequences, stream, vp

pytestmark = pytest.mark.gpu


def run(model, mode, Q, K, V, G, T, N):
    O = torch.full((N, 512), 7.0, device="cuda", dtype=torch.float16)
    call(model, "trc_attention", mode, vp(Q), vp(K), vp(V), vp(G), vp(O), 1, T, stream(model))
    return O.view(N, 8, 64)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("mode,T", [(0, 77), (0, 300), (0, 700), (1, 40)])
def test_attention_keys_not_finite(tiny_cuda, tiny_cfg, mode, T, value):
    """A key element of NaN or +inf: rows of its sequence and head whose score there is NaN or +inf are NaN, wherever the
    key lies; all other sequences and heads are as without it."""
    Fb = tiny_cfg.n_bands
    N, L = T * Fb, T if mode == 0 else Fb
    BH = N * 8 // L
    g = torch.Generator().manual_seed(T)
    Q = (torch.randn(BH, L, 64, generator=g) * 0.25).half()
    K, V = (torch.randn(BH, L, 64, generator=g) * s for s in (0.25, 1.0))
    G = torch.rand(N, 8, generator=g).cuda()
    Qd, Kd, Vd = Q.cuda(), K.half().cuda(), V.half().cuda()
    want = run(tiny_cuda, mode, Qd, Kd, Vd, G, T, N)
    spots = sorted({*range(min(L, 16)), L // 2, L - 1, *range(max(0, L - 9), L)})
    bad = torch.zeros(BH, L, 64, dtype=torch.bool)
    for i, at in enumerate(spots):  # a sequence of its own for every place
        seq = (i * 5 + 3) % BH
        Kd[seq, at, 11] = value
        bad[seq, Q[seq, :, 11] > 0 if value == float("inf") else slice(None)] = True
    got = run(tiny_cuda, mode, Qd, Kd, Vd, G, T, N)
    touched = torch.zeros(BH, L, 64, dtype=torch.bool)
    touched[[(i * 5 + 3) % BH for i in range(len(spots))]] = True
    order = lambda m: from_sequences(m.float(), 1, T, Fb, mode).reshape(N, 8, 64).numpy() > 0  # noqa: E731
    got, want = got.cpu().numpy(), want.cpu().numpy()
    assert np.isnan(got[order(bad)]).all()
    assert np.array_equal(got[~order(touched)], want[~order(touched)])
    assert np.isfinite(got[order(touched & ~bad)]).all()
