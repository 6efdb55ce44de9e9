"""The frame cache's first calls of a process inside a capture: nothing has to be loaded or set up beforehand."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from turbo_roformer_b200 import cache_plan, cache_append, cache_attention

new, past, heads, page, dt = {new}, 700, 8, 32, torch.float16
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
g = torch.Generator(device="cuda").manual_seed(0)
pages = -(-(past + new) // page)
k, v = (torch.randn(pages, heads, page, 64, device="cuda", generator=g).to(dt) for _ in range(2))
qkv = torch.randn(new, 1, 3 * heads * 64, device="cuda", generator=g).to(dt)
held = -(-past // page)
table = ints([list(range(held)) + [-1] * (pages - held)])
cached, fresh, free = ints([past]), ints([new]), ints(list(range(held, pages)) or [0])
torch.cuda.synchronize()

def push():
    plan = cache_plan(cached, fresh, table, free, page, new)
    q, _ = cache_append(qkv, plan.positions, plan.slots, k, v, heads, heads, freqs=None)
    return cache_attention(q, k, v, table, plan.cu, plan.total, new, past + new)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = push()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, push())
s = torch.einsum("qhd,hkd->hqk", qkv[:, 0, : heads * 64].view(new, heads, 64).float(),
                 k.transpose(0, 1).reshape(heads, -1, 64)[:, : past + new].float()) * 0.125
s = s.masked_fill(torch.arange(past + new, device="cuda") > torch.arange(past, past + new, device="cuda")[:, None], -torch.inf)
ref = torch.einsum("hqk,hkd->qhd", s.softmax(-1), v.transpose(0, 1).reshape(heads, -1, 64)[:, : past + new].float())
# half a step of fp16 of weights and result, on values below 5: far below a wrong page or row
assert (out.float() - ref).abs().max() < 2 * 2.0**-11 * 5
"""


@pytest.mark.parametrize("new", [1, 100, 400])
def test_first_calls_inside_a_capture(cuda_device, new):
    env = {**os.environ, "PYTHONPATH": os.path.dirname(os.path.dirname(os.path.abspath(__file__)))}
    res = subprocess.run([sys.executable, "-c", SCRIPT.format(new=new)], env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
