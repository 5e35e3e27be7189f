"""Operators whose first call in a process is the captured one: nothing is loaded, asked for or allocated outside of the graph's memory."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from graphslim_amd import ops
dev = "cuda:0"
g = torch.Generator(dev).manual_seed(1)
r = lambda *s, t=torch.bfloat16: torch.randn(*s, device=dev, generator=g).to(t)

def inputs(t, M, D, F, n, V):
    return dict(x=r(M, D, t=t), wg=r(F, D, t=t) * D ** -0.5, wu=r(F, D, t=t) * D ** -0.5, d_h=r(M, F, t=t),
                ids=torch.randint(-1, V, (n,), device=dev, generator=g, dtype=torch.int32), d=r(n, 72, t=t), table=r(V, 72, t=t), V=V,
                z=r(M, F, t=t), tv=r(M, 5, t=t), ti=torch.randint(-1, F, (M, 5), device=dev, generator=g, dtype=torch.int32),
                w=torch.rand(M, device=dev, generator=g))

def run(s):
    h, saved = ops.gated_ffn(s["x"], s["wg"], s["wu"], save=True)
    out = [h, saved, *ops.gated_ffn_grad(s["d_h"], s["x"], s["wg"], s["wu"], saved)]
    out += [ops.embedding(s["table"], s["ids"], 2.0), ops.embedding_grad(s["d"], s["ids"], s["V"])]
    loss, lse = ops.distill(s["z"], s["tv"], s["ti"], 2.0)
    return out + [loss, lse, ops.distill_grad(s["z"], s["tv"], s["ti"], lse, s["w"], 2.0), *ops.distill_loss_grad(s["z"], s["tv"], s["ti"], s["w"], 2.0)]

for t, *sizes in ((torch.bfloat16, 2100, 1032, 2050, 20000, 3000), (torch.float16, 1300, 4100, 1027, 700, 300), (torch.float32, 700, 500, 1024, 9000, 500)):
    s = inputs(t, *sizes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(s)
    for turn in range(3):
        for o in out:
            o.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        want = run(s)
        for i, (o, e) in enumerate(zip(out, want)):
            assert torch.equal(o.nan_to_num(), e.nan_to_num()), (t, turn, i)
        s["x"].mul_(0.5)
        s["ids"].copy_(s["ids"].roll(3))
    print(t, "captured", flush=True)
"""


def test_first_call_is_captured():
    out = subprocess.run([sys.executable, "-u", "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stdout[-500:] + out.stderr[-3000:]
    assert out.stdout.count("captured") == 3
