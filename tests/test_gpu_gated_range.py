"""fp32 operands beyond the largest bf16: the first of their three parts is cut, not rounded to infinity.  (24 rows and fewer are multiplied
as they are in the forward pass; these tests have more.)"""
import pytest
import torch

import ops_reference as R
from test_gpu_ops import DEV, gen, normal, ops  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu
BIG = [3.3962e38, -3.3962e38, 3.4e38, -3.4e38, torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max]
TINY = 2.0 ** -126                                       # a power of two: exact in one part


def test_the_values_need_the_cut():
    for v in BIG:
        w = torch.tensor(v)
        assert torch.isinf(w.bfloat16())
        top = (w.view(torch.int32) & -65536).view(torch.float32)
        mid = (w - top).bfloat16().float()
        low = (w - top - mid).bfloat16()               # (the parts are added in 64 bits: those of the largest fp32 pass 2^128 on the way)
        assert torch.isfinite(top) and top.double() + mid.double() + low.double() == w.double()


@pytest.mark.parametrize("M", [25, 40, 300])
def test_forward(ops, M):
    g = gen("cut", M)
    x, wg, wu = normal(g, M, 48), normal(g, 10, 48, std=0.1), normal(g, 10, 48, std=0.1)
    x[:, :2] = 0
    wg[:, :2] = wu[:, :2] = 0
    for i, v in enumerate(BIG):
        x[3 * i, 0], x[3 * i + 1, 1] = v, TINY           # a row's large value against weights of 2^-126 ...
    wg[:, 0], wu[:, 0] = TINY, TINY
    for i, v in enumerate(BIG):
        wg[i, 1], wu[9 - i, 1] = v, v                    # ... and a weight's against such values
    want = R.gated(x, wg, wu, "silu")
    h, saved = ops.gated_ffn(x.to(DEV), wg.to(DEV), wu.to(DEV), "silu", save=True)
    R.within(saved, want["saved"], "saved")
    R.within(h, want["h"], "h")


@pytest.mark.parametrize("M,F", [(5, 7), (40, 70), (300, 130)])
def test_backward(ops, M, F):
    """relu at g = u = 1: dg = du = dh, powers of two.  Sums of at most 2 M or 2 F terms that hold 24 bits and lose 4 * 2^-24 of each."""
    g = gen("cut grad", M, F)
    D = 64
    x, wg, wu = normal(g, M, D), normal(g, F, D), normal(g, F, D)
    d_h = 2.0 ** -torch.randint(110, 121, (M, F), generator=g).float() * (1 - 2 * torch.randint(0, 2, (M, F), generator=g)).float()
    for i, v in enumerate(BIG):
        x[i % M, i], wg[i % F, 10 + i], wu[(i + 1) % F, 20 + i] = v, v, v
    saved = torch.ones(2, M, F)
    got = ops.gated_ffn_grad(*(t.to(DEV) for t in (d_h, x, wg, wu, saved)), "relu")
    d, x, wg, wu = (t.double() for t in (d_h, x, wg, wu))
    want = [(d @ (wg + wu), d.abs() @ (wg.abs() + wu.abs()) * (2 * F + 4) * R.U)] + [(d.T @ x, d.T.abs() @ x.abs() * (M + 4) * R.U)] * 2
    for name, t, (value, bound) in zip(("d_x", "d_w_gate", "d_w_up"), got, want):
        R.within(t, (value, bound + 2.0 ** -140), name)
