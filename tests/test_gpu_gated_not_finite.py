"""Infinities and NaN in the gated block's backward pass: what they enter by the formulas is not finite, the rest has the bits that it has
without them.  Sizes that are no multiple of 64 repeat an operand's last row against zeros, so it is that row that holds them here."""
import math

import pytest
import torch

from test_gpu_ops import DEV, TYPES, gen, normal, ops  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F", [(5, 24, 9), (70, 72, 40), (70, 75, 64), (64, 72, 130), (2050, 72, 2050)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_backward(ops, bad, M, D, F, dtype):
    g = gen("bad", M, D, F)
    x, wg, wu, d_h = normal(g, M, D, dtype=dtype), normal(g, F, D, dtype=dtype), normal(g, F, D, dtype=dtype), normal(g, M, F, dtype=dtype)
    saved = normal(g, 2, M, F)
    clean = ops.gated_ffn_grad(*(t.to(DEV) for t in (d_h, x, wg, wu, saved)))

    def grads(**changed):
        at = {"d_h": d_h, "x": x, "wg": wg, "wu": wu, "saved": saved, **changed}
        return ops.gated_ffn_grad(*(at[k].to(DEV) for k in ("d_h", "x", "wg", "wu", "saved")))

    def others(t, was, dim, at):                       # all but one row or column are as they were, and that one is not finite
        assert not torch.isfinite(t.select(dim, at)).any()
        keep = torch.arange(t.shape[dim], device=DEV) != at
        assert torch.equal(t[keep] if dim == 0 else t[:, keep], was[keep] if dim == 0 else was[:, keep])

    y = x.clone()
    y[M - 1, 3] = bad                                  # a row's entry: the weights' gradients, in its column
    d_x, d_wg, d_wu = grads(x=y)
    assert torch.equal(d_x, clean[0])
    others(d_wg, clean[1], 1, 3)
    others(d_wu, clean[2], 1, 3)
    w = wg.clone()
    w[F - 1, 5] = bad                                  # a weight: d_x in its column
    d_x, d_wg, d_wu = grads(wg=w)
    assert torch.equal(d_wg, clean[1]) and torch.equal(d_wu, clean[2])
    others(d_x, clean[0], 1, 5)
    d = d_h.clone()
    d[M - 1, F - 1] = bad                              # a slope: d_x in its row, the weights' gradients in theirs
    d_x, d_wg, d_wu = grads(d_h=d)
    others(d_x, clean[0], 0, M - 1)
    others(d_wg, clean[1], 0, F - 1)
    others(d_wu, clean[2], 0, F - 1)
