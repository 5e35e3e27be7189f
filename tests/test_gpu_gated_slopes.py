"""dg and du of the gated block's backward pass keep fp32's range and 16 bits, whatever the operands' type: gradients against 64 bits under
bounds that count one rounding to the type, that of the result."""
import pytest
import torch

import ops_reference as R
from test_gpu_ops import BF16, DEV, F16, gen, normal, ops, strided  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu

# A rounded bf16 leaves at most 2^-8 of a value, a remainder whose exponent is at least 9 lower, and that one's rounding half a step of
# 2^-7: dg, du as two parts are off by 2^-17.  fp16 weights and x are two more parts, exactly, whose product with the second part of dg, at
# most 2^-8 2^-8, is left out.
PARTS = {BF16: 2.0 ** -17, F16: 2.0 ** -17 + 2.0 ** -16}
U = R.U


def gradients(d_h, x, wg, wu, saved, act):
    """{name: (value, bound)} from the projections that the call is given."""
    dt = x.dtype
    stretches = 3 if dt == F16 else 2
    d, x, wg, wu = (t.double() for t in (d_h, x, wg, wu))
    g, u = saved.double()
    a, da = R.act(act, g)
    ea = 16 * U * (a.abs() + 1e-30) + (4 * U * g.abs() if act == "gelu" else 0)   # as for the forward pass
    eda = 16 * U * (1 + g.abs())
    dg, du = d * u * da, d * a
    edg = d.abs() * u.abs() * eda + (PARTS[dt] + 3 * U) * dg.abs() + 2.0 ** -126
    edu = d.abs() * ea + (PARTS[dt] + 3 * U) * du.abs() + 2.0 ** -126
    adg, adu = dg.abs() + edg, du.abs() + edu
    M, F = dg.shape
    dx = dg @ wg + du @ wu
    out = {"d_x": (dx, edg @ wg.abs() + edu @ wu.abs() + (adg @ wg.abs() + adu @ wu.abs()) * 2 * F * stretches * U + R.store(dx, dt))}
    for key, s, e, m in (("d_w_gate", dg, edg, adg), ("d_w_up", du, edu, adu)):
        w = s.T @ x
        out[key] = w, (e + m * M * stretches * U).T @ x.abs() + R.store(w, dt)
    return {k: tuple(t.cpu() for t in v) for k, v in out.items()}


def check(ops, d_h, x, wg, wu, saved, act, place=lambda t: t.to(DEV)):
    dev = [place(t) for t in (d_h, x, wg, wu)]
    saved = saved.to(DEV)
    want = gradients(*dev, saved, act)
    got = ops.gated_ffn_grad(*dev, saved, act)
    for key, t in zip(("d_x", "d_w_gate", "d_w_up"), got):
        assert torch.isfinite(want[key][0]).all() and want[key][0].abs().max() < torch.finfo(t.dtype).max / 2, "the case itself is out of range"
        R.within(t, want[key], key)
    for t, again in zip(got, ops.gated_ffn_grad(*dev, saved, act)):
        assert torch.equal(t, again), "two runs differ"


# every tile and cut of the backward products: small and large, one launch or two, k cut or not, laid out first or not
SHAPES = [(1, 8, 1), (1, 64, 96), (40, 64, 96), (33, 100, 70), (130, 257, 129), (6000, 4104, 16), (6000, 4100, 9), (70, 4104, 8200),
          (700, 4104, 4104), (1300, 4104, 1032), (1300, 4100, 1027), (70, 2056, 4104), (2050, 72, 2050)]


def operands(M, D, F, dtype, d_std=1.0, u_std=1.0, x_std=1.0, w_std=None):
    g = gen("slopes", M, D, F)
    w_std = D ** -0.5 if w_std is None else w_std
    d_h, x = normal(g, M, F, std=d_std, dtype=dtype), normal(g, M, D, std=x_std, dtype=dtype)
    wg, wu = normal(g, F, D, std=w_std, dtype=dtype), normal(g, F, D, std=w_std, dtype=dtype)
    return d_h, x, wg, wu, torch.stack([normal(g, M, F), normal(g, M, F, std=u_std)])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,D,F", SHAPES)
def test_one_rounding(ops, M, D, F, dtype):
    check(ops, *operands(M, D, F, dtype), ["silu", "gelu", "sigmoid"][(M + D + F) % 3])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_rounding_of_unaligned_rows(ops, dtype):
    check(ops, *operands(70, 128, 90, dtype), "silu", lambda t: strided(t, 3, 5))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,D,F", [(5, 40, 24), (90, 128, 70), (1300, 1032, 260)])
def test_slopes_beyond_fp16(ops, M, D, F, dtype):
    """dh of thousands and u of 40: dg and du of 10^5 and more, against weights and rows of 10^-3."""
    d_h, x, wg, wu, saved = operands(M, D, F, dtype, d_std=2000.0, u_std=40.0, x_std=1e-3, w_std=1e-3)
    assert (d_h.double() * saved[1].double()).abs().max() > 65504 * 2
    check(ops, d_h, x, wg, wu, saved, "silu")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,D,F", [(5, 40, 24), (90, 128, 70), (1300, 1032, 260)])
def test_slopes_below_fp16(ops, M, D, F, dtype):
    """dh of 10^-5 and u of 10^-2: dg of about fp16's smallest step, against weights and rows of 100."""
    check(ops, *operands(M, D, F, dtype, d_std=1e-5, u_std=1e-2, x_std=100.0, w_std=100.0), "silu")


def test_one_large_slope(ops):
    """A single entry beyond fp16 leaves the other rows and columns as they are without it."""
    d_h, x, wg, wu, saved = operands(50, 64, 40, F16, x_std=0.1, w_std=0.1)
    clean = ops.gated_ffn_grad(*(t.to(DEV) for t in (d_h, x, wg, wu, saved)))
    d_h[7, 3], saved[1, 7, 3] = 2000.0, 40.0
    saved[0, 7, 3] = 1.0
    check(ops, d_h, x, wg, wu, saved, "silu")
    got = ops.gated_ffn_grad(*(t.to(DEV) for t in (d_h, x, wg, wu, saved)))
    rows, cols = [i for i in range(50) if i != 7], [i for i in range(40) if i != 3]
    assert torch.equal(got[0][rows], clean[0][rows])
    assert torch.equal(got[1][cols], clean[1][cols]) and torch.equal(got[2][cols], clean[2][cols])
