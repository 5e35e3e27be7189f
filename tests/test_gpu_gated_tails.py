"""The gated block's activations keep their digits in both tails: errors relative to the value, however small it is."""
import math

import pytest
import torch

import ops_reference as R
from test_gpu_ops import BF16, DEV, F16, F32, TYPES, ops  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu
U = R.U
POINTS = {"gelu": torch.cat([torch.arange(-12, 12, 0.125), torch.tensor([-1e-3, 1e-3])]), "silu": torch.arange(-80, 80, 0.5),
          "sigmoid": torch.arange(-80, 80, 0.5), "relu": torch.arange(-5, 5, 0.5) + 0.25}


def exact(name, g):
    """(value, slope, the bounds of both).  exp, erfc and the quotient are within 4 steps of 2^-23 each, products and sums within half of
    one.  erfc's argument is off by 2^-23 of itself, which it takes 1 + g^2 times over, e^(-g^2/2)'s by 2^-23 too, g^2 / 2 times over."""
    g = g.double()
    if name == "relu":
        return g.clamp_min(0), (g > 0).double(), 0 * g, 0 * g
    if name == "gelu":
        cdf, phi = 0.5 * torch.erfc(-g / math.sqrt(2)), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        ecdf, ephi = (2 * (1 + g * g) + 12) * U, (g * g + 14) * U
        return g * cdf, cdf + g * phi, (g * cdf).abs() * (ecdf + U), cdf * ecdf + (g * phi).abs() * (ephi + 2 * U) + U * (cdf + g * phi).abs()
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    e = 24 * U                                           # exp, 1 + e, the quotient, e times it
    if name == "silu":
        return g * s, s * (1 + g * r), (g * s).abs() * (e + U), s * ((1 + (g * r).abs()) * (e + 2 * U) + (g * r).abs() * e)
    return s, s * r, s * e, s * r * (2 * e + U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 24, 400])
@pytest.mark.parametrize("name", sorted(POINTS))
def test_values(ops, name, rows, dtype):
    """g = x itself and u = 1, by weights of (1, 0) and (0, 1): in the kernels for few rows and for many."""
    g = POINTS[name].to(dtype)
    a, _, ea, _ = exact(name, g)
    wg, wu = (torch.tensor([w], dtype=dtype, device=DEV) for w in ((1.0, 0.0), (0.0, 1.0)))
    got = []
    for at in range(0, len(g), rows):
        x = torch.stack([g[at:at + rows], torch.ones_like(g[at:at + rows])], 1)
        got.append(ops.gated_ffn(x.to(DEV), wg, wu, name))
    tiny = 2.0 ** -126                                  # (e^-80 and below: fp32's own range)
    R.within(torch.cat(got)[:, 0], (a, ea + R.store(a, dtype) + tiny), "value")


@pytest.mark.parametrize("name", sorted(POINTS))
def test_slopes(ops, name):
    """dg[m] of row m alone, by x = 1: dW_gate = dg^T x; u = d_h = 1.  Three parts hold fp32's 24 bits down to 2^-133."""
    g = POINTS[name].float()
    n = len(g)
    _, slope, _, eslope = exact(name, g)
    x = torch.eye(n, device=DEV)
    one = torch.ones(n, 1, device=DEV)
    w = torch.ones(1, n, device=DEV)
    saved = torch.stack([g[:, None].to(DEV), one])
    d_w = ops.gated_ffn_grad(one, x, w, w, saved, name)[1]
    R.within(d_w[0], (slope, eslope + 2 * U * slope.abs() + 2.0 ** -125), "slope")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_slopes_16(ops, dtype):
    """The same in 16 bits: two parts, 2^-17, and the store."""
    for name, g in POINTS.items():
        g = g.float()
        n = len(g)
        _, slope, _, eslope = exact(name, g)
        one = torch.ones(n, 1, dtype=dtype, device=DEV)
        w = torch.ones(1, n, dtype=dtype, device=DEV)
        saved = torch.stack([g[:, None], torch.ones(n, 1)]).to(DEV)
        d_w = ops.gated_ffn_grad(one, torch.eye(n, dtype=dtype, device=DEV), w, w, saved, name)[1]
        R.within(d_w[0], (slope, eslope + 2.0 ** -17 * slope.abs() + R.store(slope, dtype) + 2.0 ** -125), name)


def test_the_bounds_tell():
    """The form that loses the digits (in 32 bits on the CPU) is outside of these bounds."""
    g = torch.arange(-8, -4, 0.125)
    a, _, ea, _ = exact("gelu", g)
    lost = g * (0.5 * (1 + torch.erf(g * 0.7071067811865476)))
    assert ((lost.double() - a).abs() > ea).float().mean() > 0.9
    g = torch.arange(10, 60, 0.5)
    _, slope, _, es = exact("sigmoid", g)
    s = 1 / (1 + torch.exp(-g))
    assert ((s * (1 - s)).double() - slope).abs().gt(es).float().mean() > 0.9
