"""The operators of graphslim_amd.ops in 64 bits, with bounds on what fp32 arithmetic and one rounding to the outputs' type may be off.

Every bound counts roundings: u = 2^-24 is the largest relative error of one fp32 operation, h(t) = finfo(t).eps / 2 that of rounding
to type t (below the type's normal range: half its smallest step)."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def store(x, dtype):
    """Error of rounding x to dtype; subnormals have the absolute step smallest_normal * eps."""
    fi = torch.finfo(dtype)
    return x.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps / 2


def embedding(table, ids, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    out = torch.where(ok[..., None], table.double()[ids.clamp(0, table.shape[0] - 1).long()] * scale, 0.0)
    return out, out.abs() * 2 * U + store(out, table.dtype)       # scale as fp32, the product; the store


def embedding_grad(d_out, ids, n_rows, scale, dtype, old=None):
    d, i = d_out.double().reshape(-1, d_out.shape[-1]), ids.reshape(-1).long()
    ok = (i >= 0) & (i < n_rows)
    out, mag = (torch.zeros(n_rows, d.shape[1], dtype=torch.float64) for _ in range(2))
    out.index_add_(0, i[ok], d[ok])
    mag.index_add_(0, i[ok], d[ok].abs())
    cnt = torch.bincount(i[ok], minlength=n_rows).double()[:, None]
    out, mag = out * scale, mag * abs(scale)
    err = mag * (cnt + 3) * U        # at most cnt additions of a row's terms, in any order; scale as fp32, its product
    if old is not None:
        out = out + old.double()
        err = err + out.abs() * U
    return out, err + store(out, dtype)


# largest |act'| and |act''|
_SLOPES = {"silu": (1.1, 0.5), "gelu": (1.13, 0.8), "relu": (1.0, 0.0), "sigmoid": (0.25, 0.1)}


def act(name, g):
    if name == "relu":
        return g.clamp_min(0), (g > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (g * s, s * (1 + g * (1 - s))) if name == "silu" else (s, s * (1 - s))


def _product(a, b, extra):
    """a b^T of fp32-accumulated products, whatever their order: K additions, `extra` relative error of each product.  fp32 operands are
    sums of bf16 parts, whose smallest step is 2^-133: what is left of a value below it is lost, at most 2^-134 of each factor, and the
    product is off by that times the other factor."""
    lost = 2.0 ** -134 * (a.abs().sum(1, keepdim=True) + b.abs().sum(1)) if extra else 0.0
    return a @ b.T, (a.abs() @ b.abs().T) * (a.shape[1] * U + extra) + lost


def gated(x, wg, wu, name, d_h=None):
    """{"h": (value, bound), ...}, with the gradients if d_h is given.  Three-part fp32 operands leave out three cross products, each at
    most 2^-8 2^-16 of a product, and their last part is rounded by 2^-24: 4 * 2^-24 in all."""
    dt = x.dtype
    extra = 4 * U if dt == torch.float32 else 0.0
    s1, s2 = _SLOPES[name]
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, eg = _product(x, wg, extra)
    u, eu = _product(x, wu, extra)
    a, da = act(name, g)
    ea = s1 * eg + 16 * U * (a.abs() + 1e-30)          # exp2, reciprocal or erf and a few products: at most 16 roundings
    # (erf is small against the 1 it is added to: that sum's error is absolute, and grows with g)
    if name == "gelu":
        ea = ea + 4 * U * g.abs()
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + U * h.abs()
    out = {"h": (h, eh + store(h, dt)), "saved": (torch.stack([g, u]), torch.stack([eg, eu]) + U * torch.stack([g, u]).abs())}
    if d_h is None:
        return out
    d = d_h.double()
    eda = s2 * eg + 16 * U * (1 + g.abs()) * 1.0       # sums of terms of at most 1 + |g|
    op = 0.0 if dt == torch.float32 else half_step(dt)  # dg, du enter the products in the operands' type
    tiny = 0.0 if dt == torch.float32 else torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    dg, du = d * u * da, d * a
    edg = d.abs() * (eu * da.abs() + u.abs() * eda + eu * eda)
    edg = edg + (op + 3 * U) * (dg.abs() + edg) + tiny
    edu = d.abs() * ea
    edu = edu + (op + 3 * U) * (du.abs() + edu) + tiny
    adg, adu = dg.abs() + edg, du.abs() + edu
    F = dg.shape[1]
    dx = dg @ wg + du @ wu
    ex = edg @ wg.abs() + edu @ wu.abs() + (adg @ wg.abs() + adu @ wu.abs()) * (2 * F * U + extra)
    out["d_x"] = dx, ex + store(dx, dt)
    for key, dd, ed, ad in (("d_w_gate", dg, edg, adg), ("d_w_up", du, edu, adu)):
        w = dd.T @ x
        out[key] = w, ed.T @ x.abs() + (ad.T @ x.abs()) * (x.shape[0] * U + extra) + store(w, dt)
    return out


def distill(z, tv, ti, tau, d_loss=None, lse_in=None):
    """{"loss", "lse", "d_logits"}: (value, bound).  Rows whose logits are all -inf have q = 0."""
    dt = z.dtype
    n, V = z.shape
    z = z.double()
    ti = ti.long()
    there = (ti >= 0) & (ti < V) & (tv.double() != -math.inf)
    any_there = there.any(1)
    t = torch.where(there, tv.double() / tau, -math.inf)
    t = torch.where(any_there[:, None], t, 0.0)
    logp = torch.log_softmax(t, 1)
    p = torch.where(there, logp.exp(), 0.0)
    at = torch.where(there, ti, 0)
    zt = z / tau
    lse = torch.logsumexp(zt, 1)
    zc = zt.gather(1, at)
    # (shifted by the maximum, not by lse: at 1e38 even 64 bits hold no log-sum beside it)
    logq = torch.where(lse[:, None] == -math.inf, -math.inf, torch.log_softmax(zt, 1).gather(1, at))
    terms = torch.where(there & (p != 0), p * (logp - logq), 0.0)
    loss = tau * tau * terms.sum(1)
    # exp of a difference d: its argument carries 4 roundings of |d|, exp2 itself 2; underflow to 0 is below 2^-126
    top = zt.amax(1)
    adds = V / 64 + 40                                  # a lane's share, then the tree
    fin = torch.where(torch.isfinite(zt), zt, top[:, None])
    spread = (top[:, None] - fin).abs()
    wgt = torch.exp(fin - top[:, None])
    esum = (wgt * (4 * spread + 4 + adds) * U).sum(1) / wgt.sum(1)
    elog = 2 * U * torch.log(wgt.sum(1)).abs() + 2 * U
    else_ = esum + elog + 3 * U * (lse.abs() + top.abs())
    tmax = t.amax(1, keepdim=True)
    et = torch.where(there, 3 * U * (t.abs() + tmax.abs()) + 2 * U * (t - tmax).abs(), 0.0)
    k = ti.shape[1]
    ep = et + et.amax(1, keepdim=True) + (k + 8) * U    # relative error of p; absolute one of log p is the same and that of the log
    elp = ep + 2 * U * logp.abs()
    ez = else_[:, None] + 3 * U * (zc.abs() + lse.abs()[:, None])
    bad = ~torch.isfinite(terms)
    each = torch.where(there & (p != 0) & ~bad, p * (ep * (logp - logq).abs() + elp + ez), 0.0)
    eloss = tau * tau * (each.sum(1) + (k + 4) * U * torch.where(bad, 0.0, terms.abs()).sum(1))
    out = {"loss": (loss, eloss + 1e-30), "lse": (lse, else_ + 1e-30)}
    if d_loss is None:
        return out
    if lse_in is not None:
        lse_used = lse_in.double()
        eq = (6 * (zt - lse_used[:, None]).abs() + 8 + 2 * zt.abs()) * U          # exp2 of a difference; z / tau as two fused products
    else:
        lse_used = lse
        eq = 4 * spread * U + esum[:, None] + 10 * U
    q = torch.exp(zt - lse_used[:, None]) if lse_in is not None else torch.softmax(zt, 1)
    q = torch.where(lse_used[:, None] == -math.inf, 0.0, q)
    w = torch.where(any_there, d_loss.double() * tau, 0.0)[:, None]
    on = w[:, 0] != 0
    g, mag = torch.zeros_like(q), torch.zeros_like(q)
    g[on], mag[on] = (q * w)[on], (q * w.abs() * torch.nan_to_num(eq))[on]
    sums = torch.zeros_like(q).scatter_add_(1, at, torch.where(there, p, 0.0))
    esums = torch.zeros_like(q).scatter_add_(1, at, torch.where(there, p * (ep + 4 * U), 0.0))
    g[on] -= (sums * w)[on]
    mag[on] += (esums * w.abs())[on]
    mag = mag + g.abs().nan_to_num() * 4 * U + w.abs() * 2.0 ** -120
    out["d_logits"] = g, mag + store(g.nan_to_num(), dt)
    return out


def within(got, want, what=""):
    """got inside value +- bound everywhere; not-finite values equal."""
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(value)], value[~fine & ~torch.isnan(value)]), f"{what}: infinities differ"
    off = (got - value).abs()[fine]
    if off.numel():
        ratio = off / bound[fine].clamp_min(1e-300)
        worst = int(ratio.argmax())
        assert float(ratio[worst]) <= 1, (f"{what}: off by {float(off[worst]):.3g}, {float(bound[fine][worst]):.3g} allowed "
                                          f"(value {float(value[fine][worst]):.6g})")
