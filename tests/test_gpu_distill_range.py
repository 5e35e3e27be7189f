"""Distillation where logit / tau is beyond fp32, or its log-sum holds nothing of the classes' number: rows of the type's lowest value at
temperatures below one, teachers of such values, rows of large logits."""
import pytest
import torch

import ops_reference as R
from test_gpu_ops import BF16, DEV, F32, TYPES, gen, normal, ops, teacher  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu
U = R.U
ROWS = [33, 300, 3000, 40000, 140001]                    # a wave a row, a workgroup a row, rows that are walked


def close(got, want, bound, what):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), (what, float((off / bound).max()))


def shifted(z, tv, ti, tau, w):
    """(loss, gradient) in 64 bits from differences to the maxima alone."""
    z, t = z.double(), tv.double()
    logp = torch.log_softmax((t - t.amax(1, keepdim=True)) / tau, 1)
    p = logp.exp()
    logq = torch.log_softmax((z - z.amax(1, keepdim=True)) / tau, 1)
    terms = torch.where(p > 0, p * (logp - logq.gather(1, ti.long())), 0.0)
    grad = logq.exp().scatter_add(1, ti.long(), -p) * (w.double() * tau)[:, None]
    return tau * tau * terms.sum(1), grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", ROWS)
@pytest.mark.parametrize("tau", [0.25, 0.75])
def test_lowest_values(ops, V, tau, dtype):
    """All logits the lowest value of the type, the teacher's too: both even.  The loss is tau^2 (log V - log k), with the roundings of a
    sum of V ones, two logarithms of at most 12 and the products: 2^-24 (V / 64 + 40 + 40) of its largest term."""
    low = torch.finfo(dtype).min
    z = torch.full((3, V), low, dtype=dtype)
    tv, ti = teacher(gen("low", V), 3, V, 4, dtype, ragged=False)
    tv[:] = low
    z[2], tv[2] = -low, -low                             # the highest
    w = torch.ones(3)
    want, want_grad = shifted(z, tv, ti, tau, w)
    bound = (V / 64 + 80) * U * 12 * tau * tau
    loss, _ = ops.distill(z.to(DEV), tv.to(DEV), ti.to(DEV), tau)
    close(loss, want, bound, "loss")
    both, grad = ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV), tau)
    close(both, want, bound, "loss of the call for both")
    close(grad, want_grad, tau * (V / 64 + 80) * U + R.store(want_grad, dtype), "gradient")


@pytest.mark.parametrize("V", ROWS)
@pytest.mark.parametrize("tau", [0.5, 1.5])
def test_large_logits(ops, V, tau):
    """Logits around 10^6, a few units apart: differences to the maximum (exact here, multiples of 2^-4) carry the loss, not 10^6 / tau.
    log q of at most 60 from a sum of V terms, each of them off by 4 * 60 roundings."""
    g = gen("large", V)
    z = 1e6 + (normal(g, 4, V, std=2.0) * 16).round() / 16
    tv, ti = teacher(g, 4, V, 5, F32, ragged=False)
    tv = 1e6 + (tv * 16).round() / 16
    w = torch.ones(4)
    want, want_grad = shifted(z, tv, ti, tau, w)
    bound = (V / 64 + 40 + 4 * 60 + 8) * U * 60 * tau * tau
    loss, _ = ops.distill(z.to(DEV), tv.to(DEV), ti.to(DEV), tau)
    close(loss, want, bound, "loss")
    both, grad = ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV), tau)
    close(both, want, bound, "loss of the call for both")
    close(grad, want_grad, tau * (V / 64 + 40 + 4 * 60 + 8) * U, "gradient")
    assert bound < U * 1e6 * tau, "what a log-sum of 10^6 / tau in 32 bits may be off, times tau^2"


def test_infinite_logits(ops):
    """An infinite logit leaves no number: the loss and the gradient are NaN, in that row alone."""
    z = normal(gen("inf"), 3, 50)
    tv, ti = teacher(gen("inf t"), 3, 50, 4, F32, ragged=False)
    clean = ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), torch.ones(3, device=DEV), 0.5)
    z[1, 7] = float("inf")
    loss, grad = ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), torch.ones(3, device=DEV), 0.5)
    assert torch.isnan(loss[1]) and torch.isnan(ops.distill(z.to(DEV), tv.to(DEV), ti.to(DEV), 0.5)[0][1])
    for t, was in ((loss, clean[0]), (grad, clean[1])):
        assert torch.equal(t[[0, 2]], was[[0, 2]])


@pytest.mark.parametrize("V", ROWS)
@pytest.mark.parametrize("tau", [1.0, 1.5])
def test_small_probabilities_of_fp32_rows(ops, V, tau):
    """One class at 0 and the others at -30 to -80, in quarters: the sum is 1 to 2^-24, differences are exact, and an exponential is off by its
    own step of 2^-23 however small it is.  With the two roundings of w tau / s, the product and the sum: 12 of 2^-24."""
    g = gen("small", V)
    z = -torch.randint(120, 321, (4, V), generator=g).float() / 4 * tau
    z[:, 0] = 0
    tv, ti = torch.zeros(4, 1), torch.zeros(4, 1, dtype=torch.int32)
    w = torch.rand(4, generator=g) + 0.5
    q = torch.softmax(z.double() / tau, 1)[:, 1:]
    want = q * w.double()[:, None] * tau
    assert q.max() < 1e-12 and q.min() > 1e-36
    args = z.to(DEV), tv.to(DEV), ti.to(DEV)
    grad = ops.distill_loss_grad(*args, w.to(DEV), tau)[1][:, 1:]
    close(grad, want, 12 * U * want, "gradient of the call for both")
    # z / tau - lse is rounded once more, by 2^-24 of up to 80
    grad = ops.distill_grad(*args, ops.distill(*args, tau)[1], w.to(DEV), tau)[:, 1:]
    close(grad, want, (12 + 80) * U * want, "gradient")
