"""Distillation over more rows than one launch takes."""
import pytest
import torch

import ops_reference as R
from test_gpu_ops import DEV, F16, F32, gen, normal, ops, teacher  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,n,V", [(F16, 8_400_000, 7), (F32, 4_300_000, 40)])
def test_many_rows(ops, dtype, n, V):
    """Up to 512 threads a row: 2^32 of them and more.  Every row is that of a call of a few; rows at the ends and at the borders of
    bands are held to 64 bits."""
    g, k, tau = gen("rows", n, V), 3, 2.0
    z = (torch.randn(n, V, device=DEV, generator=torch.Generator(DEV).manual_seed(V)) * 3).to(dtype)
    tv = (torch.randn(n, k, device=DEV, generator=torch.Generator(DEV).manual_seed(k)) * 2).to(dtype)
    ti = torch.randint(-1, V, (n, k), device=DEV, dtype=torch.int32, generator=torch.Generator(DEV).manual_seed(1))
    w = torch.rand(n, device=DEV, generator=torch.Generator(DEV).manual_seed(2)) + 0.1
    loss, lse = ops.distill(z, tv, ti, tau)
    grad = ops.distill_grad(z, tv, ti, lse, w, tau)
    both, both_grad = ops.distill_loss_grad(z, tv, ti, w, tau)
    assert torch.equal(both, loss)
    step = 1_000_003
    for at in range(0, n, step):
        part = slice(at, min(at + step, n))
        few, few_lse = ops.distill(z[part], tv[part], ti[part], tau)
        assert torch.equal(loss[part], few) and torch.equal(lse[part], few_lse)
        assert torch.equal(grad[part], ops.distill_grad(z[part], tv[part], ti[part], lse[part], w[part], tau))
        assert torch.equal(both_grad[part], ops.distill_loss_grad(z[part], tv[part], ti[part], w[part], tau)[1])
    some = torch.tensor(sorted({r for b in range(0, n, 1 << 21) for r in (b - 1, b, b + 1) if 0 <= r < n} | {n - 2, n - 1}))
    zc, tc, ic, wc = (t[some.to(DEV)].cpu() for t in (z, tv, ti, w))
    want = R.distill(zc, tc, ic, tau, wc)
    R.within(loss[some.to(DEV)], want["loss"], "loss")
    R.within(lse[some.to(DEV)], want["lse"], "lse")
    R.within(both_grad[some.to(DEV)], want["d_logits"], "gradient of the call for both")
    R.within(grad[some.to(DEV)], R.distill(zc, tc, ic, tau, wc, lse[some.to(DEV)].cpu())["d_logits"], "gradient")
    ops.distill_grad(z, tv, ti, lse, w, tau, out=z)
    assert torch.equal(z, grad), "in place"
