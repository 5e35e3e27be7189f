"""graphslim_amd.ops on the GPU against the same operators in 64 bits (tests/ops_reference.py derives the tolerances)."""
import math
import zlib

import pytest
import torch

import ops_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def ops():
    from graphslim_amd import ops
    return ops


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def normal(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def strided(t, extra, offset):
    """A device copy of a matrix in rows of `extra` more elements, its first one `offset` elements into the memory; the gaps hold NaN."""
    n, c = t.shape
    flat = torch.full((offset + n * (c + extra) + 8,), float("nan"), dtype=t.dtype, device=DEV)
    view = flat[offset:offset + n * (c + extra)].view(n, c + extra)[:, :c]
    view.copy_(t)
    return view


def zipf(g, n, rows, pad=0.1):
    ids = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(rows + 1.0)) - 1).long().clamp(0, rows - 1)
    return torch.where(torch.rand(n, generator=g) < pad, -1, ids).to(torch.int32)


# ---- embedding ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,F", [(1, 1, 1), (1, 7, 3), (5, 3, 64), (64, 100, 8), (65, 33, 127), (300, 1000, 602), (7, 50, 2048)])
def test_embedding(ops, dtype, n, V, F):
    g = gen("emb", n, V, F)
    table, ids = normal(g, V, F, dtype=dtype), zipf(g, n, V)
    ids[n // 2] = V                       # beyond the table: padding too
    want = R.embedding(table, ids, 1.7)
    R.within(ops.embedding(table.to(DEV), ids.to(DEV), 1.7), want, "dense")
    tab, out = strided(table, 3, 1), strided(torch.zeros(n, F, dtype=dtype), 5, 3)
    back = ops.embedding(tab, ids.to(DEV), 1.7, out=out)
    assert back is out
    R.within(out, want, "strided")
    if n > 1:                             # what lies between the rows is left alone
        gap = out.as_strided((n - 1, 5), (F + 5, 1), out.storage_offset() + F)
        assert torch.isnan(gap).all()


def test_embedding_shapes_and_padding(ops):
    table = torch.arange(12, dtype=F32, device=DEV).view(4, 3)
    ids = torch.tensor([[0, 3], [-1, 4], [2, -2147483648]], dtype=torch.int32, device=DEV)
    got = ops.embedding(table, ids, 2.0)
    assert got.shape == (3, 2, 3)
    want = torch.zeros(3, 2, 3)
    want[0, 0], want[0, 1], want[2, 0] = 2 * table[0].cpu(), 2 * table[3].cpu(), 2 * table[2].cpu()
    assert torch.equal(got.cpu(), want)
    assert ops.embedding(table, ids[:0]).shape == (0, 2, 3)
    nan = torch.full((2, 5), float("nan"), device=DEV)
    assert torch.equal(ops.embedding(nan, torch.tensor([-1, 2], dtype=torch.int32, device=DEV)).cpu(), torch.zeros(2, 5))


GRAD_SHAPES = [(1, 1, 1), (1, 9, 5), (3, 2, 64), (64, 100, 8), (257, 33, 127), (1000, 1000, 602), (4099, 300, 40), (4096, 5, 130),
               (9001, 2500, 65), (20000, 70, 33), (300, 140001, 9),
               (7000, 270001, 5), (20, 2200003, 2), (9000, 2200003, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,F", GRAD_SHAPES)
def test_embedding_grad(ops, dtype, n, V, F):
    g = gen("embgrad", n, V, F)
    d, ids = normal(g, n, F, dtype=dtype), zipf(g, n, V)
    ids[n // 2] = V
    want = R.embedding_grad(d, ids, V, 0.3, dtype)
    got = ops.embedding_grad(d.to(DEV), ids.to(DEV), V, 0.3)
    assert got.dtype == dtype
    R.within(got, want, "dense")
    assert torch.equal(got, ops.embedding_grad(d.to(DEV), ids.to(DEV), V, 0.3)), "two runs differ"
    R.within(ops.embedding_grad(d.to(DEV), ids.to(DEV), V, 0.3, dtype=F32), R.embedding_grad(d, ids, V, 0.3, F32), "fp32 gradient")
    old = normal(g, V, F, dtype=dtype)
    out = strided(old, 5, 3)
    back = ops.embedding_grad(strided(d, 3, 1), ids.to(DEV), V, 0.3, out=out, accumulate=True)
    assert back is out
    R.within(out, R.embedding_grad(d, ids, V, 0.3, dtype, old), "strided, added")
    if V > 1:
        assert torch.isnan(out.as_strided((V - 1, 5), (F + 5, 1), out.storage_offset() + F)).all()


@pytest.mark.parametrize("n", [0, 1, 64, 700, 5000, 30000])
def test_embedding_grad_of_one_id(ops, n):
    """Every token the same row, the longest sum there is; and no token at all."""
    g = gen("same", n)
    d, ids = normal(g, n, 96), torch.full((n,), 17, dtype=torch.int32)
    R.within(ops.embedding_grad(d.to(DEV), ids.to(DEV), 40), R.embedding_grad(d, ids, 40, 1.0, F32), "one id")
    none = torch.full((n,), -1, dtype=torch.int32)
    assert not ops.embedding_grad(d.to(DEV), none.to(DEV), 40).any()
    old = torch.full((40, 96), 3.0, device=DEV)
    ops.embedding_grad(torch.full_like(d, float("nan")).to(DEV), none.to(DEV), 40, out=old, accumulate=True)
    assert (old == 3).all(), "padding reached the table"


def test_embedding_grad_order_is_the_tokens(ops):
    """Terms whose sum depends on the order: 2^24, then ones that are lost one by one, then -2^24."""
    d = torch.ones(300, 4)
    d[0], d[299] = 2.0 ** 24, -2.0 ** 24
    ids = torch.zeros(300, dtype=torch.int32)
    a = ops.embedding_grad(d.to(DEV), ids.to(DEV), 3)
    for _ in range(3):
        assert torch.equal(a, ops.embedding_grad(d.to(DEV), ids.to(DEV), 3))


def test_embedding_grad_batched_shape(ops):
    g = gen("batch")
    d, ids = normal(g, 4, 9, 20), zipf(g, 36, 11).view(4, 9)
    R.within(ops.embedding_grad(d.to(DEV), ids.to(DEV), 11), R.embedding_grad(d, ids, 11, 1.0, F32), "batched")


# ---- gated feed-forward block ------------------------------------------------------------------------------------------------------
GATED_SHAPES = [(1, 1, 1), (1, 64, 64), (2, 8, 17), (1, 130, 50), (3, 257, 129), (16, 128, 64), (17, 64, 128), (33, 100, 70),
                (64, 192, 128), (65, 63, 65), (129, 128, 192), (200, 500, 136), (260, 65, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F", GATED_SHAPES)
def test_gated(ops, dtype, M, D, F):
    g = gen("gated", M, D, F)
    act = ["silu", "gelu", "sigmoid"][(M + D + F) % 3]
    x, wg, wu = normal(g, M, D, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype)
    d_h = normal(g, M, F, dtype=dtype)
    want = R.gated(x, wg, wu, act, d_h)
    xd, wgd, wud, dd = (t.to(DEV) for t in (x, wg, wu, d_h))
    h, saved = ops.gated_ffn(xd, wgd, wud, act, save=True)
    R.within(h, want["h"], "h")
    R.within(saved, want["saved"], "saved")
    assert torch.equal(h, ops.gated_ffn(xd, wgd, wud, act)), "saving changes the result"
    got = ops.gated_ffn_grad(dd, xd, wgd, wud, saved, act)
    for key, t in zip(("d_x", "d_w_gate", "d_w_up"), got):
        assert t.dtype == dtype
        R.within(t, want[key], key)
    for t, again in zip(got, ops.gated_ffn_grad(dd, xd, wgd, wud, saved, act)):
        assert torch.equal(t, again), "two runs differ"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F,extra,offset", [(40, 64, 96, 8, 0), (40, 64, 96, 8, 8), (1, 64, 96, 3, 1), (9, 72, 40, 3, 1), (70, 128, 64, 1, 5)])
def test_gated_strides(ops, dtype, M, D, F, extra, offset):
    g = gen("gstride", M, D, F)
    x, wg, wu = normal(g, M, D, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype)
    d_h = normal(g, M, F, dtype=dtype)
    want = R.gated(x, wg, wu, "silu", d_h)
    xs, ws, us, ds = strided(x, extra, offset), strided(wg, extra, offset), strided(wu, extra, 0), strided(d_h, extra, offset)
    h, saved = ops.gated_ffn(xs, ws, us, "silu", save=True)
    R.within(h, want["h"], "h")
    for key, t in zip(("d_x", "d_w_gate", "d_w_up"), ops.gated_ffn_grad(ds, xs, ws, us, saved, "silu")):
        R.within(t, want[key], key)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_gated_activations(ops, act):
    """Pre-activations from -30 to 30 through a width of one; relu's are kept away from its corner."""
    x = torch.linspace(-30, 30, 61)[:, None] + 0.25
    wg, wu = torch.ones(5, 1), torch.linspace(-2, 2, 5)[:, None]
    d_h = torch.ones(61, 5)
    want = R.gated(x, wg, wu, act, d_h)
    args = [t.to(DEV) for t in (x, wg, wu)]
    h, saved = ops.gated_ffn(*args, act, save=True)
    R.within(h, want["h"], "h")
    for key, t in zip(("d_x", "d_w_gate", "d_w_up"), ops.gated_ffn_grad(d_h.to(DEV), *args, saved, act)):
        R.within(t, want[key], key)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_no_rows(ops, dtype):
    x, w = torch.empty(0, 12, dtype=dtype, device=DEV), torch.ones(7, 12, dtype=dtype, device=DEV)
    h, saved = ops.gated_ffn(x, w, w, save=True)
    assert h.shape == (0, 7)
    d_x, d_wg, d_wu = ops.gated_ffn_grad(h, x, w, w, saved)
    assert d_x.shape == (0, 12) and not d_wg.any() and not d_wu.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [5, 100])
def test_gated_rows_are_their_own(ops, dtype, M):
    """A row of NaN or infinities (padding nobody cleared) stays in its row."""
    g = gen("rows", M)
    x, w, u = normal(g, M, 72, dtype=dtype), normal(g, 40, 72, std=0.1, dtype=dtype), normal(g, 40, 72, std=0.1, dtype=dtype)
    clean = ops.gated_ffn(x.to(DEV), w.to(DEV), u.to(DEV))
    bad = x.clone()
    bad[1], bad[M - 1] = float("nan"), float("inf")
    got = ops.gated_ffn(bad.to(DEV), w.to(DEV), u.to(DEV))
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[M - 1]).any()
    keep = [i for i in range(M) if i not in (1, M - 1)]
    assert torch.equal(got[keep], clean[keep])


def test_gated_large_fp32_values(ops):
    """fp32 operands at the ends of their range: the three bf16 parts of a value near the largest fp32 must not round to infinity."""
    big = 3.4e38
    x = torch.tensor([[big, 0.0], [1e-30, 1.0], [0.0, 0.0]])
    wg, wu = torch.tensor([[0.0, 1.0]]), torch.tensor([[1e-38, 0.0]])
    want = R.gated(x, wg, wu, "sigmoid")
    R.within(ops.gated_ffn(x.to(DEV), wg.to(DEV), wu.to(DEV), "sigmoid")[:1], tuple(t[:1] for t in want["h"]), "h")


# ---- distillation ------------------------------------------------------------------------------------------------------------------
def teacher(g, n, V, k, dtype, ragged=True):
    k = min(k, 1024)
    tv = normal(g, n, k, std=3.0, dtype=dtype)
    if k <= V:
        ti = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(n)]).to(torch.int32)
    else:
        ti = torch.randint(0, V, (n, k), generator=g, dtype=torch.int32)
    if ragged:
        have = torch.randint(0, k + 1, (n, 1), generator=g)
        have[n // 2] = 0
        ti = torch.where(torch.arange(k) >= have, -1, ti).to(torch.int32)
    return tv, ti


def distill_all(ops, z, tv, ti, tau, w, want_in=None):
    zd, td, id_, wd = z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV)
    want = R.distill(z, tv, ti, tau, w)
    loss, lse = ops.distill(zd, td, id_, tau)
    R.within(loss, want["loss"], "loss")
    R.within(lse, want["lse"], "lse")
    both, grad = ops.distill_loss_grad(zd, td, id_, w.to(DEV), tau)
    R.within(both, want["loss"], "loss of the call for both")
    R.within(grad, want["d_logits"], "gradient of the call for both")
    R.within(ops.distill_grad(zd, td, id_, lse, wd, tau), R.distill(z, tv, ti, tau, w, lse.cpu())["d_logits"], "gradient")
    return loss, lse, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (1, 2, 2), (3, 7, 3), (9, 40, 5), (5, 64, 64), (70, 513, 17), (4, 2047, 1024), (33, 4099, 8),
                                   (3, 20001, 130), (2, 70000, 3), (2, 131072, 64)])
def test_distill(ops, dtype, n, V, k):
    g = gen("distill", n, V, k)
    z = normal(g, n, V, std=3.0, dtype=dtype)
    tv, ti = teacher(g, n, V, k, dtype, ragged=n > 2)
    distill_all(ops, z, tv, ti, [1.0, 1.5, 2.0, 4.0][(n + V) % 4], torch.rand(n, generator=g) + 0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [19, 3001, 40001])
def test_distill_strides_and_in_place(ops, dtype, V):
    g = gen("dstride", V)
    n = 6
    z = normal(g, n, V, std=2.0, dtype=dtype)
    tv, ti = teacher(g, n, V, 6, dtype)
    w = torch.rand(n, generator=g) + 0.1
    want = R.distill(z, tv, ti, 2.0, w)
    zs, td, id_, wd = strided(z, 3, 1), tv.to(DEV), ti.to(DEV), w.to(DEV)
    out = strided(torch.zeros_like(z), 5, 3)
    loss, back = ops.distill_loss_grad(zs, td, id_, wd, 2.0, out=out)
    assert back is out
    R.within(loss, want["loss"], "loss")
    R.within(out, want["d_logits"], "gradient")
    assert torch.isnan(out.as_strided((n - 1, 5), (V + 5, 1), out.storage_offset() + V)).all()
    loss, lse = ops.distill(zs, td, id_, 2.0)
    twin = zs.clone()
    ops.distill_grad(twin, td, id_, lse, wd, 2.0, out=twin)
    R.within(twin, R.distill(z, tv, ti, 2.0, w, lse.cpu())["d_logits"], "gradient in place")
    ops.distill_loss_grad(zs, td, id_, wd, 2.0, out=zs)
    assert torch.equal(zs, out), "in place and beside differ"


@pytest.mark.parametrize("V", [40, 5000, 90000])
def test_distill_repeated_classes(ops, V):
    """The same class several times in a row's list: its gradient holds the sum."""
    g = gen("twice", V)
    z = normal(g, 4, V, std=2.0)
    tv = normal(g, 4, 12)
    ti = torch.tensor([[3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3], [5, 6, 5, 6, 5, 6, 5, 6, 5, 6, 5, V - 1], [0, 1, 2, 0, 1, 2, 0, 1, 2, -1, -1, V],
                       [V - 1, V - 1, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10]], dtype=torch.int32)
    distill_all(ops, z, tv, ti, 1.5, torch.tensor([1.0, 0.5, 0.25, 2.0]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [33, 3000, 70001])
def test_distill_masks(ops, dtype, V):
    """Masked classes (-inf, the type's lowest value), rows with nothing left, padding that holds NaN, entries of -inf."""
    g = gen("mask", V)
    low = torch.finfo(dtype).min
    z = normal(g, 9, V, std=2.0, dtype=dtype)
    tv, ti = teacher(g, 9, V, 4, dtype, ragged=False)
    ti[:, :] = torch.tensor([1, V - 1, 5, 2], dtype=torch.int32)
    z[0, 8:V - 1] = -math.inf                 # most classes masked
    z[1, 8:V - 1] = low
    z[2, 1] = -math.inf                       # a class of the teacher's masked: the loss is infinite, the gradient is not
    z[3] = float("nan")
    ti[3] = -1                                # a padded row may hold anything
    z[4] = -math.inf                          # nothing left: q = 0
    ti[5, 1:] = V                             # one entry left
    tv[6, :2] = -math.inf
    tv[7] = -math.inf                         # no entry left
    w = torch.linspace(0.5, 1.5, 9)
    w[8] = 0                                  # a row without weight
    zc = z.clone()
    zc[3] = 0                                 # (what it holds does not matter)
    want = R.distill(zc, tv, ti, 2.0, w)
    assert want["loss"][0][2] == math.inf and want["loss"][0][4] == math.inf
    zd, td, id_, wd = z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV)
    loss, lse = ops.distill(zd, td, id_, 2.0)
    R.within(loss, want["loss"], "loss")
    keep = [i for i in range(9) if i != 3]
    R.within(lse[keep], tuple(t[keep] for t in want["lse"]), "lse")
    both, grad = ops.distill_loss_grad(zd, td, id_, wd, 2.0)
    R.within(both, want["loss"], "loss of the call for both")
    R.within(grad, want["d_logits"], "gradient of the call for both")
    R.within(ops.distill_grad(zd, td, id_, lse, wd, 2.0), R.distill(zc, tv, ti, 2.0, w, torch.where(torch.isnan(lse.cpu()), 0, lse.cpu()))["d_logits"], "gradient")
    for r in (3, 7, 8):
        assert not grad[r].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [33, 3000, 40000, 70001])
def test_distill_extreme_values(ops, dtype, V):
    """Rows of nothing but the type's lowest value (all classes masked that way: q is even), of its highest, and of both."""
    g = gen("extreme", V)
    big = torch.finfo(dtype).max
    z = torch.full((4, V), -big, dtype=dtype)
    z[1], z[2, ::2], z[3, 5] = big, big, 0.0
    tv, ti = teacher(g, 4, V, 4, dtype, ragged=False)
    ti[2], ti[3] = torch.tensor([0, 2, 4, 6], dtype=torch.int32), torch.tensor([5, 5, 5, 5], dtype=torch.int32)
    want = R.distill(z, tv, ti, 2.0, torch.ones(4))
    zd, td, id_, wd = z.to(DEV), tv.to(DEV), ti.to(DEV), torch.ones(4, device=DEV)
    loss, lse = ops.distill(zd, td, id_, 2.0)
    R.within(loss, want["loss"], "loss")
    R.within(lse, want["lse"], "lse")
    both, grad = ops.distill_loss_grad(zd, td, id_, wd, 2.0)
    R.within(both, want["loss"], "loss of the call for both")
    R.within(grad, want["d_logits"], "gradient of the call for both")
    # a log-sum in fp32 resolves no class beside 1e38: q is some number of [0, 1] there, and no more can be said
    assert (ops.distill_grad(zd, td, id_, lse, wd, 2.0).abs() <= 2.0 * 2).all()


def test_distill_nan_stays_in_its_row(ops):
    g = gen("nan")
    z = normal(g, 5, 300)
    tv, ti = teacher(g, 5, 300, 4, F32, ragged=False)
    w = torch.ones(5)
    clean = [t.cpu() for t in ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV))]
    z[2, 250] = float("nan")
    loss, grad = [t.cpu() for t in ops.distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), w.to(DEV))]
    assert math.isnan(loss[2]) and torch.isnan(grad[2]).all()
    lse = ops.distill(z.to(DEV), tv.to(DEV), ti.to(DEV))[1]
    assert torch.isnan(ops.distill_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), lse, w.to(DEV))[2]).all()
    keep = [0, 1, 3, 4]
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(grad[keep], clean[1][keep])


def test_distill_no_rows(ops):
    z, tv, ti = torch.empty(0, 9, device=DEV), torch.empty(0, 2, device=DEV), torch.empty(0, 2, dtype=torch.int32, device=DEV)
    loss, lse = ops.distill(z, tv, ti)
    assert loss.shape == lse.shape == (0,)
    assert ops.distill_loss_grad(z, tv, ti, loss)[1].shape == (0, 9)


def test_distill_against_differences(ops):
    """The gradient against central differences of the loss: step e = 2^-6 along a unit direction v.  The third derivative of the loss
    along v is at most 1 / tau (2 max |v| <= 2), so the difference is off by e^2 / 6 * 2, and by the loss's own error / e."""
    g = gen("diff")
    n, V, tau, e = 8, 200, 2.0, 2.0 ** -6
    z = normal(g, n, V, std=2.0)
    tv, ti = teacher(g, n, V, 6, F32, ragged=False)
    v = normal(g, n, V)
    v = v / v.norm(dim=1, keepdim=True)
    args = tv.to(DEV), ti.to(DEV)
    up, dn = (ops.distill((z + s * e * v).to(DEV), *args, tau)[0].double().cpu() for s in (1, -1))
    _, grad = ops.distill_loss_grad(z.to(DEV), *args, torch.ones(n, device=DEV), tau)
    slope = (grad.double().cpu() * v.double()).sum(1)
    noise = R.distill(z, tv, ti, tau)["loss"][1] + 2.0 ** -24 * (z.abs().amax(1).double() + 1) * tau
    assert ((up - dn) / (2 * e) - slope).abs().le(e * e / 3 + 2 * noise / e + 1e-6).all()


# ---- streams, graphs, a run of all of them -----------------------------------------------------------------------------------------
def student(g, rows=300, width=72, inner=136, classes=90, tokens=150, k=6, dtype=F32):
    s = {"table": normal(g, rows, width, dtype=dtype), "wg": normal(g, inner, width, std=width ** -0.5, dtype=dtype),
         "wu": normal(g, inner, width, std=width ** -0.5, dtype=dtype), "head": normal(g, classes, inner, std=inner ** -0.5, dtype=dtype),
         "ids": zipf(g, tokens, rows), "w": torch.rand(tokens, generator=g) / tokens}
    s["tv"], s["ti"] = teacher(g, tokens, classes, k, dtype)
    return s


def student_step(ops, s, tau=2.0):
    """One training step's gradients through the framework's calls: lookup, gated block, classifier (gs_gemm_f32), loss, and back."""
    from graphslim_amd.engine import gemm
    x = ops.embedding(s["table"], s["ids"], 0.5)
    h, saved = ops.gated_ffn(x, s["wg"], s["wu"], "silu", save=True)
    n, f = h.shape
    c = s["head"].shape[0]
    z, d_h, d_head = torch.empty(n, c, device=DEV), torch.empty(n, f, device=DEV), torch.empty(c, f, device=DEV)
    gemm(h, s["head"], z, n, c, f, (f, 1), (1, f), c)
    loss, d_z = ops.distill_loss_grad(z, s["tv"], s["ti"], s["w"], tau)
    gemm(d_z, s["head"], d_h, n, f, c, (c, 1), (f, 1), f)
    gemm(d_z, h, d_head, c, f, n, (1, c), (f, 1), f)
    d_x, d_wg, d_wu = ops.gated_ffn_grad(d_h, x, s["wg"], s["wu"], saved, "silu")
    d_table = ops.embedding_grad(d_x, s["ids"], s["table"].shape[0], 0.5)
    return {"loss": loss, "table": d_table, "wg": d_wg, "wu": d_wu, "head": d_head}


def student_plain(s, tau=2.0):
    """The same by autograd in 64 bits."""
    p = {k: s[k].double().requires_grad_() for k in ("table", "wg", "wu", "head")}
    ok = s["ids"] >= 0
    x = torch.where(ok[:, None], p["table"][s["ids"].clamp_min(0).long()] * 0.5, 0.0)
    g, u = x @ p["wg"].T, x @ p["wu"].T
    z = (torch.nn.functional.silu(g) * u) @ p["head"].T
    there = s["ti"] >= 0
    t = torch.where(there, s["tv"].double() / tau, -1e30)
    prob = torch.where(there, torch.softmax(t, 1), 0.0)
    logq = torch.log_softmax(z / tau, 1).gather(1, s["ti"].clamp_min(0).long())
    loss = tau * tau * torch.where(prob > 0, prob * (torch.log(prob.clamp_min(1e-300)) - logq), 0.0).sum(1)
    (loss * s["w"].double()).sum().backward()
    return {"loss": loss.detach(), **{k: v.grad for k, v in p.items()}}


def on_gpu(s):
    return {k: v.to(DEV) for k, v in s.items()}


def test_a_training_step_of_all_of_them(ops):
    """Errors of a chain of fp32 steps, each of about sqrt(length) roundings and none cancelling: 2^-24 * 64 of the largest value."""
    s = student(gen("step"))
    got, want = student_step(ops, on_gpu(s)), student_plain(s)
    for k in want:
        off = (got[k].double().cpu() - want[k]).abs().max() / want[k].abs().max()
        assert off < 64 * 2.0 ** -24, (k, float(off))


def test_training_step_against_differences(ops):
    """The table's gradient of the whole step against central differences of the step's own loss along one direction: step e of the
    direction's unit vector; truncation e^2 times a third derivative of order 1, the loss's noise 64 u |loss| over e."""
    g = gen("stepdiff")
    s = student(g)
    v = normal(g, *s["table"].shape)
    v /= v.norm()
    e = 2.0 ** -3
    weigh = lambda q: float((student_step(ops, on_gpu(q))["loss"].double().cpu() * s["w"].double()).sum())
    up, dn = weigh({**s, "table": s["table"] + e * v}), weigh({**s, "table": s["table"] - e * v})
    got = student_step(ops, on_gpu(s))
    slope = float((got["table"].double().cpu() * v.double()).sum())
    total = float((got["loss"].double().cpu() * s["w"].double()).sum())
    assert abs((up - dn) / (2 * e) - slope) <= e * e / 6 * 1.0 + 64 * 2.0 ** -24 * total / e


def test_on_another_stream(ops):
    s = on_gpu(student(gen("stream")))
    want = student_step(ops, s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = student_step(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_two_captured_graphs(ops):
    """Two steps captured each into a graph of its own, replayed in turn with eager work between: equal to the eager results, on
    changed inputs too."""
    sets = [on_gpu(student(gen("graph", i), tokens=150 + 57 * i, classes=90 + 11 * i)) for i in range(2)]
    pool = []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            student_step(ops, s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = student_step(ops, s)
        pool.append((graph, out))
    for turn in range(4):
        for s, (graph, out) in zip(sets, pool):
            want = {k: v.clone() for k, v in student_step(ops, s).items()}
            for v in out.values():
                v.fill_(-7)
            graph.replay()
            torch.cuda.synchronize()
            for k in want:
                assert torch.equal(out[k], want[k]), (turn, k)
        for s in sets:                       # the next turn's inputs, in place
            s["table"].mul_(0.9)
            s["ids"].copy_(s["ids"].roll(1))


def test_two_streams_at_once(ops):
    sets = [on_gpu(student(gen("two", i), tokens=400, rows=900)) for i in range(2)]
    want = [student_step(ops, s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(student_step(ops, sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for k in want[i]:
                assert torch.equal(r[k], want[i][k]), (i, k)
