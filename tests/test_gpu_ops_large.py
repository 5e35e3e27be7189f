"""graphslim_amd.ops on the GPU at the sizes that take the large tiles, sliced products, sorted tokens and rows past the caches, and at
offsets beyond 32 bits; the tolerances are those of tests/ops_reference.py."""
import pytest
import torch

import ops_reference as R
from test_gpu_ops import BF16, DEV, F16, F32, gen, normal, ops, strided, zipf  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu

# What each shape is for: the tile of 256 rows in the forward product (fwd), in dx and dW one after the other (dx, dw) or in one launch
# (pair), cut along k (/) or not; 16-bit rows that do not consist of whole chunks are laid out first, or read through registers (raw).
WIDE_16 = [(6000, 64, 700), (2050, 72, 2050), (2000, 75, 2100), (4100, 1035, 2050),   # fwd; rows that end inside a step of k; raw; laid out
           (6000, 4104, 16), (6000, 4100, 9),                       # dx; laid out
           (70, 4104, 8200), (70, 4100, 8200),                      # dw; laid out, forward raw and cut
           (700, 4104, 4104),                                       # dx/
           (1300, 4104, 1032), (1300, 4100, 1027),                  # pair; laid out, forward raw
           (4100, 4104, 9), (70, 2056, 4104), (70, 2060, 4100)]     # pair, dw/; pair, dx/; the same laid out
WIDE_32 = [(3000, 64, 700), (8200, 515, 9),                         # fwd; fwd/
           (3000, 4100, 9), (260, 1032, 8200),                      # dx, dw/; dx/
           (70, 515, 8200), (4100, 4100, 70),                       # dw; dw/
           (515, 4100, 260), (4100, 515, 9), (70, 515, 2056), (515, 64, 4100)]   # pair; dw/; dx/; both/


def gated_case(ops, M, D, F, dtype, place=lambda t: t.to(DEV)):
    g = gen("wide", M, D, F)
    act = ["silu", "gelu", "relu", "sigmoid"][(M + D + F) % 4]
    x, wg, wu = normal(g, M, D, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype), normal(g, F, D, std=D ** -0.5, dtype=dtype)
    d_h = normal(g, M, F, dtype=dtype)
    xd, wgd, wud, dd = (place(t) for t in (x, wg, wu, d_h))
    want = {key: tuple(t.cpu() for t in pair) for key, pair in R.gated(xd, wgd, wud, act, dd).items()}
    h, saved = ops.gated_ffn(xd, wgd, wud, act, save=True)
    R.within(h, want["h"], "h")
    R.within(saved, want["saved"], "saved")
    got = ops.gated_ffn_grad(dd, xd, wgd, wud, saved, act)
    for key, t in zip(("d_x", "d_w_gate", "d_w_up"), got):
        R.within(t, want[key], key)
    for _ in range(3):                    # waves that overtake each other would differ from run to run
        assert torch.equal(h, ops.gated_ffn(xd, wgd, wud, act)), "saving changes the result"
        for t, again in zip(got, ops.gated_ffn_grad(dd, xd, wgd, wud, saved, act)):
            assert torch.equal(t, again), "two runs differ"


@pytest.mark.parametrize("M,D,F", WIDE_16)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_wide_16(ops, M, D, F, dtype):
    gated_case(ops, M, D, F, dtype)


@pytest.mark.parametrize("M,D,F", WIDE_32)
def test_gated_wide_32(ops, M, D, F):
    gated_case(ops, M, D, F, F32)


@pytest.mark.parametrize("M,D,F", [(2000, 128, 2100), (130, 128, 70), (4100, 1032, 2050)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_wide_unaligned(ops, M, D, F, dtype):
    """Whole chunks in a row, but rows that begin anywhere: read through registers, read so in the small tile, laid out."""
    gated_case(ops, M, D, F, dtype, lambda t: strided(t, 3, 5))


@pytest.mark.parametrize("M,D,F", [(5, 1, 1), (40, 3, 70), (300, 7, 130), (9, 8, 130), (30, 9, 66), (260, 15, 300)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_gated_narrow(ops, M, D, F, dtype):
    gated_case(ops, M, D, F, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,F", [(8192, 3000, 600), (8193, 3000, 600), (262144, 700, 3), (262145, 700, 3), (300001, 40000, 8), (270000, 3, 130)])
def test_embedding_grad_many_tokens(ops, n, V, F, dtype):
    g = gen("many", n, V, F)
    d, ids = normal(g, n, F, dtype=dtype), zipf(g, n, V)
    got = ops.embedding_grad(d.to(DEV), ids.to(DEV), V, 0.3)
    R.within(got, R.embedding_grad(d, ids, V, 0.3, dtype), "gradient")
    assert torch.equal(got, ops.embedding_grad(d.to(DEV), ids.to(DEV), V, 0.3)), "two runs differ"


@pytest.mark.parametrize("dtype,n,V", [(BF16, 2100, 32000), (F32, 1010, 32001), (F32, 600, 60001), (F16, 1100, 60003), (BF16, 600, 120001)])
def test_distill_past_the_caches(ops, dtype, n, V):
    """More logits than the caches keep take other loads and stores: the same bits as a few rows at a time, a few rows checked."""
    g = gen("past", n, V)
    tau, k = 2.0, 9
    z = torch.randn(n, V, device=DEV, generator=torch.Generator(DEV).manual_seed(V)).to(dtype) * 3
    tv = normal(g, n, k, std=3.0, dtype=dtype).to(DEV)
    ti = torch.randint(-1, V, (n, k), generator=g, dtype=torch.int32).to(DEV)
    w = (torch.rand(n, generator=g) + 0.1).to(DEV)
    loss, grad = ops.distill_loss_grad(z, tv, ti, w, tau)
    for at in range(0, n, 300):
        part = slice(at, min(at + 300, n))
        few, few_grad = ops.distill_loss_grad(z[part], tv[part], ti[part], w[part], tau)
        assert torch.equal(loss[part], few) and torch.equal(grad[part], few_grad)
    some = torch.cat([torch.arange(5), torch.randint(0, n, (10,), generator=g), torch.tensor([n - 1])])
    want = R.distill(z[some].cpu(), tv[some].cpu(), ti[some].cpu(), tau, w[some].cpu())
    R.within(loss[some], want["loss"], "loss")
    R.within(grad[some], want["d_logits"], "gradient")
    ops.distill_loss_grad(z, tv, ti, w, tau, out=z)
    assert torch.equal(z, grad), "in place"


# ---- offsets beyond 32 bits ----------------------------------------------------------------------------------------------------------
def test_embedding_beyond_32_bits(ops):
    V, F, n = 2_200_000, 1000, 3000
    g = gen("far")
    table = torch.zeros(V, F, dtype=BF16, device=DEV)
    rows = torch.cat([torch.tensor([V - 1, V - 2, 2147483, 2147484, 2147485]), torch.randint(0, V, (n - 5,), generator=g)])
    values = normal(g, n, F, dtype=BF16).to(DEV)
    table[rows.to(DEV)] = values
    ids = rows.to(torch.int32).to(DEV)
    assert torch.equal(ops.embedding(table, ids), table[rows.to(DEV)])
    R.within(ops.embedding_grad(values, ids, V, 0.5)[rows.unique().to(DEV)],
             tuple(t[rows.unique()] for t in R.embedding_grad(values.cpu(), ids.cpu(), V, 0.5, BF16)), "gradient")


def test_gated_beyond_32_bits(ops):
    """saved has 2 x 2^31 elements and more; rows at the end are as those of a call of their own."""
    M, D, F = 70000, 64, 32768
    g = gen("far gated")
    x, wg, wu = (normal(g, a, D, std=0.3, dtype=BF16).to(DEV) for a in (M, F, F))
    h, saved = ops.gated_ffn(x, wg, wu, "silu", save=True)
    tail = slice(M - 3000, M)
    few, few_saved = ops.gated_ffn(x[tail], wg, wu, "silu", save=True)
    assert torch.equal(h[tail], few) and torch.equal(saved[:, tail], few_saved)
    d_h = torch.zeros_like(h)
    d_h[tail] = h[tail]
    d_x = ops.gated_ffn_grad(d_h, x, wg, wu, saved)[0]
    assert not d_x[:M - 3000].any()
    want = R.gated(x[tail], wg, wu, "silu", d_h[tail])["d_x"]
    R.within(d_x[tail], tuple(t.cpu() for t in want), "d_x")


def test_distill_beyond_32_bits(ops):
    n, V, k = 70000, 32000, 4
    g = gen("far distill")
    z = torch.zeros(n, V, dtype=BF16, device=DEV)
    tail = slice(n - 40, n)
    end = normal(g, 40, V, std=3.0, dtype=BF16)
    z[tail] = end.to(DEV)
    tv = normal(g, n, k, dtype=BF16).to(DEV)
    ti = torch.randint(0, V, (n, k), generator=g, dtype=torch.int32).to(DEV)
    w = torch.ones(n, device=DEV)
    want = R.distill(end, tv[tail].cpu(), ti[tail].cpu(), 1.0, w[tail].cpu())
    loss, grad = ops.distill_loss_grad(z, tv, ti, w)
    R.within(loss[tail], want["loss"], "loss")
    R.within(grad[tail], want["d_logits"], "gradient")
    other, lse = ops.distill(z, tv, ti)
    R.within(other[tail], want["loss"], "loss alone")
    want = R.distill(end, tv[tail].cpu(), ti[tail].cpu(), 1.0, w[tail].cpu(), lse[tail].cpu())
    R.within(ops.distill_grad(z, tv, ti, lse, w, out=z)[tail], want["d_logits"], "gradient in place")
