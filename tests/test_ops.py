"""What graphslim_amd.ops and its C entry points refuse, without a GPU; and the 64-bit reference of the GPU tests against differences."""
import math
import os
import subprocess

import pytest
import torch

import ops_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def L():
    from graphslim_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        subprocess.run(["make", "-C", os.path.join(ROOT, "graphslim_amd", "csrc"), "-j4"], check=True)
    return _lib.lib()


@pytest.fixture()
def ops(monkeypatch):
    """The module with its device check off, so that a CPU tensor reaches the checks behind it; nothing here reaches a launch."""
    from graphslim_amd import ops

    class NoLaunch:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(ops, "_device", lambda **t: torch.device("cpu"))
    monkeypatch.setattr(ops._lib, "lib", lambda: NoLaunch())
    return ops


def test_cpu_tensors_are_refused():
    from graphslim_amd import ops
    w, ids = torch.zeros(3, 4), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.embedding(w, ids), lambda: ops.embedding_grad(w[:2], ids, 3), lambda: ops.gated_ffn(w, w, w),
                 lambda: ops.gated_ffn_grad(w, w, w, w, w), lambda: ops.distill(w, w[:, :1], torch.zeros(3, 1, dtype=torch.int32)),
                 lambda: ops.embedding([1.0], ids)):
        with pytest.raises(ValueError, match="no CPU path|is a tensor"):
            call()


def test_embedding_refusals(ops):
    w, ids = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32)
    for match, call in [("int32", lambda: ops.embedding(w, ids.long())), ("dense", lambda: ops.embedding(w, torch.zeros(6, dtype=torch.int32)[::2])),
                        ("two dimensions", lambda: ops.embedding(w[0], ids)), ("not dense", lambda: ops.embedding(w.T, ids)),
                        ("fp32, fp16 or bf16", lambda: ops.embedding(w.double(), ids)), ("no rows", lambda: ops.embedding(w[:0], ids)),
                        ("no columns", lambda: ops.embedding(w[:, :0], ids)), ("overlap", lambda: ops.embedding(w[:1].expand(5, 4), ids)),
                        ("columns", lambda: ops.embedding(w, ids, out=torch.zeros(3, 5))), ("rows", lambda: ops.embedding(w, ids, out=torch.zeros(4, 4))),
                        ("other arguments", lambda: ops.embedding(w, ids, out=torch.zeros(3, 4, dtype=F16)))]:
        with pytest.raises(ValueError, match=match):
            call()
    d = torch.zeros(3, 4)
    for match, call in [("int32", lambda: ops.embedding_grad(d, ids.long(), 5)), ("rows", lambda: ops.embedding_grad(d[:2], ids, 5)),
                        ("a table of 0 rows", lambda: ops.embedding_grad(d, ids, 0)), ("missing", lambda: ops.embedding_grad(d, ids, 5, accumulate=True)),
                        ("or torch.float32", lambda: ops.embedding_grad(d, ids, 5, dtype=F16)),
                        ("or torch.float32", lambda: ops.embedding_grad(d, ids, 5, out=torch.zeros(5, 4, dtype=BF16))),
                        ("dtype", lambda: ops.embedding_grad(d, ids, 5, out=torch.zeros(5, 4), dtype=F16)),
                        ("columns", lambda: ops.embedding_grad(d, ids, 5, out=torch.zeros(5, 3))),
                        ("d_out is", lambda: ops.embedding_grad(torch.zeros(2, 3, 4), ids, 5)),
                        ("dense, or a matrix", lambda: ops.embedding_grad(torch.zeros(3, 2, 4).transpose(0, 1)[:, :, :], torch.zeros(2, 3, dtype=torch.int32), 5))]:
        with pytest.raises(ValueError, match=match):
            call()


def test_gated_refusals(ops):
    x, w = torch.zeros(3, 4), torch.zeros(6, 4)
    for match, call in [("act is one of", lambda: ops.gated_ffn(x, w, w, "swish")), ("columns", lambda: ops.gated_ffn(x, w[:, :3], w[:, :3])),
                        ("rows", lambda: ops.gated_ffn(x, w, w[:5])), ("other arguments", lambda: ops.gated_ffn(x, w.half(), w)),
                        ("one row stride", lambda: ops.gated_ffn(x, torch.zeros(6, 5)[:, :4], w)), ("no rows", lambda: ops.gated_ffn(x, w[:0], w[:0])),
                        ("two dimensions", lambda: ops.gated_ffn(x[None], w, w)), ("not dense", lambda: ops.gated_ffn(torch.zeros(4, 3).T, w, w))]:
        with pytest.raises(ValueError, match=match):
            call()
    d_h, saved = torch.zeros(3, 6), torch.zeros(2, 3, 6)
    for match, call in [("columns", lambda: ops.gated_ffn_grad(d_h[:, :5], x, w, w, saved)), ("saved is what", lambda: ops.gated_ffn_grad(d_h, x, w, w, saved[:, :2])),
                        ("saved is what", lambda: ops.gated_ffn_grad(d_h, x, w, w, saved.half())),
                        ("other arguments", lambda: ops.gated_ffn_grad(d_h.half(), x, w, w, saved))]:
        with pytest.raises(ValueError, match=match):
            call()


def test_shared_and_broadcast_rows_are_refused(ops):
    """A broadcast gradient or input has rows that overlap: it is made dense by the caller, not read with a stride of 0."""
    w, ids = torch.zeros(6, 4), torch.zeros(3, dtype=torch.int32)
    row = torch.zeros(1, 4)
    for call in (lambda: ops.embedding_grad(row.expand(3, 4), ids, 5), lambda: ops.gated_ffn(row.expand(3, 4), w, w),
                 lambda: ops.gated_ffn(row.expand(3, 4), w, row.expand(6, 4)),
                 lambda: ops.distill(row.expand(3, 4), torch.zeros(3, 1), torch.zeros(3, 1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="overlap"):
            call()


def test_distill_refusals(ops):
    z, tv, ti, v = torch.zeros(3, 9), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3)
    for match, call in [("one row a row", lambda: ops.distill(z, tv[:2], ti)), ("top_values are", lambda: ops.distill(z, tv.half(), ti)),
                        ("top_ids are", lambda: ops.distill(z, tv, ti[:, :1])), ("int32", lambda: ops.distill(z, tv, ti.long())),
                        ("teacher entries", lambda: ops.distill(z, torch.zeros(3, 0), torch.zeros(3, 0, dtype=torch.int32))),
                        ("teacher entries", lambda: ops.distill(z, torch.zeros(3, 1025), torch.zeros(3, 1025, dtype=torch.int32))),
                        ("temperature", lambda: ops.distill(z, tv, ti, 0.0)), ("temperature", lambda: ops.distill(z, tv, ti, -1.0)),
                        ("temperature", lambda: ops.distill(z, tv, ti, math.nan)), ("temperature", lambda: ops.distill(z, tv, ti, math.inf)),
                        ("dense vector", lambda: ops.distill_grad(z, tv, ti, v[:2], v)), ("dense vector", lambda: ops.distill_loss_grad(z, tv, ti, v[:1].expand(3))),
                        ("float32", lambda: ops.distill_loss_grad(z, tv, ti, v.half())), ("columns", lambda: ops.distill_loss_grad(z, tv, ti, v, out=torch.zeros(3, 8))),
                        ("other arguments", lambda: ops.distill_loss_grad(z, tv, ti, v, out=z.half()))]:
        with pytest.raises(ValueError, match=match):
            call()


def test_c_entry_points_refuse(L):
    """Argument checks come before any GPU call: they answer here, with a message, and never end the process."""
    ARG, UNSUPPORTED = -1, -4
    N = None
    assert L.gs_embedding_fwd(N, 4, 5, 4, 7, N, 3, 1.0, N, 4, N) == ARG and b"element type" in L.gs_last_error()
    assert L.gs_embedding_fwd(N, 3, 5, 4, 0, N, 3, 1.0, N, 4, N) == ARG and b"stride" in L.gs_last_error()
    assert L.gs_embedding_fwd(N, 4, 5, 4, 0, N, 3, 1.0, N, 4, N) == ARG and b"null" in L.gs_last_error()
    assert L.gs_embedding_fwd(N, 4, 5, 4, 0, N, 0, 1.0, N, 4, N) == 0
    assert L.gs_embedding_fwd(N, 4, 1 << 33, 4, 0, N, 3, 1.0, N, 4, N) == UNSUPPORTED
    assert L.gs_embedding_bwd(N, 4, 1, N, 3, 5, 4, 1.0, 0, N, 4, 2, N, N) == ARG and b"type of d_out" in L.gs_last_error()
    assert L.gs_embedding_bwd(N, 4, 1, N, 3, 5, 4, 1.0, 0, N, 4, 0, N, N) == ARG
    assert L.gs_gated_fwd(N, 4, N, N, 4, 0, 2, 4, 6, 9, N, 6, N, N, N) == ARG and b"activation" in L.gs_last_error()
    assert L.gs_gated_fwd(N, 4, N, N, 3, 0, 2, 4, 6, 0, N, 6, N, N, N) == ARG
    assert L.gs_gated_fwd(N, 4, N, N, 4, 0, 2, 4, 6, 0, N, 5, N, N, N) == ARG
    assert L.gs_gated_fwd(N, 4, N, N, 4, 0, 2, 4, 6, 0, N, 6, N, N, N) == ARG and b"null" in L.gs_last_error()
    assert L.gs_gated_fwd(N, 4, N, N, 4, 0, 0, 4, 6, 0, N, 6, N, N, N) == 0
    assert L.gs_gated_bwd(N, 6, N, 4, N, N, 4, N, 0, 2, 4, 6, 0, N, 4, N, N, 4, N, N) == ARG
    assert L.gs_gated_fwd_scratch_bytes(0, 4, 6, 0, 1) == L.gs_gated_bwd_scratch_bytes(0, 4, 6, 1, 1) == 0
    assert L.gs_gated_fwd_scratch_bytes(-1, 4, 6, 0, 1) == 0 and L.gs_gated_fwd_scratch_bytes(2, 4, 6, 5, 1) == 0
    assert L.gs_distill_fwd(N, 9, 0, 3, 9, N, N, 2, 1.0, N, N, N) == ARG
    buf = 4096                                          # never read: the checks below come first
    assert L.gs_distill_fwd(buf, 9, 0, 3, 9, buf, buf, 1025, 1.0, buf, buf, N) == UNSUPPORTED
    assert L.gs_distill_fwd(buf, 9, 0, 3, 9, buf, buf, 2, 0.0, buf, buf, N) == ARG and b"temperature" in L.gs_last_error()
    assert L.gs_distill_fwd(buf, 8, 0, 3, 9, buf, buf, 2, 1.0, buf, buf, N) == ARG and b"stride" in L.gs_last_error()
    assert L.gs_distill_fwd(buf, 9, 0, 3, 9, buf, buf, 2, 1e-40, buf, buf, N) == ARG and b"reciprocal" in L.gs_last_error()
    assert L.gs_distill_loss_grad(buf, 12, 0, 3, 9, buf, buf, 2, 1.0, buf, buf, buf, 9, N) == ARG and b"in place" in L.gs_last_error()
    assert L.gs_distill_bwd(N, 9, 0, 3, 9, N, N, 2, 1.0, N, N, N, 9, N) == ARG
    assert L.gs_distill_loss_grad(N, 9, 0, 0, 9, N, N, 2, 1.0, N, N, N, 9, N) == 0


def test_scratch_sizes(L):
    """For every shape from one row to a large batch: enough for the laid-out operands, and no more than a small multiple of them."""
    for typ, parts in ((0, 3), (1, 1), (2, 1)):
        for M in (1, 5, 33, 128, 1000, 8192):
            for D, F in ((1, 1), (64, 64), (500, 1024), (1433, 4096), (2048, 8192)):
                up = lambda n: (n + 63) // 64 * 64
                slopes = up(M) * 2 * up(F) * 2 * parts
                bwd = L.gs_gated_bwd_scratch_bytes(M, D, F, typ, 1)
                assert bwd >= slopes
                laid = slopes + (parts > 1) * (up(M) + 2 * up(F)) * up(D) * 2 * parts
                outputs = 4 * (M * D + 2 * up(F) * D)
                assert bwd <= laid + 64 * outputs, (typ, M, D, F, bwd)
                fwd = L.gs_gated_fwd_scratch_bytes(M, D, F, typ, 1)
                assert fwd <= (parts > 1) * (up(M) + 2 * up(F)) * up(D) * 2 * parts + 64 * 8 * M * F
                copies = (typ > 0) * (up(M) + 2 * up(F)) * up(D) * 2      # of 16-bit operands whose rows are not whole chunks
                assert L.gs_gated_bwd_scratch_bytes(M, D, F, typ, 0) == bwd + copies
                assert L.gs_gated_fwd_scratch_bytes(M, D, F, typ, 0) - fwd in (0, copies)


def _slope(f, x, v, e=1e-6):
    return (f(x + e * v) - f(x - e * v)) / (2 * e)


@pytest.mark.parametrize("name", ["silu", "gelu", "relu", "sigmoid"])
def test_reference_gradients_against_differences(name):
    """Central differences in 64 bits: 1e-12 of truncation and 1e-16 / 1e-6 of rounding per unit of the value."""
    g = torch.Generator().manual_seed(3)
    x, wg, wu, d = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (6, 7), (6, 7), (5, 6)))
    full = lambda x, wg, wu: (lambda a, u: (a * u * d).sum())(R.act(name, x @ wg.T)[0], x @ wu.T)
    ref = R.gated(x.float(), wg.float(), wu.float(), name, d.float())
    x, wg, wu, d = (t.float().double() for t in (x, wg, wu, d))
    for key, at, f in (("d_x", x, lambda t: full(t, wg, wu)), ("d_w_gate", wg, lambda t: full(x, t, wu)), ("d_w_up", wu, lambda t: full(x, wg, t))):
        v = torch.randn(at.shape, generator=g, dtype=torch.float64)
        assert abs(_slope(f, at, v) - (ref[key][0] * v).sum()) < 1e-7


def test_reference_distill_gradient_against_differences():
    g = torch.Generator().manual_seed(4)
    z, tv = torch.randn(4, 30, generator=g), torch.randn(4, 5, generator=g)
    ti = torch.randint(-1, 30, (4, 5), generator=g, dtype=torch.int32)
    w = torch.rand(4, generator=g)
    ref = R.distill(z, tv, ti, 1.5, w)["d_logits"][0]
    z, v = z.double(), torch.randn(4, 30, generator=g, dtype=torch.float64)
    f = lambda t: (R.distill(t, tv, ti, 1.5)["loss"][0] * w.double()).sum()
    assert abs(_slope(f, z, v) - (ref * v).sum()) < 1e-7
