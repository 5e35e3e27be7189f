"""Outputs that lie on other operands are refused, by graphslim_amd.ops and by the C entry points; neighbours are not.  No GPU."""
import random

import pytest
import torch

from test_ops import F16, F32, L, ops  # noqa: F401 (fixtures)

ARG = -1


def elements(at, rows, ld, cols):
    return {at + r * ld + c for r in range(rows) for c in range(cols)}


def reaches_the_launch(call):
    with pytest.raises(AssertionError, match="was reached"):
        call()


def test_embedding_out(ops):
    buf, ids = torch.zeros(400), torch.zeros(3, dtype=torch.int32)
    table = buf[:40].view(10, 4)
    for match, out in [("table", buf[:12].view(3, 4)), ("table", buf[39:51].view(3, 4)), ("table", buf[36:48].view(3, 4))]:
        with pytest.raises(ValueError, match=f"out lies on {match}"):
            ops.embedding(table, ids, out=out)
    reaches_the_launch(lambda: ops.embedding(table, ids, out=buf[40:52].view(3, 4)))
    wide = torch.zeros(10, 8)
    reaches_the_launch(lambda: ops.embedding(wide[:, :4], ids, out=wide[:3, 4:]))
    with pytest.raises(ValueError, match="lies on table"):
        ops.embedding(wide[:, :4], ids, out=wide[:3, 3:7])
    words = torch.zeros(64)
    with pytest.raises(ValueError, match="lies on ids"):
        ops.embedding(table, words.view(torch.int32)[2:5], out=words[:12].view(3, 4))


def test_embedding_grad_out(ops):
    buf, ids = torch.zeros(400), torch.zeros(5, dtype=torch.int32)
    d = buf[:20].view(5, 4)
    for out in (buf[:24].view(6, 4), buf[19:43].view(6, 4)):
        with pytest.raises(ValueError, match="lies on d_out"):
            ops.embedding_grad(d, ids, 6, out=out, accumulate=True)
    reaches_the_launch(lambda: ops.embedding_grad(d, ids, 6, out=buf[20:44].view(6, 4)))


def test_distill_out(ops):
    n, V, k = 4, 9, 2
    buf = torch.zeros(200)
    z, w, ti = buf[:36].view(n, V), buf[150:154], torch.zeros(n, k, dtype=torch.int32)
    tv = buf[160:168].view(n, k)
    for match, out in [("logits", buf[1:37].view(n, V)), ("logits", buf[35:71].view(n, V)), ("logits", buf[:40].view(n, V + 1)[:, :V]),
                       ("top_values", buf[126:162].view(n, V)), ("d_loss", buf[118:154].view(n, V))]:
        for call in (lambda: ops.distill_loss_grad(z, tv, ti, w, out=out), lambda: ops.distill_grad(z, tv, ti, torch.zeros(n), w, out=out)):
            with pytest.raises(ValueError, match=f"lies on {match}"):
                call()
    reaches_the_launch(lambda: ops.distill_loss_grad(z, tv, ti, w, out=z))
    reaches_the_launch(lambda: ops.distill_loss_grad(z, tv, ti, w, out=buf[36:72].view(n, V)))
    both = torch.zeros(n, 2 * V)
    reaches_the_launch(lambda: ops.distill_loss_grad(both[:, :V], tv, ti, w, out=both[:, V:]))
    reaches_the_launch(lambda: ops.distill_loss_grad(both[:, V:], tv, ti, w, out=both[:, :V]))
    with pytest.raises(ValueError, match="lies on logits"):
        ops.distill_loss_grad(both[:, :V], tv, ti, w, out=both[:, V - 1:-1])
    reaches_the_launch(lambda: ops.distill_loss_grad(both[1:2, :V], tv[:1], ti[:1], w[:1], out=both[1:2, V:]))


def test_apart_against_sets(ops):
    """One row stride or single rows: exactly the pairs that share an element; other strides: those, and pairs that are interwoven."""
    rng = random.Random(5)
    buf = torch.zeros(200)
    for _ in range(3000):
        n, m, a, b = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 6), rng.randint(1, 6)
        s = rng.randint(max(a, b), 12)
        r = s if rng.random() < 0.7 else rng.randint(b, 12)
        p, q = rng.randint(0, 60), rng.randint(0, 60)
        out, t = (torch.as_strided(buf, (rows, c), (ld, 1), at) for rows, c, ld, at in ((n, a, s, p), (m, b, r, q)))
        ld, lt = (s if n > 1 else a), (r if m > 1 else b)
        share = bool(elements(p, n, ld, a) & elements(q, m, lt, b))
        try:
            ops._apart(out, ld, t=(t, lt))
            refused = False
        except ValueError:
            refused = True
        assert refused or not share, (n, m, a, b, s, r, p, q)
        if n == 1 or m == 1 or s == r:
            assert refused == share, (n, m, a, b, s, r, p, q)


def test_c_outputs_against_sets(L):
    """gs_gated_fwd's h against x, by calls whose scratch is misaligned: refused in any case, for the first reason that is found."""
    rng = random.Random(6)
    for _ in range(3000):
        M, D, F = rng.randint(25, 27), rng.randint(1, 6), rng.randint(1, 6)
        ld = rng.randint(max(D, F), 12)
        ldx = ld if rng.random() < 0.7 else rng.randint(D, 12)
        p, q = rng.randint(0, 400), rng.randint(0, 400)
        assert L.gs_gated_fwd(4 * (10 ** 6 + q), ldx, 64, 1024, D, 0, M, D, F, 0, 4 * (10 ** 6 + p), ld, None, 8, None) == ARG
        said = L.gs_last_error()
        refused = b"lies on another operand" in said
        assert refused or b"16-byte aligned" in said
        share = bool(elements(p, M, ld, F) & elements(q, M, ldx, D))
        assert refused or not share
        if ld == ldx:
            assert refused == share, (M, D, F, ld, p, q)


def test_c_refusals(L):
    A, B, C, D, E, G = (1 << 20) * 1, (1 << 20) * 2, (1 << 20) * 3, (1 << 20) * 4, (1 << 20) * 5, (1 << 20) * 6
    lies = lambda rc: rc == ARG and b"lies on another operand" in L.gs_last_error()
    assert lies(L.gs_embedding_fwd(A, 4, 5, 4, 0, B, 3, 1.0, A + 16, 4, None))
    assert lies(L.gs_embedding_fwd(A, 4, 5, 4, 0, B, 3, 1.0, B - 16, 4, None))
    assert lies(L.gs_embedding_bwd(A, 4, 0, B, 3, 5, 4, 1.0, 0, A, 4, 0, C, None))
    assert lies(L.gs_distill_loss_grad(A, 9, 0, 3, 9, B, C, 2, 1.0, D, E, A + 4, 9, None))
    assert lies(L.gs_distill_loss_grad(A, 9, 0, 3, 9, B, C, 2, 1.0, D, A, G, 9, None))
    assert lies(L.gs_distill_loss_grad(A, 9, 0, 3, 9, B, C, 2, 1.0, D, E, D - 8, 9, None))
    assert lies(L.gs_distill_loss_grad(A, 9, 0, 3, 9, B, C, 2, 1.0, D, G, G, 9, None))
    assert lies(L.gs_distill_bwd(A, 9, 0, 3, 9, B, C, 2, 1.0, D, E, D, 9, None))
    assert lies(L.gs_distill_fwd(A, 9, 0, 3, 9, B, C, 2, 1.0, D, D + 4, None))
    assert lies(L.gs_gated_fwd(A, 4, B, B, 4, 0, 2, 4, 6, 0, C, 6, C + 16, None, None))
    assert lies(L.gs_gated_fwd(A, 4, B, B, 4, 0, 2, 4, 6, 0, C, 6, A, None, None))
    assert lies(L.gs_gated_bwd(A, 6, B, 4, C, C, 4, D, 0, 2, 4, 6, 0, B, 4, E, G, 4, 1 << 24, None))
    assert lies(L.gs_gated_bwd(A, 6, B, 4, C, C, 4, D, 0, 2, 4, 6, 0, G, 4, E, E, 4, 1 << 24, None))
