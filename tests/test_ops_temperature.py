"""Temperatures that fp32 holds no factor log2(e) / tau for are refused, by graphslim_amd.ops and by the C entry points.  No GPU."""
import pytest
import torch

from test_ops import L, ops  # noqa: F401 (fixtures)

BAD = [4.2e-39, 3e-39, 1e-46, 1e39]
GOOD = [4.3e-39, 1e-30, 1.0, 3.4e38]


def test_python(ops):
    z, tv, ti = torch.zeros(3, 9), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    for tau in BAD:
        with pytest.raises(ValueError, match="temperature"):
            ops.distill(z, tv, ti, tau)
    for tau in GOOD:
        with pytest.raises(AssertionError, match="was reached"):
            ops.distill(z, tv, ti, tau)


def test_c(L):
    buf = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20]
    for tau in BAD:
        assert L.gs_distill_fwd(buf[0], 9, 0, 3, 9, buf[1], buf[2], 2, tau, buf[3], buf[4], None) == -1 and b"temperature" in L.gs_last_error()
    for tau in GOOD:                                     # (no rows: nothing is launched)
        assert L.gs_distill_fwd(buf[0], 9, 0, 0, 9, buf[1], buf[2], 2, tau, buf[3], buf[4], None) == 0
