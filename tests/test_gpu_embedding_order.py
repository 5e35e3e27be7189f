"""The order in which the table's gradient is summed: partial sums of consecutive tokens, cut where the ids and sizes say, bit for bit."""
import numpy as np
import pytest
import torch

from test_gpu_ops import DEV, gen, normal, ops, zipf  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu


def parts(rows, d, waves):
    """{row: its sum} over tokens that are sorted by row: cut into `waves` parts of about equal length, each row's tokens of a part summed
    one after the other, then the parts' sums."""
    n, out = len(rows), {}
    for g in range(waves):
        sums = {}
        for i in range(n * g // waves, n * (g + 1) // waves):
            sums[rows[i]] = sums.get(rows[i], np.zeros_like(d[0])) + d[i]
        for r, s in sums.items():
            out[r] = out[r] + s if r in out else s
    return out


def summed(d, ids, V):
    """The gradient in fp32 on the host, a bucket of the table's rows after the other."""
    d, ids = d.numpy(), ids.numpy()
    n, F = d.shape
    lanes = 64 * (4 if F >= 256 else 2 if F >= 128 else 1)          # columns of a wave; the other waves of a workgroup share the tokens
    most = 16 if 512 < n <= 8192 else 8
    beside = 1
    while beside < most and beside * lanes < F:
        beside *= 2
    if n <= 8192:
        R, span = min(max(-(-V // (1024 if n <= 512 else 256)), 4), 64), n
    else:
        R, span = 4, 256
        while -(-V // R) > 1024 and R < 64:
            R *= 2
    out = np.zeros((V, F), np.float32)
    for row0 in range(0, V, R):
        mine = np.flatnonzero((ids >= row0) & (ids < min(row0 + R, V)))
        for s in range(0, len(mine), max(span, 1)):
            t = mine[s:s + span]
            t = t[np.argsort(ids[t], kind="stable")]
            for r, v in parts(ids[t], d[t], most // beside).items():
                out[r] = out[r] + v
    return torch.from_numpy(out)


@pytest.mark.parametrize("n,V,F", [(40, 9, 4), (500, 30, 200), (3000, 300, 5), (5001, 1007, 130), (9000, 7, 3), (12000, 900, 300)])
def test_the_order_of_the_sum(ops, n, V, F):
    g = gen("order", n, V, F)
    d, ids = normal(g, n, F) * torch.exp(4 * torch.randn(n, 1, generator=g)), zipf(g, n, V)
    got = ops.embedding_grad(d.to(DEV), ids.to(DEV), V).cpu()
    assert torch.equal(got, summed(d, ids, V))


def test_terms_that_cancel(ops):
    """2^24, then ones that a sum beginning there loses, then -2^24: eight parts of 37 or 38 keep those of all but the first."""
    d = torch.ones(300, 4)
    d[0], d[299] = 2.0 ** 24, -2.0 ** 24
    ids = torch.zeros(300, dtype=torch.int32)
    want = summed(d, ids, 3)
    assert (want[0] == want[0, 0]).all() and 200 < want[0, 0] < 299 and not want[1:].any()
    assert torch.equal(ops.embedding_grad(d.to(DEV), ids.to(DEV), 3).cpu(), want)
