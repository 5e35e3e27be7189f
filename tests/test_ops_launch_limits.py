"""A launch has fewer than 2^32 threads: sizes that need more are refused before anything is launched.  No GPU."""
from test_ops import L  # noqa: F401 (a fixture)

UNSUPPORTED = -4
A = [(i + 1) << 40 for i in range(8)]


def test_few_rows_of_many_weights(L):
    """Eight weights a workgroup of 256 threads: 2^24 workgroups are one too many."""
    for typ, M in ((0, 24), (1, 4), (2, 1)):
        assert L.gs_gated_fwd(A[0], 1, A[1], A[2], 1, typ, M, 1, 8 * (1 << 24) - 7, 0, A[3], 1 << 30, None, None, None) == UNSUPPORTED
        assert b"beyond one launch" in L.gs_last_error()


def test_many_ids(L):
    """A workgroup of 512 threads per 256 ids and one per bucket of rows."""
    n = 2 ** 31 - 1
    assert L.gs_embedding_bwd(A[0], 1, 0, A[1], n, 5000, 1, 1.0, 0, A[2], 1, 0, A[3], None) == UNSUPPORTED
    assert b"beyond one launch" in L.gs_last_error()
