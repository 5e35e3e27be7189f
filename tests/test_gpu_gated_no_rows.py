"""The gradient of no tokens is zero, whatever the weights' size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,F,D", [(torch.bfloat16, 70000, 64000), (torch.float32, 5, 3), (torch.float16, 4097, 4099)])
def test_zero_gradient(dtype, F, D):
    """70000 x 64000 are more than 2^32 elements, one a thread no longer."""
    from graphslim_amd import ops
    dev = "cuda:0"
    w = torch.empty(F, D, dtype=dtype, device=dev)
    junk = torch.full((F, D), 7.0, dtype=dtype, device=dev)        # (what the allocator hands out next is not zero by itself)
    del junk
    x, d_h = torch.empty(0, D, dtype=dtype, device=dev), torch.empty(0, F, dtype=dtype, device=dev)
    saved = torch.empty(2, 0, F, device=dev)
    d_x, d_wg, d_wu = ops.gated_ffn_grad(d_h, x, w, w, saved)
    assert d_x.shape == (0, D)
    for t in (d_wg, d_wu):
        assert t.shape == (F, D)
        for at in range(0, F, 10000):
            assert not t[at:at + 10000].any()
