"""Cross entropy (svae_cf_amd.ops) at sizes that take each of its kernels' forms, by the tolerances of tests/test_gpu_xent.py."""
import numpy as np
import pytest
import torch

from test_gpu_xent import BF16, F16, F32, U, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V", [(1000, 65536 * 256 + 7000), (300000, 65536)])
def test_loss_whose_statistics_are_joined_in_several_goes(R, V):
    """More than 512 MiB of them, few rows and many.  Logits that are the bias alone: every sum is known."""
    from svae_cf_amd import ops
    b = torch.zeros(V, dtype=BF16, device="cuda")
    b[[5, V // 2, V - 1]] = torch.tensor([2.0, 4.0, 6.0], device="cuda").to(BF16)
    t = torch.arange(R, device="cuda", dtype=torch.int32) * max(1, V // R) % V
    t[:3] = torch.tensor([5, V // 2, V - 1])
    h, w = torch.randn(R, 8, device="cuda").to(BF16), torch.zeros(V, 8, dtype=BF16, device="cuda")
    nll, lse = ops.linear_nll(h, w, t, bias=b)
    want = np.log(V - 3 + np.exp(2.0) + np.exp(4.0) + np.exp(6.0))
    tol = (V / 16384 + 200) * U + 2.0 ** -22 + 2 * U * want        # as in test_loss_of_more_tiles_than_a_launch_takes
    assert float((lse.double() - want).abs().max()) <= tol
    assert float((nll.double() - (want - b.double()[t.long()])).abs().max()) <= tol + U * want
    wt = torch.full((R,), 1.0 / R, device="cuda")
    got = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert torch.equal(got[0], nll) and torch.equal(got[1], lse)
