"""Cross entropy (svae_cf_amd.ops) at sizes that take each of its kernels' forms, by the tolerances of tests/test_gpu_xent.py."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_xent import BF16, F16, F32, U, check, make

pytestmark = pytest.mark.gpu
TYPES = [BF16, F16, F32]


def takes_weight_as_it_lies(R, V, D, dtype):
    """Whether a call is one for the kernels for few rows: a loss over a weight at an odd address has no copy of it in its workspace."""
    from svae_cf_amd import _lib
    n = ctypes.c_longlong()
    _lib.call("svae_xent_bytes", 2, D, {F32: 0, BF16: 1, F16: 2}[dtype], R, V, D, 0, ctypes.byref(n))
    return n.value < 2 * V * D


# four tiles of rows at each division of the columns (up to 64, up to 128, more), and one tile against more than 2^19 entries
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,D", [(64, 131073, 64), (33, 140001, 61), (33, 100003, 96), (50, 90001, 97), (64, 65537, 128), (50, 40000, 260), (64, 12001, 700),
                                   (13, 600001, 33), (16, 530001, 20), (1, 700001, 13)])
def test_few_rows_against_large_weights(R, V, D, dtype):
    assert takes_weight_as_it_lies(R, V, D, dtype)
    check(*make(R, V, D, dtype, bias=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,D", [(64, 112001, 75), (47, 131329, 65), (64, 140001, 61), (39, 33001, 257)])
def test_four_tiles_of_rows_strides_masks_and_left_out_rows(R, V, D, dtype):
    """As test_few_rows_strides_masks_and_left_out_rows, where 16-bit types take the kernels for few rows too."""
    from svae_cf_amd import ops
    assert takes_weight_as_it_lies(R, V, D, dtype)
    h, w, b, t, wt = make(R, V, D, dtype, bias=True)
    b[100:900] = -float("inf")
    t = torch.where((t >= 100) & (t < 900), t % 100, t)
    t[3], t[4], wt[5] = -1, V, 0.0
    check(h, w, b, t, wt)
    want = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert bool((want[3][100:900] == 0).all()) and bool((want[4][100:900] == 0).all())
    wide_h, wide_w = torch.full((R, D + 6), float("nan"), dtype=dtype, device="cuda"), torch.full((V, D + 8), float("nan"), dtype=dtype, device="cuda")
    wide_h[:, 1:1 + D], wide_w[:, 3:3 + D] = h, w
    wide_h[3], wide_h[4], wt[3], wt[4] = float("nan"), float("inf"), float("inf"), float("nan")
    got = ops.linear_nll_grad(wide_h[:, 1:1 + D], wide_w[:, 3:3 + D], t.int(), wt, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    wide_h[5] = float("nan")                                       # weight 0: no part in the gradient, its loss is its own
    got = ops.linear_nll_grad(wide_h[:, 1:1 + D], wide_w[:, 3:3 + D], t, wt, bias=b)
    here = (t >= 0) & (t < V)                                      # (row 5 has no target in one of the sizes: no loss either)
    assert all(torch.equal(x, y) for x, y in zip(got[2:], want[2:])) and torch.isnan(got[0]).nonzero().view(-1).tolist() == ([5] if bool(here[5]) else [])
    every = ops.linear_nll_grad(wide_h[:, 1:1 + D], w, torch.full_like(t, -1), wt, bias=b)
    assert all(float(x.float().abs().max()) == 0 for x in every)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,D", [(60, 131329, 64), (60, 90001, 97), (13, 600001, 33)])
def test_confident_rows_against_large_weights(R, V, D, dtype):
    """Targets of a probability near 1, where errors of z and of lse cancel only if both come from the same bits."""
    assert takes_weight_as_it_lies(R, V, D, dtype)
    h, w, b, t, wt = make(R, V, D, dtype, bias=True, pad=0.0)
    t = torch.arange(R, device="cuda") * 7
    w[t] = (h.float() * (26 / D)).to(dtype)
    check(h, w, b, t, wt)


# 17 x 17 tiles of 128 rows: each width of a tile, one to four tiles of the width
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [40, 100, 150, 190, 200, 256, 300, 500, 1000])
def test_tiles_of_128_rows(D, dtype):
    check(*make(2100, 4100, D, dtype, bias=D % 3 == 1))


# G of a piece takes 128 MiB here: 62 tiles of the vocabulary for 4097 rows of 16 bits (20 of fp32), 11 for 21800 (several slabs of dW)
@pytest.mark.parametrize("R,V,D,dtype", [(4097, 40000, 300, BF16), (4097, 33000, 72, F16), (4097, 20001, 500, F16), (4097, 12000, 300, F32), (21800, 6000, 200, BF16),
                                         (21800, 8700, 90, F16), (21800, 3500, 130, F32)])
def test_several_pieces(R, V, D, dtype):
    check(*make(R, V, D, dtype, bias=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [12, 24, 150, 2000])
def test_light_rows(R, dtype):
    """Rows 2^20 lighter than others: w (softmax - onehot) has steps of 2^-38 of the largest weight in fp16 (of more than 16 rows), the
    other types' do not show."""
    h, w, b, t, wt = make(R, 700, 64, dtype, bias=True)
    wt[::3] *= 2.0 ** -20
    check(h, w, b, t, wt)


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
