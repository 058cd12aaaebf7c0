"""Cross entropy (svae_cf_amd.ops) with entries of the vocabulary masked by large finite numbers, over whole tiles of it and over all
of it.  A masked entry is at least 9000 below the row's others, so its probability is below 2^-12000 and the result is that of -inf,
with the tolerances of tests/test_gpu_xent.py for that."""
import pytest
import torch

from test_gpu_xent import BF16, F16, F32, U, Ref, make, near

pytestmark = pytest.mark.gpu

VALUES = [(BF16, "lowest"), (BF16, -1e4), (BF16, -1e10), (BF16, -1e30), (F16, "lowest"), (F16, -1e4), (F32, "lowest"), (F32, -1e4), (F32, -1e10), (F32, -1e30)]
SIZES = [(6, 1500), (60, 131329), (200, 1500), (2000, 1500)]              # 60 rows: 2^23 numbers of weight, so few rows in every type


def value_of(dtype, value):
    return torch.finfo(dtype).min if value == "lowest" else value


@pytest.mark.parametrize("R,V", SIZES)
@pytest.mark.parametrize("dtype,value", VALUES)
def test_masked_tiles(R, V, dtype, value):
    from svae_cf_amd import ops
    h, w, b, t, wt = make(R, V, 64, dtype, bias=True)
    at = torch.arange(V, device="cuda")
    out = (at < 600) | ((at >= 700) & (at < V - 300))
    live = at[~out]
    t = torch.where((t >= 0) & (t < V), live[t.clamp(0, V - 1) % len(live)], t)
    ref = Ref(h, w, b.masked_fill(out, -float("inf")), t, wt)
    b = b.masked_fill(out, value_of(dtype, value))
    nll, lse = ops.linear_nll(h, w, t, bias=b)
    near(nll, ref.nll, ref.tol_nll, "nll")
    near(lse, ref.lse_out, ref.tol_lse, "lse")
    nll2, lse2, dh, dw, db = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert torch.equal(nll, nll2) and torch.equal(lse, lse2)
    near(dh, ref.dh, ref.tol_dh, "dh")
    near(dw, ref.dw, ref.tol_dw, "dw")
    near(db, ref.db, ref.tol_db, "db")
    assert bool((dw[out] == 0).all()) and bool((db[out] == 0).all())
    # a target that is masked: a finite loss, the gradient of the rest.  nll is a difference of two fp32 numbers, one of them the
    # rounded sum of the mask and some logit below 100
    t[0] = 5
    nll, lse, dh, dw, _ = ops.linear_nll_grad(h, w, t, wt, bias=b)
    far = float(b[5])
    assert abs(float(nll[0]) + far) <= 4 * U * abs(far) + 200
    assert bool(torch.isfinite(lse).all()) and bool(torch.isfinite(dh.float()).all()) and bool(torch.isfinite(dw.float()).all())


@pytest.mark.parametrize("R,V", SIZES)
@pytest.mark.parametrize("dtype,value", VALUES)
def test_everything_masked(R, V, dtype, value):
    """All logits far from 0: lse is the mask and some logit below 100 more, in fp32; the loss is a difference of two such numbers."""
    from svae_cf_amd import ops
    h, w, _, t, wt = make(R, V, 64, dtype, bias=False)
    b = torch.full((V,), value_of(dtype, value), dtype=dtype, device="cuda")
    far = float(b[0])
    here = (t >= 0) & (t < V)
    nll, lse, dh, dw, db = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert bool(((lse[here].double() - far).abs() <= 100 + 2 * U * abs(far)).all()) and bool((nll.abs() <= 200 + 4 * U * abs(far)).all())
    assert all(bool(torch.isfinite(x.float()).all()) for x in (dh, dw, db))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", SIZES)
@pytest.mark.parametrize("shift", [100.0, -130.0, -30000.0])
def test_logits_far_from_zero(shift, R, V, dtype):
    """A shift of all logits changes lse and nothing else.  The sums of z start from the bias, so each of their roundings counts it
    too: the tolerances are those of a column more, of ones in hidden and of the bias in weight."""
    from svae_cf_amd import ops
    h, w, _, t, wt = make(R, V, 64, dtype, bias=False)
    b = torch.full((V,), shift, dtype=dtype, device="cuda")
    ref = Ref(torch.cat((h, torch.ones_like(h[:, :1])), 1), torch.cat((w, b[:, None]), 1), None, t, wt)
    nll, lse, dh, dw, db = ops.linear_nll_grad(h, w, t, wt, bias=b)
    near(nll, ref.nll, ref.tol_nll, "nll")
    near(lse, ref.lse_out, ref.tol_lse, "lse")
    near(dh, ref.dh[:, :64], ref.tol_dh[:, :64], "dh")
    near(dw, ref.dw[:, :64], ref.tol_dw[:, :64], "dw")
    near(db, ref.dw[:, 64], ref.tol_dw[:, 64], "db")
