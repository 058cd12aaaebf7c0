"""Softmax cross entropy behind a linear layer (svae_cf_amd.ops) against the formulas in 64 bits.

Tolerances count roundings.  u = 2^-24, h = half a step of the inputs' type, |x| the matrix of magnitudes:
  z        sums of D exact products in fp32, in groups of at least 16: ez = (D / 16 + 64) u |H| |W|^T, + u |z|; fp32 inputs are three
           bf16 parts, of whose nine products the three smallest and the rests are left out: + 6 u |H| |W|^T, and six times the terms
  lse      max ez over the row + 2^-22 (exp and log, a unit each) + (V / 16384 + 200) u (sum of exponentials) + u |lse|
  G        w (p (ez + else + 2^-22 (1 + |z - lse|)) + u) + h |G| (rounded to the inputs' type) + half a subnormal step
  dH, dW   E_G |X| + (K / 16 + 64) u |G| |X| + h |result|"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


class Ref:
    def __init__(self, h, w, b, t, weight=None):
        self.dtype = h.dtype
        R, (V, D) = t.numel(), w.shape
        h, t = h.reshape(R, D).double(), t.reshape(-1).long()
        w = w.double()
        here = (t >= 0) & (t < V)
        at = torch.where(here, t, 0)
        h = torch.where(here[:, None], h, 0.0)
        split = self.dtype == F32
        mag = h.abs() @ w.abs().t()
        z = h @ w.t()
        z = z if b is None else z + b.double()
        ez = ((6 if split else 1) * D / 16 + 64 + (6 if split else 0)) * U * mag + U * z.abs().nan_to_num(posinf=0.0)
        self.lse = torch.logsumexp(z, 1)
        zt = z.gather(1, at[:, None])[:, 0]
        big = torch.where(z == -float("inf"), 0.0, ez).amax(1)
        elss = big + 2.0 ** -22 + (V / 16384 + 200) * U + U * self.lse.abs()
        self.nll = torch.where(here, self.lse - zt, 0.0)
        self.tol_lse = torch.where(here, elss, 0.0)
        self.tol_nll = torch.where(here, elss + big + 2 * U * zt.abs().nan_to_num(posinf=0.0), 0.0)
        self.lse_out = torch.where(here, self.lse, 0.0)
        if weight is None:
            return
        wr = torch.where(here, weight.reshape(-1).double(), 0.0)
        live = (wr != 0)[:, None]
        h = torch.where(live, h, 0.0)
        p = torch.exp(z - self.lse[:, None])
        x = (z - self.lse[:, None]).abs().nan_to_num(posinf=0.0)
        g = p.clone()
        g[torch.arange(R, device=g.device), at] -= 1
        g = torch.where(live, g * wr[:, None], 0.0)
        # half a subnormal step: of G's type after its scale (largest weight at 2^14 for fp16, at 1 for bf16 and bf16 parts), of fp32
        top, fine = (2.0 ** 14, 2.0 ** -25) if self.dtype == F16 else (1.0, 2.0 ** -134)
        sub = fine / top * float(wr.abs().max()) + 2.0 ** -150
        eg = wr.abs()[:, None] * (p * (torch.where(z == -float("inf"), 0.0, ez) + elss[:, None] + 2.0 ** -22 * (1 + x)) + U * (g != 0)) + half(self.dtype) * g.abs() + sub
        eg = torch.where(live, eg, 0.0)
        ga = g.abs()
        k = 6 if split else 1
        fin = half(self.dtype)
        low = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}[self.dtype]     # of the result: steps are 2^-24, 2^-133, 2^-149
        self.dh, self.dw, self.db = g @ w, g.t() @ h, g.sum(0)
        self.tol_dh = eg @ w.abs() + (k * V / 16 + 64 + 6) * U * (ga @ w.abs()) + fin * self.dh.abs() + low
        self.tol_dw = eg.t() @ h.abs() + (k * R / 16 + 64 + 6) * U * (ga.t() @ h.abs()) + fin * self.dw.abs() + low
        self.tol_db = eg.sum(0) + (k * R / 16 + 64 + 6) * U * ga.sum(0) + fin * self.db.abs() + low


def near(got, want, tol, what):
    err = (got.double().reshape(want.shape) - want).abs()
    bad = ~(err <= tol * (1 + 1e-3) + 1e-300)
    assert not bool(bad.any()), "%s: %d off, worst %g over a tolerance of %g" % (what, int(bad.sum()), float(err[bad].max()), float(tol[bad].max()))


def make(R, V, D, dtype, bias, pad=0.1, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + R * 7 + V * 3 + D)

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda")

    h, w = normal(R, D).to(dtype), (normal(V, D) * spread / D ** 0.5).to(dtype)
    b = normal(V).to(dtype) if bias else None
    t = torch.randint(0, V, (R,), generator=g, device="cuda")
    if R > 3:
        t[torch.rand(R, generator=g, device="cuda") < pad] = -1
        t[1] = V + 3
    wt = (0.5 + torch.rand(R, generator=g, device="cuda")) / R * (256 if dtype == F16 else 1)
    return h, w, b, t, wt


def check(h, w, b, t, wt):
    from svae_cf_amd import ops
    ref = Ref(h, w, b, t, wt)
    nll, lse = ops.linear_nll(h, w, t, bias=b)
    near(nll, ref.nll, ref.tol_nll, "nll")
    near(lse, ref.lse_out, ref.tol_lse, "lse")
    nll2, lse2, dh, dw, db = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert torch.equal(nll, nll2) and torch.equal(lse, lse2)
    assert dh.dtype == dw.dtype == h.dtype and dh.shape == h.shape and dw.shape == w.shape
    near(dh, ref.dh, ref.tol_dh, "dh")
    near(dw, ref.dw, ref.tol_dw, "dw")
    if b is not None:
        near(db, ref.db, ref.tol_db, "db")
    again = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert all(x is y is None or torch.equal(x, y) for x, y in zip(again, (nll2, lse2, dh, dw, db)))


SIZES = [(1, 1, 1), (1, 1000, 64), (2, 255, 8), (7, 300, 33), (64, 257, 200), (65, 513, 72), (257, 1025, 150), (300, 5000, 256), (513, 3001, 97),
         (40, 700, 1000), (1000, 9000, 130), (2100, 600, 320)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R,V,D", SIZES)
def test_loss_and_gradients(R, V, D, dtype):
    check(*make(R, V, D, dtype, bias=(R + V) % 2 == 1))


FEW = [(5, 70000, 3), (9, 90001, 8), (16, 1000, 300), (17, 40000, 65), (31, 31, 128), (32, 4097, 129), (33, 2000, 96), (50, 20000, 260), (64, 33, 4), (64, 70001, 64), (41, 33000, 260), (64, 140001, 61)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R,V,D", FEW)
def test_few_rows(R, V, D, dtype):
    check(*make(R, V, D, dtype, bias=(R + D) % 2 == 1))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R", [6, 30, 64])
def test_few_rows_strides_masks_and_left_out_rows(R, dtype):
    """Rows of odd length and distance at odd addresses between NaN, as with tensors of their own; left out rows hold anything."""
    from svae_cf_amd import ops
    V, D = 1333, 75
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
    assert bool((got[2][[3, 4, 5]] == 0).all()) and float(got[0][3]) == 0 and float(got[1][4]) == 0
    wide_h[5] = float("nan")                                       # weight 0: no part in the gradient, its loss is its own
    got = ops.linear_nll_grad(wide_h[:, 1:1 + D], wide_w[:, 3:3 + D], t, wt, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(got[2:], want[2:])) and torch.isnan(got[0]).nonzero().tolist() == [[5]]
    every = ops.linear_nll_grad(wide_h[:, 1:1 + D], w, torch.full_like(t, -1), wt, bias=b)
    assert all(float(x.float().abs().max()) == 0 for x in every)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R", [20, 100])
def test_only_one_gradient(R, dtype):
    """Gradients that are asked for alone have the bits that they have together."""
    from svae_cf_amd import ops
    h, w, b, t, _ = make(R, 800, 70, dtype, bias=True)
    full = [x.clone().requires_grad_() for x in (h, w, b)]
    ops.linear_cross_entropy(full[0], full[1], t, full[2], reduction="sum").backward()
    for k in range(3):
        some = [x.clone().requires_grad_(k == j) for j, x in enumerate((h, w, b))]
        ops.linear_cross_entropy(some[0], some[1], t, some[2], reduction="sum").backward()
        assert torch.equal(some[k].grad, full[k].grad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R", [24, 150])
@pytest.mark.parametrize("size", [2.0 ** -110, 1e-20, 2.0 ** 60])
def test_row_weights_of_any_size(size, R, dtype):
    h, w, b, t, wt = make(R, 500, 64, dtype, bias=True)
    wt = wt * size
    wt[::3] *= -1e-3
    check(h, w, b, t, wt)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R", [16, 60, 200])
def test_confident_rows(R, dtype):
    """Targets of a probability near 1, where errors of z and of lse cancel only if both come from the same bits."""
    h, w, b, t, wt = make(R, 2000, 64, dtype, bias=True, pad=0.0)
    t = torch.arange(R, device="cuda") * 7
    w[t] = (h.float() * 0.4).to(dtype)
    check(h, w, b, t, wt)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_than_one_piece_of_the_vocabulary(dtype):
    """G of all columns would take more than a piece of it may."""
    check(*make(4097, 70001 if dtype == BF16 else 25000, 64, dtype, bias=True))


def test_rows_far_apart_and_large_logits():
    """A row's largest logit far behind or in front of the target's, in another tile; logits beyond the range of exp."""
    h, w, b, t, wt = make(130, 1500, 64, BF16, bias=True, spread=60.0)
    check(h, w, b, t, wt)
    w[700] = h[5] * 8
    t[5] = 3
    check(h, w, b, t, wt)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_vocabulary(dtype):
    """-inf in the bias takes entries out: probability and gradient 0; the type's lowest value does the same."""
    from svae_cf_amd import ops
    h, w, b, t, wt = make(90, 900, 48, dtype, bias=True)
    b[200:800] = -float("inf")
    b[810] = torch.finfo(dtype).min
    t = torch.where((t >= 200) & (t <= 810), t % 200, t)
    check(h, w, b, t, wt)
    _, _, _, dw, db = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert bool((dw[200:800] == 0).all()) and bool((db[200:800] == 0).all()) and float(dw[810].float().abs().max()) == 0
    t[0] = 300                                                     # a target that is masked: infinite loss, gradient of the rest
    nll, lse, dh, _, _ = ops.linear_nll_grad(h, w, t, wt, bias=b)
    assert float(nll[0]) == float("inf") and bool(torch.isfinite(lse).all()) and bool(torch.isfinite(dh.float()).all())


def test_left_out_rows_may_hold_anything():
    from svae_cf_amd import ops
    h, w, b, t, wt = make(200, 400, 80, BF16, bias=True)
    t[3], t[50], wt[7] = -1, 400, 0.0
    clean = ops.linear_nll_grad(h, w, t, wt, bias=b)
    h2, wt2 = h.clone(), wt.clone()
    h2[3], h2[50], wt2[3], wt2[50] = float("nan"), float("inf"), float("nan"), float("inf")
    dirty = ops.linear_nll_grad(h2, w, t, wt2, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(clean, dirty))
    assert bool((dirty[2][[3, 7, 50]] == 0).all()) and float(dirty[0][3]) == 0 and float(dirty[1][50]) == 0
    h2[7] = float("nan")                                           # weight 0: no part in the gradient, its loss is its own
    third = ops.linear_nll_grad(h2, w, t, wt2, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(clean[2:], third[2:])) and bool(torch.isnan(third[0][7]))
    every = ops.linear_nll_grad(h2, w, torch.full_like(t, -1), wt2, bias=b)
    assert all(float(x.float().abs().max()) == 0 for x in every)


def test_nan_shows_in_its_own_row():
    from svae_cf_amd import ops
    h, w, _, t, _ = make(70, 600, 64, BF16, bias=False, pad=0.0)
    t[1] = 1
    h[9, 3] = float("nan")
    nll, lse = ops.linear_nll(h, w, t)
    bad = torch.isnan(nll)
    assert bad.tolist() == [r == 9 for r in range(70)] and torch.equal(torch.isnan(lse), bad)


@pytest.mark.parametrize("off,ld", [(0, 80), (8, 80), (1, 81), (0, 72)])
def test_strides(off, ld):
    """Views of wider tensors whose other columns hold NaN; targets of 32 bits, three dimensions."""
    from svae_cf_amd import ops
    D, V, R = 64, 530, 150
    h, w, b, t, wt = make(R, V, D, BF16, bias=True)
    want = ops.linear_nll_grad(h, w, t, wt, bias=b)
    wide_w, wide_h = torch.full((V, ld + off), float("nan"), dtype=BF16, device="cuda"), torch.full((R, ld + off), float("nan"), dtype=BF16, device="cuda")
    wide_w[:, off:off + D], wide_h[:, off:off + D] = w, h
    got = ops.linear_nll_grad(wide_h[:, off:off + D].view(R, D).unflatten(0, (3, 50)), wide_w[:, off:off + D], t.int().view(3, 50), wt.view(3, 50), bias=b)
    assert got[0].shape == (3, 50) and got[2].shape == (3, 50, D)
    assert all(torch.equal(x.reshape(y.shape), y) for x, y in zip(got, want))
    # transposed weight: a copy is made
    got = ops.linear_nll_grad(h, w.t().contiguous().t(), t, wt, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_no_rows():
    from svae_cf_amd import ops
    w, b = torch.randn(5, 16, device="cuda", requires_grad=True), torch.randn(5, device="cuda", requires_grad=True)
    h, t = torch.empty(0, 16, device="cuda", requires_grad=True), torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops.linear_nll(h, w, t)[0].shape == (0,)
    assert bool((ops.linear_nll_grad(h, w, t, torch.empty(0, device="cuda"), bias=b)[3] == 0).all())
    loss = ops.linear_cross_entropy(h, w, t, b)
    loss.backward()
    assert float(loss.detach()) == 0 and h.grad.shape == (0, 16) and bool((w.grad == 0).all()) and bool((b.grad == 0).all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_autograd(reduction, dtype):
    from svae_cf_amd import ops
    h, w, b, t, wt = make(120, 350, 72, dtype, bias=True)
    for x in (h, w, b):
        x.requires_grad_()
    up = 3.0 * wt if reduction == "none" else torch.tensor(2.5, device="cuda")
    out = ops.linear_cross_entropy(h.view(2, 60, 72), w, t.view(2, 60), b, reduction=reduction)
    assert out.dtype == F32 and out.shape == ((2, 60) if reduction == "none" else ())
    out.backward(up.view(out.shape))
    n = int(((t >= 0) & (t < 350)).sum())
    rows = up if reduction == "none" else torch.full((120,), 2.5 / (n if reduction == "mean" else 1), device="cuda")
    ref = Ref(h.detach(), w.detach(), b.detach(), t, rows)
    total = ref.nll if reduction == "none" else ref.nll.sum() / (n if reduction == "mean" else 1)
    tol = ref.tol_nll if reduction == "none" else ref.tol_nll.sum() / (n if reduction == "mean" else 1) + U * total.abs()
    near(out.detach(), total.view(out.shape), tol.view(out.shape), "loss")
    slack = 4 * U                                                  # the row weight is itself the result of two roundings
    for got, want, tol in ((h.grad, ref.dh, ref.tol_dh), (w.grad, ref.dw, ref.tol_dw), (b.grad, ref.db, ref.tol_db)):
        near(got, want, tol + slack * want.abs(), "gradient")


def test_autograd_of_some_inputs_and_of_no_rows_with_targets():
    from svae_cf_amd import ops
    h, w, b, t, _ = make(66, 300, 40, F32, bias=True)
    full = [x.clone().requires_grad_() for x in (h, w, b)]
    ops.linear_cross_entropy(full[0], full[1], t, full[2]).backward()
    for k in range(3):
        some = [x.clone().requires_grad_(k == j) for j, x in enumerate((h, w, b))]
        ops.linear_cross_entropy(some[0], some[1], t, some[2]).backward()
        assert torch.equal(some[k].grad, full[k].grad)
    full[0].grad = None
    loss = ops.linear_cross_entropy(full[0], w, torch.full_like(t, -1), b)
    loss.backward()
    assert float(loss.detach()) == 0 and bool((full[0].grad == 0).all())


def test_gradients_against_differences():
    """Central differences of the formula in 64 bits along random directions; step 1e-4: their own error is of the order of 1e-8."""
    from svae_cf_amd import ops
    h, w, b, t, wt = make(50, 260, 36, F32, bias=True)
    _, _, *got = ops.linear_nll_grad(h, w, t, wt, bias=b)
    ref = Ref(h, w, b, t, wt)

    def loss(h, w, b):
        here = (t >= 0) & (t < 260)
        z = h @ w.t() + b
        return (torch.where(here, wt.double(), 0.0) * (torch.logsumexp(z, 1) - z.gather(1, torch.where(here, t, 0)[:, None])[:, 0])).sum()

    x = [v.double() for v in (h, w, b)]
    for k, tol in enumerate((ref.tol_dh, ref.tol_dw, ref.tol_db)):
        d = torch.randn(x[k].shape, dtype=torch.float64, device="cuda")
        e = 1e-4
        up, dn = list(x), list(x)
        up[k], dn[k] = x[k] + e * d, x[k] - e * d
        diff = float((loss(*up) - loss(*dn)) / (2 * e))
        assert abs(diff - float((got[k].double() * d).sum())) <= float((tol * d.abs()).sum()) + 1e-6


@pytest.mark.parametrize("R", [3, 96])
def test_weight_past_32_bit_offsets(R):
    from svae_cf_amd import ops
    V, D = (1 << 20) + 77, 2304                                    # 4.8 GB of weights
    w = torch.zeros(V, D, dtype=BF16, device="cuda")
    h = torch.ones(R, D, dtype=BF16, device="cuda")
    w[-2:, 0] = torch.tensor([4.0, 8.0], device="cuda").to(BF16)
    t = torch.tensor([V - 1, V - 2, 0], device="cuda").repeat(R // 3)
    want = np.log(V - 2 + np.exp(4.0) + np.exp(8.0))
    nll, lse, dh, dw, _ = ops.linear_nll_grad(h, w, t, torch.ones(R, device="cuda"))
    assert np.allclose(lse.cpu().numpy(), want, rtol=1e-6) and np.allclose(nll.cpu().numpy(), [want - 8, want - 4, want] * (R // 3), rtol=1e-6)
    p = np.exp(np.array([8.0, 4.0]) - want)
    tol = R * 2.0 ** -8 * (1 + 2.0 ** -8)                          # R entries of G of at most 1, each rounded to bf16, and their sum
    assert abs(float(dw[-1, 5]) - (R * p[0] - R // 3)) <= tol and abs(float(dw[-2, -1]) - (R * p[1] - R // 3)) <= tol
    assert abs(float(dh[0, 0]) - (4 * p[1] + 8 * (p[0] - 1))) <= 3 * 2.0 ** -8 * 8 and float(dh[0, 1]) == 0


def test_loss_of_more_tiles_than_a_launch_takes():
    """2^24 rows and 130 tiles of the vocabulary: three launches.  Logits that are the bias alone: every sum is known."""
    from svae_cf_amd import ops
    R, V = 1 << 24, 33100
    b = torch.zeros(V, dtype=BF16, device="cuda")
    b[[5, 16384, V - 1]] = torch.tensor([2.0, 4.0, 6.0], device="cuda").to(BF16)
    t = torch.arange(R, device="cuda", dtype=torch.int32) % V
    nll, lse = ops.linear_nll(torch.randn(R, 8, device="cuda").to(BF16), torch.zeros(V, 8, dtype=BF16, device="cuda"), t, bias=b)
    want = np.log(V - 3 + np.exp(2.0) + np.exp(4.0) + np.exp(6.0))
    tol = (V / 16384 + 200) * U + 2.0 ** -22 + 2 * U * want        # as Ref's, with exact logits
    assert float((lse.double() - want).abs().max()) <= tol
    assert float((nll.double() - (want - b.double()[t.long()])).abs().max()) <= tol + U * want


def test_captured_gradients_two_graphs():
    """Two graphs of different sizes replayed in turn on new inputs, with eager calls between: every replay equals the eager result."""
    from svae_cf_amd import ops
    made, graphs = [], []
    for R, V, D, dt in ((300, 2000, 96, BF16), (90, 700, 50, F16), (12, 3000, 130, F32), (20, 1000, 64, BF16)):
        x = make(R, V, D, dt, bias=True)
        ops.linear_nll_grad(x[0], x[1], x[3], x[4], bias=x[2])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.linear_nll_grad(x[0], x[1], x[3], x[4], bias=x[2])
        made.append((x, out))
        graphs.append(g)
    for k in range(4):
        for (x, out), g in zip(made, graphs):
            new = make(*x[0].shape[:1], *x[1].shape, x[0].dtype, bias=True, seed=100 + k)
            for a, b in zip(x, new):
                a.copy_(b)
            g.replay()
        torch.cuda.synchronize()
        for x, out in made:
            want = ops.linear_nll_grad(x[0], x[1], x[3], x[4], bias=x[2])
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_model_of_both_ends_with_a_shared_table():
    """ids -> embedding -> dropout -> linear cross entropy with the table as output weights: loss and gradient as in 64 bits."""
    from svae_cf_amd import ops
    from test_gpu_ops import philox
    V, D, B, T, p = 500, 40, 6, 30, 0.2
    g = torch.Generator().manual_seed(3)
    table = (torch.randn(V, D, generator=g) * 0.5).cuda().requires_grad_()
    bias = torch.randn(V, generator=g).cuda().requires_grad_()
    ids = torch.randint(0, V, (B, T + 1), generator=g).cuda()
    ids[2, 20:] = -1
    x, t = ids[:, :-1], ids[:, 1:]
    scale = D ** 0.5
    y = ops.dropout(ops.embedding(table, x, scale=scale), p, 5, step=2)
    loss = ops.linear_cross_entropy(y, table, t, bias)
    loss.backward()
    k = int(p * 65536 + 0.5)
    keep = torch.from_numpy(philox(B * T, D, 5, 2) >= k).cuda().view(B, T, D)
    wt, wb = table.detach().double().requires_grad_(), bias.detach().double().requires_grad_()
    e = torch.where((x >= 0)[..., None], wt[x.clamp(min=0)] * scale, 0.0)
    h = torch.where(keep, e * (65536 / (65536 - k)), 0.0)
    ref = torch.nn.functional.cross_entropy((h @ wt.t() + wb).view(-1, V), t.reshape(-1), ignore_index=-1)
    ref.backward()
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-6 * float(ref.detach())
    # fp32 throughout: the two gradients of the table are sums of at most 180 terms each, off by some 1e-6 of their size
    for got, want in ((table.grad, wt.grad), (bias.grad, wb.grad)):
        assert float((got.double() - want).norm() / want.norm()) <= 180 * U
