"""Embedding lookup with its gradient by sorted tokens, and counter-based dropout (svae_cf_amd.ops), against plain forms in
64 bits.  Tolerances count roundings: a sum of n fp32 terms is off by at most n 2^-24 of the sum of magnitudes, a result by
half a step of its type (and, for fp16, half a subnormal step)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == F16 else 0.0


def make_tokens(kind, R, V, g, dtype=torch.int32):
    if kind == "same":
        t = torch.full((R,), V // 2)
    elif kind == "padded":
        t = torch.full((R,), -1)
    else:
        t = (torch.exp(torch.rand(R, generator=g, dtype=torch.float64) * np.log(V + 1)) - 1).long().clamp_(0, V - 1)
        if kind == "padding":
            t[torch.rand(R, generator=g) < 0.3] = -1
            t[torch.rand(R, generator=g) < 0.1] = V + 5
    return t.to(dtype).cuda()


def ref_grad(dy, tok, V, scale, pad=None):
    """(sum, sum of magnitudes, number of terms) of each table row in 64 bits, on the CPU."""
    tok, dy = tok.reshape(-1).long().cpu(), dy.reshape(tok.numel(), -1).double().cpu()
    ok = (tok >= 0) & (tok < V)
    if pad is not None:
        ok &= tok != pad
    tok, dy = tok[ok], dy[ok]
    s = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, tok, dy) * scale
    m = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, tok, dy.abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, tok, torch.ones(len(tok), dtype=torch.float64))
    return s, m, n


def check_grad(got, dy, tok, V, scale, pad=None, old=None):
    s, m, n = ref_grad(dy, tok, V, scale, pad)
    if old is not None:
        s, m = s + old.double().cpu(), m + old.double().cpu().abs()
    tol = (n[:, None] + 3) * U * m * (1 + 1e-6) + half_step(got.dtype) * s.abs() * (1 + 1e-3) + tiny(got.dtype)
    err = (got.double().cpu() - s).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


LOOKUPS = [  # R, V, D, kind, table type, out type
    (1, 5, 1, "zipf", F32, F32), (1, 20000, 256, "zipf", F32, BF16), (7, 3, 33, "padding", BF16, F32), (257, 1000, 150, "padding", F16, F16),
    (300, 2047, 64, "same", F32, F32), (300, 2048, 66, "padded", F16, BF16), (4097, 20000, 200, "zipf", BF16, BF16),
    (5000, 100, 1024, "padding", BF16, BF16), (9001, 70001, 36, "zipf", F32, F16), (64, 64, 2100, "zipf", F16, F32), (1030, 1, 257, "zipf", F32, F32)]


@pytest.mark.parametrize("R,V,D,kind,tt,ot", LOOKUPS)
@pytest.mark.parametrize("tok64", [False, True])
def test_lookup_and_gradient(R, V, D, kind, tt, ot, tok64):
    from svae_cf_amd import ops
    g = torch.Generator().manual_seed(R + V + D)
    tok = make_tokens(kind, R, V, g, torch.int64 if tok64 else torch.int32)
    table, dy = torch.randn(V, D, generator=g).to(tt).cuda(), torch.randn(R, D, generator=g).to(ot).cuda()
    scale = 1.7
    y = ops.embedding(table, tok, scale=scale, out_dtype=ot)
    ok = (tok >= 0) & (tok < V)
    want = torch.where(ok[:, None], table[tok.long().clamp(0, V - 1)].double() * np.float32(scale), 0.0)
    assert y.dtype == ot and y.shape == (R, D)
    assert bool(((y.double() - want).abs() <= (U * 2 + half_step(ot)) * want.abs() * (1 + 1e-3) + tiny(ot)).all())
    assert bool((y[~ok] == 0).all())
    grad = ops.embedding_grad(dy, tok, V, scale=scale, dtype=tt)
    assert grad.dtype == tt
    check_grad(grad, dy, tok, V, float(np.float32(scale)))
    assert torch.equal(grad, ops.embedding_grad(dy, tok, V, scale=scale, dtype=tt))


def test_lookup_no_tokens():
    from svae_cf_amd import ops
    table = torch.randn(11, 12, device="cuda")
    tok = torch.empty(0, 3, dtype=torch.int64, device="cuda")
    assert ops.embedding(table, tok).shape == (0, 3, 12)
    dy = torch.empty(0, 3, 12, device="cuda")
    assert torch.equal(ops.embedding_grad(dy, tok, 11), torch.zeros(11, 12, device="cuda"))
    out = torch.ones(11, 12, device="cuda")
    ops.embedding_grad(dy, tok, 11, out=out, accumulate=True)
    assert bool((out == 1).all())


def test_sort_is_stable_over_every_digit_split():
    """One, two and three digits; keys of one workgroup and of the most there are; the place order inside a token kept."""
    from svae_cf_amd import _lib, ops
    for R, V in ((1, 1), (63, 2), (64, 1023), (4096, 2047), (4097, 2048), (70000, 4194303), (12345, 5000000), (1200001, 300)):
        g = torch.Generator().manual_seed(V)
        tok = torch.randint(-2, V + 2, (R,), generator=g).cuda()
        pad = V // 3
        keys, perm = torch.empty(R, dtype=torch.int32, device="cuda"), torch.empty(R, dtype=torch.int32, device="cuda")
        n = ops._bytes("svae_token_sort_bytes", R, V)
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        _lib.call("svae_token_sort", tok.data_ptr(), 1, R, V, pad, keys.data_ptr(), perm.data_ptr(), work.data_ptr(), n,
                  torch.cuda.current_stream().cuda_stream)
        k = torch.where((tok < 0) | (tok >= V) | (tok == pad), V, tok)
        wk, wp = torch.sort(k, stable=True)
        assert torch.equal(keys.long(), wk) and torch.equal(perm.long(), wp), (R, V)


def test_gradient_long_segments_at_chunk_edges():
    """Segments that start and end at, before and behind multiples of the kernel's chunk, beside short and empty ones."""
    from svae_cf_amd import ops
    lens = [64, 64, 65, 1, 0, 63, 66, 200, 62, 0, 64, 128, 129, 1, 1, 700, 64, 3, 65, 65]
    V, D = len(lens) + 4, 130
    tok = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    g = torch.Generator().manual_seed(5)
    tok = tok[torch.randperm(len(tok), generator=g)].cuda()
    dy = torch.randn(len(tok), D, generator=g).cuda()
    check_grad(ops.embedding_grad(dy, tok, V), dy, tok, V, 1.0)


def test_gradient_padding_idx_accumulate_and_strides():
    from svae_cf_amd import ops
    g = torch.Generator().manual_seed(6)
    V, D, R = 301, 40, 2000
    tok = torch.randint(0, V // 2, (20, 100), generator=g).cuda()
    tok[:, 50:90] = 7
    wide = torch.randn(20, 100, 3 * D, generator=g).cuda()
    dy = wide[..., D:2 * D]
    store = torch.full((V + 2, D + 8), 3.0, device="cuda")
    out = store[1:-1, 4:-4]
    old = torch.randn(V, D, generator=g).cuda()
    out.copy_(old)
    got = ops.embedding_grad(dy, tok, V, scale=0.5, padding_idx=7, out=out, accumulate=True)
    assert got.data_ptr() == out.data_ptr()
    check_grad(out, dy, tok, V, 0.5, pad=7, old=old)
    assert torch.equal(out[V // 2:], old[V // 2:]) and torch.equal(out[7], old[7])
    edge = store.clone()
    edge[1:-1, 4:-4] = 3.0
    assert bool((edge == 3.0).all())
    table = torch.randn(V, 2 * D, generator=g).cuda()[:, 1:D + 1]      # odd start: no vector loads
    y = ops.embedding(table, tok)
    assert torch.equal(y, table[tok])
    assert torch.equal(ops.embedding(table.t().contiguous().t(), tok), y)


def test_lookup_autograd_and_shared_table():
    """A table used twice gets both gradients, also through broadcast (expanded) upstream gradients."""
    from svae_cf_amd import ops
    V, D = 50, 24
    g = torch.Generator().manual_seed(7)
    table = torch.randn(V, D, generator=g).cuda().requires_grad_()
    a, b = torch.randint(-1, V, (4, 9), generator=g).cuda(), torch.randint(0, V, (13,), generator=g).cuda()
    (ops.embedding(table, a, scale=2.0).sum() + 3 * ops.embedding(table, b, padding_idx=1).sum()).backward()
    want = ref_grad(torch.ones(36, D), a, V, 2.0)[0] + ref_grad(torch.full((13, D), 3.0), b, V, 1.0, pad=1)[0]
    assert torch.equal(table.grad.double().cpu(), want)                # small whole numbers: exact


def test_lookup_past_32_bit_offsets():
    from svae_cf_amd import ops
    V, D = (1 << 21) + 3, 1024
    table = torch.zeros(V, D, dtype=BF16, device="cuda")
    table[-3:] = torch.arange(3, device="cuda", dtype=BF16)[:, None] + 1
    tok = torch.tensor([V - 1, 0, V - 3, V - 2, V - 1], device="cuda")
    y = ops.embedding(table, tok)
    assert y[:, 0].tolist() == [3, 0, 1, 2, 3] and y[:, -1].tolist() == [3, 0, 1, 2, 3]
    grad = ops.embedding_grad(y, tok, V)
    assert grad[-3:, 0].tolist() == [1, 2, 6] and grad[-3:, -1].tolist() == [1, 2, 6]
    assert float(grad[:-3].float().abs().max()) == 0


# ---- dropout -------------------------------------------------------------------------------------------------------------
def philox(rows, cols, seed, step, key=None):
    """16-bit draws [rows, cols] by Philox4x32-10 in numpy."""
    key = np.arange(rows, dtype=np.uint64) if key is None else key.cpu().numpy().astype(np.uint64)
    ng, M, S = -(-cols // 8), np.uint64(0xFFFFFFFF), np.uint64(32)
    shape = (rows, ng)
    c = [np.broadcast_to((key & M)[:, None], shape), np.broadcast_to((key >> S)[:, None], shape),
         np.broadcast_to(np.arange(ng, dtype=np.uint64) + np.uint64(1 << 31), shape), np.full(shape, step & 0xFFFFFFFF, np.uint64)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> S) ^ c[1] ^ np.uint64(k0), p1 & M, (p0 >> S) ^ c[3] ^ np.uint64(k1), p0 & M]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    w = np.stack(c, 2)
    return np.stack((w & np.uint64(0xFFFF), w >> np.uint64(16)), 3).reshape(rows, ng * 8)[:, :cols].astype(np.int64)


def want_dropout(x, p, seed, step, key=None):
    k = int(p * 65536 + 0.5)
    keep = torch.from_numpy(philox(x.shape[0], x.shape[1], seed, step, key) >= k).to(x.device)
    up = torch.tensor(65536.0 / (65536 - k) if k < 65536 else 0.0, dtype=F32).to(x.device)
    return torch.where(keep, x.float() * up, torch.zeros((), device=x.device)).to(x.dtype)


@pytest.mark.parametrize("R,C", [(1, 1), (1, 8), (3, 7), (5, 150), (64, 256), (1000, 33), (17, 2052), (300, 12)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_bits(R, C, dtype):
    from svae_cf_amd import ops
    g = torch.Generator().manual_seed(R * C)
    x = torch.randn(R, C, generator=g).to(dtype).cuda()
    for p, seed, step, keyed in ((0.1, 5, 0, False), (0.5, (1 << 63) + 12345678901, 7, True), (1 / 65536, 1, (1 << 32) - 1, True), (0.9999, 3, 2, False)):
        key = torch.randint(0, 1 << 62, (R,), generator=g).cuda() if keyed else None
        got = ops.dropout(x, p, seed, step=step, row_key=key)
        assert torch.equal(got, want_dropout(x, p, seed, step, key)), (p, seed, step)
    assert torch.equal(ops.dropout(x, 0.0, 9), x) and bool((ops.dropout(x, 1.0, 9) == 0).all())


def test_dropout_share_of_zeros_and_mean():
    from svae_cf_amd import ops
    n = 1 << 22
    y = ops.dropout(torch.ones(n // 1024, 1024, device="cuda"), 0.3, 11, step=4).double()
    k = int(0.3 * 65536 + 0.5) / 65536
    assert abs(float((y == 0).double().mean()) - k) < 5 * (k * (1 - k) / n) ** 0.5       # five sigma of the binomial
    assert abs(float(y.mean()) - 1) < 5 * (k / (1 - k) / n) ** 0.5


def test_dropout_nan_and_inf_in_dropped_places():
    from svae_cf_amd import ops
    x = torch.randn(40, 64, device="cuda")
    keep = want_dropout(torch.ones_like(x), 0.5, 21, 3) != 0
    x[~keep] = float("nan")
    x[0, ~keep[0]] = float("inf")
    y = ops.dropout(x, 0.5, 21, step=3)
    assert bool((y[~keep] == 0).all()) and bool((y[keep] == 2 * x[keep]).all())


def test_dropout_strides_in_place_and_sharding():
    from svae_cf_amd import ops
    wide = torch.randn(60, 300, device="cuda")
    x = wide[::2, 30:180]
    want = want_dropout(x.contiguous(), 0.2, 77, 1)
    assert torch.equal(ops.dropout(x, 0.2, 77, step=1), want)
    key = torch.arange(30, device="cuda")
    lo, hi = ops.dropout(x[:13], 0.2, 77, step=1, row_key=key[:13]), ops.dropout(x[13:], 0.2, 77, step=1, row_key=key[13:])
    assert torch.equal(torch.cat((lo, hi)), want)                      # a mask belongs to its row, wherever the row is
    y = x.contiguous()
    assert ops.dropout(y, 0.2, 77, step=1, out=y) is y and torch.equal(y, want)
    deep = torch.randn(4, 5, 6, 16, device="cuda").transpose(0, 2)
    assert torch.equal(ops.dropout(deep, 0.4, 1), want_dropout(deep.reshape(-1, 16), 0.4, 1, 0).view(deep.shape))


def test_dropout_gradient_uses_the_same_mask():
    from svae_cf_amd import ops
    x = torch.randn(33, 50, device="cuda", requires_grad=True)
    step = torch.tensor([6], device="cuda")
    y = ops.dropout(x, 0.25, 5, step=step)
    step += 1                                                          # the program goes on before the backward pass
    dy = torch.randn(33, 50, device="cuda")
    y.backward(dy)
    assert torch.equal(y.detach(), want_dropout(x.detach(), 0.25, 5, 6)) and torch.equal(x.grad, want_dropout(dy, 0.25, 5, 6))


def test_captured_lookup_dropout_and_gradient():
    """One graph, replayed on new tokens and a step that advances on the device, between eager calls of the same operators."""
    from svae_cf_amd import ops
    V, D, R = 3000, 72, 1500
    g = torch.Generator().manual_seed(8)
    table = torch.randn(V, D, generator=g).cuda()
    tok, dy, step = make_tokens("padding", R, V, g), torch.randn(R, D, generator=g).cuda(), torch.zeros(1, dtype=torch.int64, device="cuda")

    def once(step):
        y = ops.dropout(ops.embedding(table, tok, scale=3.0), 0.3, 99, step=step)
        return y, ops.embedding_grad(ops.dropout(dy, 0.3, 99, step=step), tok, V, scale=3.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grad = once(step)
        step += 1
    for k in range(4):
        tok.copy_(make_tokens("padding", R, V, g))
        graph.replay()
        torch.cuda.synchronize()
        wy, wg = once(k)
        assert int(step) == k + 1 and torch.equal(y, wy) and torch.equal(grad, wg)


def test_operators_on_another_stream():
    from svae_cf_amd import ops
    V, D, R = 5000, 64, 20000
    g = torch.Generator().manual_seed(9)
    tok, dy = make_tokens("zipf", R, V, g), torch.randn(R, D, generator=g).cuda()
    want = ops.embedding_grad(dy, tok, V)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.embedding_grad(dy, tok, V) for _ in range(3)]
    both = ops.embedding_grad(dy, tok, V)
    torch.cuda.synchronize()
    assert all(torch.equal(w, want) for w in got + [both])


def test_calls_that_are_refused():
    from svae_cf_amd import ops
    table, tok = torch.randn(10, 8, device="cuda", requires_grad=True), torch.tensor([1, 2], device="cuda")
    with pytest.raises(ValueError, match="padding_idx"):           # (not only in the backward pass)
        ops.embedding(table, tok, padding_idx=10)
    x = torch.randn(40, 16, device="cuda")
    for out in (x.view(-1)[8:8 + 320].view(20, 16), x[10:30]):
        with pytest.raises(ValueError, match="apart"):
            ops.dropout(x[:20], 0.5, 1, out=out)
    with pytest.raises(ValueError, match="apart"):                 # rows of the input behind others of the output
        ops.dropout(x[::2], 0.5, 1, out=x[:20])
    with pytest.raises(ValueError, match="apart"):
        ops.embedding_grad(x[:2], tok, 10, out=x[:10])
    key = torch.arange(5, device="cuda")
    y = ops.dropout(torch.randn(5, 8, device="cuda", requires_grad=True), 0.5, 1, row_key=key)
    key += 1                                                       # the mask of the backward pass would be another
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_more_threads_than_32_bits_count():
    """16 777 221 rows of 257 numbers, 256 threads each; 2^29 tokens, whose chunks of 64 are more than 2^23 workgroups."""
    from svae_cf_amd import ops
    table = torch.randn(50, 257, device="cuda").to(BF16)
    tok = (torch.arange((1 << 24) + 5, device="cuda") % 50).int()
    y = ops.embedding(table, tok)
    for at in (0, (1 << 23) - 3, (1 << 23), (1 << 24) - 2, (1 << 24)):
        assert torch.equal(y[at:at + 5], table[tok[at:at + 5].long()])
    del y
    R, V = (1 << 29) + 77, 1000
    tok = (torch.arange(R, device="cuda") % V).int()
    grad = ops.embedding_grad(torch.ones(R, 1, dtype=BF16, device="cuda"), tok, V, dtype=F32)
    want = R // V + (torch.arange(V, device="cuda") < R % V)       # sums of ones, below 2^24: exact
    assert torch.equal(grad.view(-1).long(), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 3, 7, 9, 13, 141, 515])
def test_odd_widths_between_other_columns(D, dtype):
    """Rows at any address: the bits of aligned copies, NaN beside the inputs is not read, what lies beside the output stays."""
    from svae_cf_amd import ops
    g = torch.Generator(device="cuda").manual_seed(D)
    R, V = 3000, 45
    tok = torch.randint(0, V, (R,), generator=g, device="cuda")
    tok[:700] = 11                                                 # a segment of many chunks
    wide = torch.full((R, D + 5), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:3 + D] = torch.randn(R, D, generator=g, device="cuda").to(dtype)
    dy, flat = wide[:, 3:3 + D], wide[:, 3:3 + D].contiguous()
    want = ops.embedding_grad(flat, tok, V)
    buf = torch.full((V, D + 4), 7.0, dtype=dtype, device="cuda")
    ops.embedding_grad(dy, tok, V, out=buf[:, 1:1 + D])
    assert torch.equal(buf[:, 1:1 + D], want) and bool((buf[:, :1] == 7).all()) and bool((buf[:, 1 + D:] == 7).all())
    one = torch.full((V, D + 4), 1.0, dtype=dtype, device="cuda")
    ops.embedding_grad(dy, tok, V, out=one[:, 1:1 + D], accumulate=True)
    two = torch.full((V, D), 1.0, dtype=dtype, device="cuda")
    ops.embedding_grad(flat, tok, V, out=two, accumulate=True)
    assert torch.equal(one[:, 1:1 + D], two) and bool((one[:, :1] == 1).all()) and bool((one[:, 1 + D:] == 1).all())
    assert torch.equal(ops.embedding(dy[:V], tok), flat[tok])
    y = ops.dropout(dy, 0.3, 9, step=4)
    assert torch.equal(y, ops.dropout(flat, 0.3, 9, step=4)) and not bool(torch.isnan(y).any())
    assert torch.equal(ops.dropout(flat, 0.3, 9, step=4, out=flat), y)
