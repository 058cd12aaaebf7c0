"""The operators at the two ends of a token model -- embedding lookup with its gradient by sorted tokens, dropout from a
counter-based generator, and the softmax cross entropy behind a linear layer over a large vocabulary -- as cases that can
be timed and compared: inputs, the plain form of each operator in torch, and the same call through the package.

Conventions shared with the package: a token or target outside [0, vocabulary) marks a padded place (zero row, no loss,
no gradient); a row of weight 0 takes no part in a gradient; dropout's mask is a function of (seed, step, row key, column)."""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # serving: the newest item of each of 256 users (the repository's batch), fp32 table, bf16 activations; latency counts
        dict(name="embed serve 256", op="embed", train=False, rows=256, vocab=20000, dim=256, table="float32", out="bfloat16", scale=1.0, pad=0.0),
        # one training batch of the ML-20M shape: 256 users, about 21.8k rows
        dict(name="embed train 21800", op="embed", train=True, rows=21800, vocab=20000, dim=256, table="float32", out="float32", scale=1.0, pad=0.0),
        # the large catalogue: few rows, a million of them in the dense gradient
        dict(name="embed train 1M items", op="embed", train=True, rows=11603, vocab=1000000, dim=256, table="float32", out="bfloat16", scale=16.0, pad=0.02),
        # a wide model on long sequences, everything in bf16, a tenth of the places padding
        dict(name="embed train wide", op="embed", train=True, rows=131072, vocab=131072, dim=1024, table="bfloat16", out="bfloat16", scale=32.0, pad=0.1),
        # dropout on one step's rows when serving-sized batches are trained
        dict(name="dropout 256 rows", op="dropout", rows=256, dim=256, dtype="float32", p=0.5, keyed=True, train=True),
        # the embedded items of one ML-20M batch, odd width (the decoder's 150)
        dict(name="dropout 21800 x 150", op="dropout", rows=21800, dim=150, dtype="bfloat16", p=0.1, keyed=True, train=True),
        # activations of a wide model
        dict(name="dropout 65536 x 2048", op="dropout", rows=65536, dim=2048, dtype="bfloat16", p=0.1, keyed=False, train=True),
        # log-probability of one token: the weights are read once and nothing else matters
        dict(name="nll serve 1", op="nll", train=False, rows=1, vocab=131072, dim=1024, dtype="bfloat16", bias=False, pad=0.0),
        # scoring a batch of 256 users against a million items
        dict(name="nll serve 256 x 1M", op="nll", train=False, rows=256, vocab=1000000, dim=256, dtype="float16", bias=True, pad=0.0),
        # the reference's precision at the Netflix shape, decoder width, a ragged batch
        dict(name="nll train fp32", op="nll", train=True, rows=2049, vocab=17770, dim=150, dtype="float32", bias=True, pad=0.05),
        # one ML-20M batch at the recurrent width
        dict(name="nll train 21800", op="nll", train=True, rows=21800, vocab=20000, dim=200, dtype="bfloat16", bias=True, pad=0.05),
        # a large vocabulary behind a wide model
        dict(name="nll train 128k", op="nll", train=True, rows=8192, vocab=131072, dim=1024, dtype="bfloat16", bias=False, pad=0.1),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def padding(rows):  # a handful of rows might else hold nothing but padding
        return pad if rows >= 16 else 0.0

    op = rng.choice(["embed", "dropout", "nll", "nll"])
    dims = [64, 96, 150, 160, 200, 256, 320, 384, 512, 640, 768, 1024]
    dim = rng.choice(dims) if rng.random() < 0.75 else log(33, 1024)
    pad = rng.choice([0.0, 0.0, 0.02, 0.1, 0.5])
    if op == "embed":
        table = rng.choice(list(DTYPES))
        out = rng.choice([table, "float32", "bfloat16"])
        vocab, rows = log(1000, 1000000), log(1, 131072)
        while vocab * dim > 1000000 * 256:
            vocab = log(1000, 1000000)
        while rows * dim > 131072 * 1024:
            rows = log(1, 131072)
        return dict(op=op, train=rng.random() < 0.7, rows=rows, vocab=vocab, dim=dim, table=table, out=out, scale=rng.choice([1.0, 2.0, math.sqrt(dim)]), pad=padding(rows))
    if op == "dropout":
        rows, dim = log(1, 131072), rng.choice([dim, 2048, log(33, 4096)])
        while rows * dim > 65536 * 2048:
            rows = log(1, 131072)
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(list(DTYPES)), p=rng.choice([0.05, 0.1, 0.2, 0.5, 0.9]), keyed=rng.random() < 0.5, train=rng.random() < 0.7)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.7
    most = (1 << 40) if dtype != "float32" else (1 << 37)
    while True:
        rows, vocab = log(1, 32768), log(1000, 1000000)
        if rows * vocab * dim <= most and rows * vocab <= 1 << 30 and vocab * dim <= 1 << 28:
            return dict(op=op, train=train, rows=rows, vocab=vocab, dim=dim, dtype=dtype, bias=rng.random() < 0.5, pad=padding(rows))


def tokens_like(case, g, n):
    """Token ids with a popularity of one over the rank, ranks dealt to ids by a fixed odd step; a share of `pad` is -1."""
    V = case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    t = (rank * 7919 + 13) % V
    t[torch.rand(n, generator=g, device="cuda") < case["pad"]] = -1
    return t.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, dtype, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(DTYPES[dtype])

    s = dict(case=dict(case))
    R, D = case["rows"], case["dim"]
    if case["op"] == "embed":
        s["table"] = normal((case["vocab"], D), case["table"], 0.02 if case["scale"] > 1 else 1.0)
        s["tokens"] = tokens_like(case, g, R)
        if case["train"]:
            s["dout"] = normal((R, D), case["out"], 1e-3)
    elif case["op"] == "dropout":
        s["x"] = normal((R, D), case["dtype"])
        s["seed"], s["step"] = int(seed) * 1000003 + 17, int(seed) % 1000
        s["key"] = torch.randint(0, 1 << 40, (R,), generator=g, device="cuda") if case["keyed"] else None
        if case["train"]:
            s["dy"] = normal((R, D), case["dtype"], 1e-3)
    else:
        V = case["vocab"]
        s["hidden"] = normal((R, D), case["dtype"])
        s["weight"] = normal((V, D), case["dtype"], 2.0 / math.sqrt(D))
        s["bias"] = normal((V,), case["dtype"]) if case["bias"] else None
        s["targets"] = tokens_like(case, g, R)
        if case["train"]:
            # a mean over the rows, some heavier than others; half-precision training scales its loss so that gradients keep their bits
            s["row_weight"] = (0.5 + torch.rand(R, generator=g, device="cuda")) / R * (4096 if case["dtype"] == "float16" else 1)
    return s


def run(s):
    c = s["case"]
    if own:
        from svae_cf_amd import ops
        if c["op"] == "embed":
            y = ops.embedding(s["table"], s["tokens"], scale=c["scale"], out_dtype=DTYPES[c["out"]])
            if not c["train"]:
                return y
            return y, ops.embedding_grad(s["dout"], s["tokens"], c["vocab"], scale=c["scale"], dtype=DTYPES[c["table"]])
        if c["op"] == "dropout":
            y = ops.dropout(s["x"], c["p"], s["seed"], step=s["step"], row_key=s["key"])
            return (y, ops.dropout(s["dy"], c["p"], s["seed"], step=s["step"], row_key=s["key"])) if c["train"] else y
        if not c["train"]:
            return ops.linear_nll(s["hidden"], s["weight"], s["targets"], bias=s["bias"])
        return ops.linear_nll_grad(s["hidden"], s["weight"], s["targets"], s["row_weight"], bias=s["bias"])
    return {"embed": plain_embed, "dropout": plain_dropout, "nll": plain_nll}[c["op"]](s)


def plain_embed(s):
    c = s["case"]
    tok = s["tokens"].long()
    here = (tok >= 0) & (tok < c["vocab"])
    at = torch.where(here, tok, 0)
    y = torch.where(here[:, None], s["table"][at].float() * c["scale"], 0.0).to(DTYPES[c["out"]])
    if not c["train"]:
        return y
    d = torch.where(here[:, None], s["dout"].float(), 0.0)
    grad = torch.zeros((c["vocab"], c["dim"]), device=d.device).index_add_(0, at, d)
    return y, (grad * c["scale"]).to(DTYPES[c["table"]])


def mulhilo(m, x):
    """High and low word of the product of two 32-bit numbers, in 64-bit integers that have a sign."""
    lo, hi = (x & 0xFFFF) * m, (x >> 16) * m           # below 2^48
    mid = hi + (lo >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def plain_keep(rows, dim, p, seed, step, key, device):
    """Which elements stay: Philox4x32-10 with key (seed) and counter (row key, group of 8 columns + 2^31, step); word j of
    a block has the random halves of columns 2 j (low) and 2 j + 1 (high); a column is dropped if its half is below p 2^16."""
    groups = (dim + 7) // 8
    key = torch.arange(rows, device=device) if key is None else key
    c = [(key & 0xFFFFFFFF)[:, None].expand(rows, groups), ((key >> 32) & 0xFFFFFFFF)[:, None].expand(rows, groups),
         (torch.arange(groups, device=device) + (1 << 31))[None, :].expand(rows, groups), torch.full((rows, groups), step & 0xFFFFFFFF, device=device)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = mulhilo(0xD2511F53, c[0])
        h1, l1 = mulhilo(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack(c, 2)
    halves = torch.stack((words & 0xFFFF, words >> 16), 3).reshape(rows, groups * 8)[:, :dim]
    return halves >= drop_below(p)


def drop_below(p):
    return int(math.floor(p * 65536 + 0.5))


def plain_dropout(s):
    c = s["case"]
    keep = plain_keep(c["rows"], c["dim"], c["p"], s["seed"], s["step"], s["key"], s["x"].device)
    up = 65536.0 / (65536 - drop_below(c["p"]))

    def one(x):
        return torch.where(keep, x.float() * up, 0.0).to(x.dtype)

    return (one(s["x"]), one(s["dy"])) if c["train"] else one(s["x"])


def plain_nll(s):
    c = s["case"]
    t = s["targets"].long()
    here = (t >= 0) & (t < c["vocab"])
    at = torch.where(here, t, 0)
    h, w = torch.where(here[:, None], s["hidden"].float(), 0.0), s["weight"].float()
    z = h @ w.T
    if s["bias"] is not None:
        z += s["bias"].float()
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    nll = torch.where(here, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    lse = torch.where(here, lse, 0.0)
    if not c["train"]:
        return nll, lse
    g = torch.exp(z - lse[:, None])
    g[torch.arange(len(t), device=t.device), at] -= 1.0
    weight = torch.where(here, s["row_weight"], 0.0)
    g = torch.where((weight != 0)[:, None], g * weight[:, None], 0.0)
    dh, dw = (g @ w).to(s["hidden"].dtype), (g.T @ h).to(s["weight"].dtype)
    return nll, lse, dh, dw, None if s["bias"] is None else g.sum(0).to(s["bias"].dtype)


def work(case):
    R, D = case["rows"], case["dim"]
    if case["op"] == "embed":
        V, t, o = case["vocab"], SIZE[case["table"]], SIZE[case["out"]]
        fwd = 4 * R + min(R, V) * D * t + R * D * o
        return dict(bytes=fwd + (4 * R + R * D * o + V * D * t if case["train"] else 0), flops=R * D * (2 if case["train"] else 1))
    if case["op"] == "dropout":
        passes = 2 if case["train"] else 1
        return dict(bytes=passes * 2 * R * D * SIZE[case["dtype"]] + (8 * R if case["keyed"] else 0), flops=passes * R * D)
    V, e = case["vocab"], SIZE[case["dtype"]]
    once = (R * D + V * D + (V if case["bias"] else 0)) * e
    return dict(bytes=once * (2 if case["train"] else 1) + 4 * R * 3, flops=(6 if case["train"] else 2) * R * V * D)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        V = case["vocab"]
        tok = s["tokens"].cpu().numpy().astype(np.int64)
        full = torch.cat((s["table"].double() * case["scale"], torch.zeros((1, case["dim"]), device="cuda", dtype=torch.float64)))
        at = torch.from_numpy(np.where((tok < 0) | (tok >= V), V, tok)).cuda()
        y = full.index_select(0, at)
        if not case["train"]:
            return y
        full.zero_()
        full.index_put_((at,), s["dout"].double(), accumulate=True)
        return y, full[:V] * case["scale"]
    if case["op"] == "dropout":
        rows, cols = np.arange(case["rows"], dtype=np.uint64) if s["key"] is None else s["key"].cpu().numpy().astype(np.uint64), case["dim"]
        half, low, bits = np.uint64(32), np.uint64(0xFFFFFFFF), np.uint64(16)
        word = np.arange(-(-cols // 8), dtype=np.uint64)[None, :] | np.uint64(0x80000000)
        a, b = np.broadcast_arrays(rows[:, None] & low, word)
        r, q = np.broadcast_arrays(rows[:, None] >> half, np.full_like(word, s["step"]))
        k = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            x, y = a * np.uint64(0xD2511F53), b * np.uint64(0xCD9E8D57)
            a, r, b, q = (y >> half) ^ r ^ np.uint64(k[0]), y & low, (x >> half) ^ q ^ np.uint64(k[1]), x & low
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        draws = np.empty((case["rows"], word.shape[1], 8), np.uint16)
        for j, v in enumerate((a, r, b, q)):
            draws[:, :, 2 * j], draws[:, :, 2 * j + 1] = v & np.uint64(0xFFFF), v >> bits
        gone = int(case["p"] * 65536 + 0.5)
        factor = torch.from_numpy((draws.reshape(case["rows"], -1)[:, :cols] >= gone).astype(np.uint8)).cuda().double() * (65536 / (65536 - gone))
        y = s["x"].double() * factor
        return (y, s["dy"].double() * factor) if case["train"] else y
    V = case["vocab"]
    t = s["targets"].long()
    left = ((t < 0) | (t >= V)).double()
    w = s["weight"].double()
    x = s["hidden"].double() * (1 - left)[:, None]
    z = torch.addmm(torch.zeros(V, device="cuda", dtype=torch.float64) if s["bias"] is None else s["bias"].double(), x, w.t())
    lse = torch.logsumexp(z, 1)
    there = torch.take_along_dim(z, t.clamp(0, V - 1)[:, None], 1)[:, 0]
    first = [(lse - there) * (1 - left), lse * (1 - left)]
    if not case["train"]:
        return first
    weight = s["row_weight"].double() * (1 - left)
    z.sub_(lse[:, None]).exp_().mul_(weight[:, None])
    z.scatter_add_(1, t.clamp(0, V - 1)[:, None], -weight[:, None])
    return first + [z.mm(w), z.t().mm(x), None if s["bias"] is None else z.sum(0)]
