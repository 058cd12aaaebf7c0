"""Operators at the two ends of a token model, for any width, vocabulary and element type (fp32, bf16, fp16): embedding
lookup with its gradient by sorted tokens, dropout from a counter-based generator, and the softmax cross entropy behind a
linear layer over a large vocabulary.  Hand-written HIP kernels (csrc/lookup.hip, dropout.hip, xent.hip) behind the C-ABI.

Conventions
  - tensors live on a GPU (there is no CPU fallback); work is enqueued on the current stream of the tensors' device, nothing
    synchronises, workspaces come from torch's allocator, so every call can be captured into a graph;
  - a token or target outside [0, vocabulary) marks a padded place: zero row, no loss, no gradient (the package pads with -1);
  - sums, softmax statistics and losses are fp32; a result is rounded once, to its tensor's type (the cross entropy's gradients of
    more than 16 rows of bf16 or fp16 have w (softmax - onehot) in that type too, see ``linear_nll_grad``);
  - results are the same in every run (no floating-point atomics).

``embedding``, ``dropout`` and ``linear_cross_entropy`` take part in autograd (reverse mode, once; tensors with forward-mode
tangents are refused); ``embedding_grad``, ``linear_nll`` and ``linear_nll_grad`` are the same kernels for programs that run their
own backward pass (and for graph capture).
"""
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


_raw_stream = torch._C._cuda_getCurrentRawStream


class _On:
    """The device of a tensor as the current one, for the time of a call; gives that device's current stream."""
    __slots__ = ("index", "back")

    def __init__(self, t):
        self.index = t.get_device()

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _no_tangent(t, what):
    if forward_ad._current_level >= 0 and isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:      # (a kernel would drop it)
        raise NotImplementedError("%s has a tangent: forward-mode differentiation is not supported" % what)


def _check(t, what, types=_TYPES, device=None):
    """Type code of a tensor that has one of `types` and is on the GPU (the one of `device`, a number, if given)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (what, type(t).__name__))
    code = types.get(t.dtype)
    if code is None:
        raise TypeError("%s has type %s: %s are supported" % (what, t.dtype, ", ".join(str(k)[6:] for k in types)))
    _no_tangent(t, what)
    if not t.is_cuda:
        raise RuntimeError("%s is on %s: the HIP path has no CPU fallback" % (what, t.device))
    if device is not None and t.get_device() != device:
        raise ValueError("%s is on %s, the other tensors on cuda:%d" % (what, t.device, device))
    return code


_IDS = {torch.int32: 0, torch.int64: 1}
_INT64 = {torch.int64: 0}
_FLOAT = {torch.float32: 0}


def _rows(t):
    """(t, distance of its rows in elements) for a 2-D tensor, a copy if its rows cannot be addressed (unit stride inside a row,
    rows that do not overlap)."""
    n, c = t.shape
    ld, inner = t.stride()
    if n <= 1:
        ld = c
    if (inner != 1 and c != 1) or ld < c:
        t, ld = t.contiguous(), c
    return t, ld


def _apart(a, b):
    """Whether two tensors share no address."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return not a.numel() or not b.numel() or a1 <= b0 or b1 <= a0


def _written(t):
    """Tells autograd that a caller's tensor has new values: a graph that has kept it refuses its backward pass."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _flat(t):
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


@functools.lru_cache(maxsize=4096)
def _bytes(name, *args):
    n = ctypes.c_longlong()
    _lib.call(name, *args, ctypes.byref(n))
    return n.value


def _size(v, what, most=0x7ffffffe):
    if not 0 < v <= most:
        raise ValueError("%s = %d is outside 1 .. %d" % (what, v, most))


# ---- embedding lookup -----------------------------------------------------------------------------------------------------
def _lookup(table, tokens, scale, out_dtype):
    R, (V, D) = tokens.numel(), table.shape
    tok, (tab, ld) = _flat(tokens), _rows(table)
    out = table.new_empty((R, D), dtype=out_dtype)
    if R:
        with _On(table) as st:
            _lib.call("svae_lookup_fwd", tab.data_ptr(), _TYPES[tab.dtype], ld, tok.data_ptr(), _IDS[tok.dtype], out.data_ptr(),
                      _TYPES[out_dtype], D, R, V, D, scale, st)
    return out if tokens.dim() == 1 else out.view(tokens.shape + (D,))


def _pad(padding_idx, V):
    if padding_idx is None:
        return -1
    if not 0 <= int(padding_idx) < V:
        raise ValueError("padding_idx %d is outside the table of %d rows" % (padding_idx, V))
    return int(padding_idx)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx, out_dtype):
        ctx.save_for_backward(tokens)
        ctx.args = (table.shape[0], scale, padding_idx, table.dtype)
        return _lookup(table, tokens, scale, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        V, scale, padding_idx, dtype = ctx.args
        return embedding_grad(dout, ctx.saved_tensors[0], V, scale, padding_idx, dtype), None, None, None, None


def embedding(table, tokens, scale=1.0, padding_idx=None, out_dtype=None):
    """``scale * table[tokens]`` as ``out_dtype`` (default: the table's), shape ``tokens.shape + (D,)``.

    table [V, D] (rows may be strided), tokens int32 / int64 of any shape.  A token outside [0, V) gives a zero row and no
    gradient; ``padding_idx`` is looked up like any other and gets no gradient.  The gradient is dense, in the table's type."""
    _check(table, "table")
    _check(tokens, "tokens", _IDS, table.get_device())
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype %s is not supported" % (out_dtype,))
    if table.dim() != 2:
        raise ValueError("table must be [vocabulary, width], got %s" % (tuple(table.shape),))
    _size(table.shape[0], "vocabulary")
    _size(table.shape[1], "width", 1 << 24)
    _size(tokens.numel() + 1, "tokens + 1", (1 << 30) + 1)
    _pad(padding_idx, table.shape[0])
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(table, tokens, float(scale), padding_idx, out_dtype)
    return _lookup(table, tokens, float(scale), out_dtype)


def embedding_grad(dout, tokens, num_rows, scale=1.0, padding_idx=None, dtype=None, out=None, accumulate=False):
    """Gradient of ``embedding`` for the table: ``[num_rows, D]`` in ``dtype`` (default: dout's), every row written.

    Tokens are sorted on the device (stable; equal tokens are added in an order that is the same in every run).  ``out``: the tensor to write (rows may
    be strided); with ``accumulate`` the sums are added to what ``out`` holds, as for a table that another gradient shares."""
    _check(dout, "dout")
    _check(tokens, "tokens", _IDS, dout.get_device())
    if dout.dim() < 1 or dout.shape[:-1] != tokens.shape:
        raise ValueError("dout %s does not have one row for each token of %s" % (tuple(dout.shape), tuple(tokens.shape)))
    R, D, V = tokens.numel(), dout.shape[-1], int(num_rows)
    _size(V, "vocabulary")
    _size(D, "width", 1 << 24)
    _size(R + 1, "tokens + 1", (1 << 30) + 1)
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError("accumulate needs out")
        dtype = dout.dtype if dtype is None else dtype
        if dtype not in _TYPES:
            raise TypeError("dtype %s is not supported" % (dtype,))
        out = torch.empty((V, D), dtype=dtype, device=dout.device)
    else:
        _check(out, "out", device=dout.get_device())
        if tuple(out.shape) != (V, D) or (D > 1 and out.stride(1) != 1) or (V > 1 and out.stride(0) < D) or dtype not in (None, out.dtype):
            raise ValueError("out must be [%d, %d] with rows that can be addressed%s" % (V, D, "" if dtype is None else " and type %s" % dtype))
        if not _apart(out, dout):
            raise ValueError("out must lie apart from dout")
    pad = _pad(padding_idx, V)
    tok, (dy, ld) = _flat(tokens), _rows(dout if dout.dim() == 2 else dout.reshape(R, D))
    n_sort, n_sum = _bytes("svae_token_sort_bytes", R, V), _bytes("svae_lookup_bwd_bytes", R, D)
    keep = (2 * R + 127) // 128 * 512                     # keys and places, then what either call needs
    work = torch.empty(keep + max(n_sort, n_sum, 1), dtype=torch.uint8, device=dout.device)
    keys = work.data_ptr()
    perm, rest = keys + 4 * R, keys + keep
    with _On(dout) as st:
        _lib.call("svae_token_sort", tok.data_ptr(), _IDS[tok.dtype], R, V, pad, keys, perm, rest, n_sort, st)
        _lib.call("svae_lookup_bwd", dy.data_ptr(), _TYPES[dy.dtype], ld, keys, perm, R, V, D, scale, out.data_ptr(), _TYPES[out.dtype],
                  out.stride(0) if V > 1 else D, int(accumulate), rest, n_sum, st)
    if given:
        _written(out)
    return out


# ---- dropout --------------------------------------------------------------------------------------------------------------
def _dropout(x, p, seed, step, row_key, out=None):
    C = x.shape[-1]
    x2, ld = _rows(x if x.dim() == 2 else x.reshape(-1, C))
    R = x2.shape[0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if out is None else out
    if R:
        dev = isinstance(step, torch.Tensor)
        with _On(x) as st:
            _lib.call("svae_dropout", x2.data_ptr(), ld, y.data_ptr(), C, _TYPES[x.dtype], R, C, p, seed & 0xFFFFFFFFFFFFFFFF,
                      0 if dev else step & 0xFFFFFFFF, step.data_ptr() if dev else None, None if row_key is None else row_key.data_ptr(), st)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, step, row_key):
        # (a step on the device is copied: the program may advance it before the backward pass makes the mask again)
        step = step.clone() if isinstance(step, torch.Tensor) else step
        ctx.save_for_backward(row_key)
        ctx.args = (p, seed, step)
        return _dropout(x, p, seed, step, row_key)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _dropout(dy, *ctx.args, *ctx.saved_tensors), None, None, None, None


def dropout(x, p, seed, step=0, row_key=None, out=None):
    """Dropout of ``x [..., C]`` whose mask is a function of (seed, step, row key, column) and is never stored.

    p: probability of a zero, kept as the nearest multiple of 2^-16 (the scale of what stays uses that one, so the mean is
    kept); 0 and 1 are allowed, other values must not round to them.  seed: 64 bits.  step: int, or an int64 tensor of one
    element on the GPU that the kernel reads, so that a captured graph draws a new mask at every replay.  row_key: int64, one
    for each row (default: the row's index); with keys that travel with the rows a mask does not depend on how rows are dealt
    to GPUs.  The gradient is the same call on dy.  ``out`` (contiguous; x itself or apart from it) is for calls outside autograd."""
    _check(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have columns, got %s" % (tuple(x.shape),))
    rows = x.numel() // x.shape[-1]
    _size(rows + 1, "rows + 1", 0x7fffffff)
    _size(x.shape[-1], "columns", 1 << 30)
    p = float(p)
    k = int(p * 65536.0 + 0.5) if 0.0 <= p <= 1.0 else -1
    if k < 0 or (k == 0) != (p == 0.0) or (k == 65536) != (p == 1.0):
        raise ValueError("p = %r must be 0, 1 or a probability that is at least 2^-17 from both" % (p,))
    if isinstance(step, torch.Tensor):
        _check(step, "step", _INT64, x.get_device())
        if step.numel() != 1:
            raise ValueError("step must have one element")
    if row_key is not None:
        _check(row_key, "row_key", _INT64, x.get_device())
        if row_key.numel() != rows:
            raise ValueError("row_key has %d elements, x has %d rows" % (row_key.numel(), rows))
        row_key = _flat(row_key)
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise ValueError("out is for calls outside autograd")
        return _Dropout.apply(x, p, int(seed), step if isinstance(step, torch.Tensor) else int(step), row_key)
    if out is not None:
        _check(out, "out", {x.dtype: 0}, x.get_device())
        if out.shape != x.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and shaped like x")
        if not _apart(x, out) and not (x.is_contiguous() and x.data_ptr() == out.data_ptr()):
            raise ValueError("out must be x itself or lie apart from it")
    y = _dropout(x, p, int(seed), step if isinstance(step, torch.Tensor) else int(step), row_key, out)
    if out is not None:
        _written(out)
    return y


# ---- softmax cross entropy behind a linear layer ----------------------------------------------------------------------------
def _xent_args(hidden, weight, targets, bias):
    """Checks; returns (hidden rows, weight rows, bias, flat targets, R, V, D)."""
    _check(hidden, "hidden")
    _check(weight, "weight", {hidden.dtype: 0}, hidden.get_device())
    _check(targets, "targets", _IDS, hidden.get_device())
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("hidden %s and weight %s do not fit: [..., D] and [V, D]" % (tuple(hidden.shape), tuple(weight.shape)))
    if targets.shape != hidden.shape[:-1]:
        raise ValueError("targets %s do not have one entry for each row of hidden %s" % (tuple(targets.shape), tuple(hidden.shape)))
    V, D = weight.shape
    R = targets.numel()
    _size(V, "vocabulary", 1 << 28)
    _size(D, "width", 1 << 16)
    _size(R + 1, "rows + 1", (1 << 24) + 1)
    if bias is not None:
        _check(bias, "bias", {hidden.dtype: 0}, hidden.get_device())
        if tuple(bias.shape) != (V,):
            raise ValueError("bias %s must be [%d]" % (tuple(bias.shape), V))
        bias = _flat(bias)
    h, w = _rows(hidden if hidden.dim() == 2 else hidden.reshape(R, D)), _rows(weight)
    if w[1] > 1 << 20:
        w = (weight.contiguous(), D)
    return h, w, bias, _flat(targets), R, V, D


def _ptr(t):
    return None if t is None else t.data_ptr()


def _xent(name, args, grad, middle, out):
    """One of svae_xent_fwd / _bwd / _fwd_bwd with its workspace; middle: pointers behind D, out: those behind."""
    (h, ldh), (w, ldw), bias, tok, R, V, D = args
    n = _bytes("svae_xent_bytes", w.data_ptr() % 16, ldw, _TYPES[h.dtype], R, V, D, int(grad))
    work = torch.empty(n, dtype=torch.uint8, device=h.device)
    with _On(h) as st:
        _lib.call(name, h.data_ptr(), ldh, w.data_ptr(), ldw, _ptr(bias), tok.data_ptr(), _IDS[tok.dtype], _TYPES[h.dtype], R, V, D,
                  *middle, *out, work.data_ptr(), n, st)


def _xent_fwd(args):
    h, R = args[0][0], args[4]
    nll, lse = torch.empty(R, dtype=torch.float32, device=h.device), torch.empty(R, dtype=torch.float32, device=h.device)
    _xent("svae_xent_fwd", args, False, (nll.data_ptr(), lse.data_ptr()), ())
    return nll, lse


def _xent_grads(args, need):
    h, R, V, D = args[0][0], *args[4:]
    new = dict(dtype=h.dtype, device=h.device)
    dh = torch.empty((R, D), **new) if need[0] else None
    dw = torch.empty((V, D), **new) if need[1] or need[2] else None
    db = torch.empty(V, **new) if need[2] else None
    return (dh, dw, db), (_ptr(dh), D, _ptr(dw), D, _ptr(db))


def linear_nll(hidden, weight, targets, bias=None):
    """(nll, lse) of ``softmax(hidden @ weight.T + bias)`` for the targets, fp32, shaped like targets; no logits are kept.

    Entries of the vocabulary are masked by -inf or any low number in the bias (with -inf for all of them loss and gradients are
    NaN, as the formula is).
    hidden [..., D], weight [V, D], bias [V] of one type; targets int32 / int64.  A row whose target is outside [0, V) is left
    out: both are 0.  For scoring, and for programs that run their own backward pass (``linear_nll_grad``)."""
    args = _xent_args(hidden, weight, targets, bias)
    if args[4] == 0:
        nll = torch.empty(targets.shape, dtype=torch.float32, device=hidden.device)
        return nll, nll.clone()
    nll, lse = _xent_fwd(args)
    return (nll, lse) if targets.dim() == 1 else (nll.view(targets.shape), lse.view(targets.shape))


def linear_nll_grad(hidden, weight, targets, row_weight, bias=None):
    """(nll, lse, dhidden, dweight, dbias): ``linear_nll`` and the gradients of ``sum(row_weight * nll)`` in the inputs' type
    (dbias None without a bias).  row_weight: fp32, shaped like targets; a row of weight 0 takes no part in the gradient.

    For bf16 and fp16, w (softmax - onehot) is rounded to that type in front of its products, but for 16 rows or fewer: off by half a
    step of it, and in fp16 by 2^-39 of the largest weight at least, so that rows 2^20 lighter lose probabilities below 2^-19.
    softmax is exp(logit - lse) with the lse that comes back, in fp32: off by 2^-24 |lse|.  Logits are not kept, but for few rows (up
    to 32, or 64), whose R x V logits lie in the workspace of the call."""
    args = _xent_args(hidden, weight, targets, bias)
    _check(row_weight, "row_weight", _FLOAT, hidden.get_device())
    if row_weight.shape != targets.shape:
        raise ValueError("row_weight %s must be shaped like targets %s" % (tuple(row_weight.shape), tuple(targets.shape)))
    (h, _), R = args[0], args[4]
    nll, lse = torch.empty(R, dtype=torch.float32, device=h.device), torch.empty(R, dtype=torch.float32, device=h.device)
    if R == 0:
        return nll.view(targets.shape), lse.view(targets.shape), torch.empty_like(hidden), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias)
    (dh, dw, db), out = _xent_grads(args, (True, True, bias is not None))
    wr = _flat(row_weight)
    _xent("svae_xent_fwd_bwd", args, True, (wr.data_ptr(), nll.data_ptr(), lse.data_ptr()), out)
    if targets.dim() == 1:
        return nll, lse, dh, dw, db
    return nll.view(targets.shape), lse.view(targets.shape), dh.view(hidden.shape), dw, db


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, reduction):
        args = _xent_args(hidden, weight, targets, bias)
        (h, ldh), (w, ldw), b, tok, R, V, D = args
        ctx.shapes, ctx.reduction = (hidden.shape, ldh, ldw, R, V, D), reduction
        out = torch.zeros(2, dtype=torch.float32, device=h.device)
        if R == 0:
            ctx.save_for_backward(h, w, b, tok, out, out)
            return out.new_empty(targets.shape) if reduction == "none" else out[0].clone()
        nll, lse = _xent_fwd(args)
        if reduction != "none":
            with _On(h) as st:
                _lib.call("svae_xent_reduce", nll.data_ptr(), tok.data_ptr(), _IDS[tok.dtype], R, V, int(reduction == "mean"), out.data_ptr(), st)
        ctx.save_for_backward(h, w, b, tok, lse, out)
        return nll.view(targets.shape) if reduction == "none" else out[0].clone()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        h, w, b, tok, lse, out = ctx.saved_tensors
        shape, ldh, ldw, R, V, D = ctx.shapes
        if R == 0:
            return h.new_empty(shape), torch.zeros_like(w), None if b is None else torch.zeros_like(b), None, None
        weight = dloss.reshape(-1).float().contiguous() if ctx.reduction == "none" else (dloss.float() * out[1]).expand(R).contiguous()
        args = ((h, ldh), (w, ldw), b, tok, R, V, D)
        need = ctx.needs_input_grad[:3]
        (dh, dw, db), outs = _xent_grads(args, need)
        _xent("svae_xent_bwd", args, True, (lse.data_ptr(), weight.data_ptr()), outs)
        return None if dh is None else dh.view(shape), dw if need[1] else None, db, None, None


def linear_cross_entropy(hidden, weight, targets, bias=None, reduction="mean"):
    """Softmax cross entropy of the logits ``hidden @ weight.T + bias``, fp32, without keeping them from forward to backward.

    hidden [..., D], weight [V, D], bias [V] of one type (fp32, bf16, fp16); targets int32 / int64, shaped ``hidden.shape[:-1]``;
    a target outside [0, V) leaves its row out.  reduction: "mean" over the rows with a target (0 if there are none), "sum" or
    "none".  The backward pass makes the logits again, in pieces of the vocabulary (of few rows all of them, in its workspace);
    gradients have the inputs' type, with the roundings that ``linear_nll_grad`` names."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be mean, sum or none, got %r" % (reduction,))
    for t, what in ((hidden, "hidden"), (weight, "weight"), (bias, "bias")):        # (gone inside the function)
        _no_tangent(t, what)
    return _LinearCrossEntropy.apply(hidden, weight, bias, targets, reduction)
