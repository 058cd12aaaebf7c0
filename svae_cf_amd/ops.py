"""Operators at the two ends of a token model, for any width, vocabulary and element type (fp32, bf16, fp16): embedding
lookup with its gradient by sorted tokens, dropout from a counter-based generator, and the softmax cross entropy behind a
linear layer over a large vocabulary.  Hand-written HIP kernels (csrc/lookup.hip, dropout.hip, xent.hip) behind the C-ABI.

Conventions
  - tensors live on a GPU (there is no CPU fallback); work is enqueued on the current stream of the tensors' device, nothing
    synchronises, workspaces come from torch's allocator, so every call can be captured into a graph;
  - a token or target outside [0, vocabulary) marks a padded place: zero row, no loss, no gradient (the package pads with -1);
  - sums, softmax statistics and losses are fp32; a result is rounded once, to its tensor's type;
  - results are the same in every run (no floating-point atomics).

``embedding``, ``dropout`` and ``linear_cross_entropy`` take part in autograd; ``embedding_grad``, ``linear_nll`` and
``linear_nll_grad`` are the same kernels for programs that run their own backward pass (and for graph capture).
"""
import ctypes

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _On:
    """The device of a tensor as the current one, for the time of a call."""
    __slots__ = ("index", "back")

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _check(t, what, types=_TYPES, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (what, type(t).__name__))
    if t.dtype not in types:
        raise TypeError("%s has type %s: %s are supported" % (what, t.dtype, ", ".join(str(k)[6:] for k in types)))
    if t.device.type != "cuda":
        raise RuntimeError("%s is on %s: the HIP path has no CPU fallback" % (what, t.device))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, the other tensors on %s" % (what, t.device, device))
    return t


_IDS = {torch.int32: 0, torch.int64: 1}


def _rows(t):
    """A 2-D tensor whose rows can be addressed (unit stride inside a row, rows that do not overlap): itself or a copy."""
    if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _ld(t):
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


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
    tok, tab = tokens.reshape(-1).contiguous(), _rows(table)
    out = torch.empty((R, D), dtype=out_dtype, device=table.device)
    if R:
        with _On(table) as st:
            _lib.call("svae_lookup_fwd", tab.data_ptr(), _TYPES[tab.dtype], _ld(tab), tok.data_ptr(), _IDS[tok.dtype], out.data_ptr(),
                      _TYPES[out_dtype], D, R, V, D, scale, st)
    return out.view(tokens.shape + (D,))


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
    _check(tokens, "tokens", _IDS, table.device)
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype %s is not supported" % (out_dtype,))
    if table.dim() != 2:
        raise ValueError("table must be [vocabulary, width], got %s" % (tuple(table.shape),))
    _size(table.shape[0], "vocabulary")
    _size(table.shape[1], "width", 1 << 24)
    _size(tokens.numel() + 1, "tokens + 1", (1 << 30) + 1)
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(table, tokens, float(scale), padding_idx, out_dtype)
    return _lookup(table, tokens, float(scale), out_dtype)


def embedding_grad(dout, tokens, num_rows, scale=1.0, padding_idx=None, dtype=None, out=None, accumulate=False):
    """Gradient of ``embedding`` for the table: ``[num_rows, D]`` in ``dtype`` (default: dout's), every row written.

    Tokens are sorted on the device (stable, so equal tokens are added in their order).  ``out``: the tensor to write (rows may
    be strided); with ``accumulate`` the sums are added to what ``out`` holds, as for a table that another gradient shares."""
    _check(dout, "dout")
    _check(tokens, "tokens", _IDS, dout.device)
    if dout.dim() < 1 or dout.shape[:-1] != tokens.shape:
        raise ValueError("dout %s does not have one row for each token of %s" % (tuple(dout.shape), tuple(tokens.shape)))
    R, D, V = tokens.numel(), dout.shape[-1], int(num_rows)
    _size(V, "vocabulary")
    _size(D, "width", 1 << 24)
    _size(R + 1, "tokens + 1", (1 << 30) + 1)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        dtype = dout.dtype if dtype is None else dtype
        if dtype not in _TYPES:
            raise TypeError("dtype %s is not supported" % (dtype,))
        out = torch.empty((V, D), dtype=dtype, device=dout.device)
    else:
        _check(out, "out", device=dout.device)
        if tuple(out.shape) != (V, D) or (D > 1 and out.stride(1) != 1) or (V > 1 and out.stride(0) < D) or dtype not in (None, out.dtype):
            raise ValueError("out must be [%d, %d] with rows that can be addressed%s" % (V, D, "" if dtype is None else " and type %s" % dtype))
    tok, dy = tokens.reshape(-1).contiguous(), _rows(dout.reshape(R, D))
    pad = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and not 0 <= pad < V:
        raise ValueError("padding_idx %d is outside the table of %d rows" % (pad, V))
    n_sort, n_sum = _bytes("svae_token_sort_bytes", R, V), _bytes("svae_lookup_bwd_bytes", R, D)
    work = torch.empty(max(1, (2 * R + 127) // 128 * 128 * 4 + max(n_sort, n_sum)), dtype=torch.uint8, device=dout.device)
    keys, perm, rest = work.data_ptr(), work.data_ptr() + 4 * R, work.data_ptr() + (2 * R + 127) // 128 * 128 * 4
    with _On(dout) as st:
        _lib.call("svae_token_sort", tok.data_ptr(), _IDS[tok.dtype], R, V, pad, keys, perm, rest, n_sort, st)
        _lib.call("svae_lookup_bwd", dy.data_ptr(), _TYPES[dy.dtype], _ld(dy), keys, perm, R, V, D, scale, out.data_ptr(), _TYPES[out.dtype],
                  _ld(out), int(accumulate), rest, n_sum, st)
    return out


# ---- dropout --------------------------------------------------------------------------------------------------------------
def _dropout(x, p, seed, step, row_key, out=None):
    C = x.shape[-1]
    x2 = _rows(x.reshape(-1, C))
    R = x2.shape[0]
    y = torch.empty((R, C), dtype=x.dtype, device=x.device) if out is None else out.view(R, C)
    if R:
        dev = isinstance(step, torch.Tensor)
        with _On(x) as st:
            _lib.call("svae_dropout", x2.data_ptr(), _ld(x2), y.data_ptr(), _ld(y), _TYPES[x.dtype], R, C, p, seed & 0xFFFFFFFFFFFFFFFF,
                      0 if dev else step & 0xFFFFFFFF, step.data_ptr() if dev else None, None if row_key is None else row_key.data_ptr(), st)
    return y.view(x.shape) if out is None else out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, step, row_key):
        # (a step on the device is copied: the program may advance it before the backward pass makes the mask again)
        step = step.clone() if isinstance(step, torch.Tensor) else step
        ctx.args = (p, seed, step, row_key)
        return _dropout(x, p, seed, step, row_key)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _dropout(dy, *ctx.args), None, None, None, None


def dropout(x, p, seed, step=0, row_key=None, out=None):
    """Dropout of ``x [..., C]`` whose mask is a function of (seed, step, row key, column) and is never stored.

    p: probability of a zero, kept as the nearest multiple of 2^-16 (the scale of what stays uses that one, so the mean is
    kept); 0 and 1 are allowed, other values must not round to them.  seed: 64 bits.  step: int, or an int64 tensor of one
    element on the GPU that the kernel reads, so that a captured graph draws a new mask at every replay.  row_key: int64, one
    for each row (default: the row's index); with keys that travel with the rows a mask does not depend on how rows are dealt
    to GPUs.  The gradient is the same call on dy.  ``out`` (contiguous, may be x) is for calls outside autograd."""
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
        _check(step, "step", {torch.int64: 0}, x.device)
        if step.numel() != 1:
            raise ValueError("step must have one element")
    if row_key is not None:
        _check(row_key, "row_key", {torch.int64: 0}, x.device)
        if row_key.numel() != rows:
            raise ValueError("row_key has %d elements, x has %d rows" % (row_key.numel(), rows))
        row_key = row_key.reshape(-1).contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise ValueError("out is for calls outside autograd")
        return _Dropout.apply(x, p, int(seed), step if isinstance(step, torch.Tensor) else int(step), row_key)
    if out is not None:
        _check(out, "out", {x.dtype: 0}, x.device)
        if out.shape != x.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and shaped like x")
    return _dropout(x, p, int(seed), step if isinstance(step, torch.Tensor) else int(step), row_key, out)
