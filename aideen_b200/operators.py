"""Operators on the caller's CUDA tensors: embedding lookup, layer
normalisation and the cross entropy of a linear head, each with its gradient.

They stand beside `GpuDeqBackend` (which owns the DEQ block's buffers) for the
token side of a model whose tensors the caller holds: torch tensors in float32,
bfloat16 or float16.  Every call goes through `libaideen_b200.so`
(include/aideen_b200.h has the formulas and the rules on ids and targets);
there is no CPU fallback.  Work is queued on torch's current stream of the
tensors' device, outputs and scratch memory come from torch's allocator, and
nothing waits, so every call can be captured into a CUDA graph.  Arguments that
cannot be served raise `AideenError` before anything is launched.  No call looks
for a bounded device-side wait that ran out: `check` does, and waits.

The calls are outside autograd: inputs that require gradients are read like any
others, outputs carry no history, and the backward pass is the caller's chain of
the `_grad` calls (a `torch.autograd.Function` can wrap a pair of them).

A matrix may have any row stride as long as its last dimension is contiguous
and its leading dimensions share one stride; 16-byte aligned rows are fastest.
"""
from __future__ import annotations

import ctypes as C

import torch

from .backend import AideenError, EmbedArgs, LayerNormArgs, LinearCeArgs, load_library

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_REDUCTIONS = {"mean": 0, "sum": 1}
_COUNTS = 1 << 31  # the library's own limits lie below; from here on a count would not fit its field


def _check(rc: int, what: str):
    if rc != 0:
        raise AideenError(f"{what}: status {rc}: {load_library().aideen_operator_error().decode()}")


def _tensor(t, what: str, name: str, like=None, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise AideenError(f"{what}: {name} must be a CUDA tensor")
    if dtype is not None:
        if t.dtype != dtype:
            raise AideenError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    elif t.dtype not in _DTYPES:
        raise AideenError(f"{what}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    if like is not None and t.device != like.device:
        raise AideenError(f"{what}: {name} is on {t.device}, not on {like.device}")
    return t


def _rows(t, what: str, name: str):
    """(rows, dim, row stride) of a matrix with any number of leading dimensions."""
    if t.dim() < 1 or t.shape[-1] < 1:
        raise AideenError(f"{what}: {name} needs a last dimension of at least 1")
    dim = t.shape[-1]
    n = t.numel() // dim
    if n >= _COUNTS or dim >= _COUNTS:
        raise AideenError(f"{what}: {name} has more rows or columns than the library counts")
    if t.is_contiguous():
        return n, dim, dim
    if t.dim() == 1:
        t = t.unsqueeze(0)
    elif t.dim() > 2:
        try:
            t = t.view(-1, dim)
        except RuntimeError:
            raise AideenError(f"{what}: {name}'s leading dimensions have no common row stride") from None
    if dim > 1 and t.stride(1) != 1:
        raise AideenError(f"{what}: {name}'s last dimension is not contiguous")
    ld = t.stride(0) if n > 1 else dim
    if ld < dim:
        raise AideenError(f"{what}: {name}'s rows overlap")
    return n, dim, ld


def _vector(t, what: str, name: str, n: int, like, dtype=None):
    if t is None:
        return None
    _tensor(t, what, name, like, dtype or like.dtype)
    if t.numel() != n or not t.is_contiguous():
        raise AideenError(f"{what}: {name} must be contiguous with {n} elements")
    return t.data_ptr()


def _out(t, what: str, name: str, shape, like):
    """A given output, checked."""
    _tensor(t, what, name, like, like.dtype)
    if tuple(t.shape) != tuple(shape):
        raise AideenError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _apart(what: str, name: str, out, **inputs):
    """Refuses an output that shares bytes with an input.  Column blocks of one buffer
    (rows of the same stride, side by side) share none."""
    def place(t):
        n, dim, ld = _rows(t, what, name) if t.dim() > 0 else (1, 1, 1)
        el = t.element_size()
        return t.data_ptr(), n, dim * el, ld * el
    if out.numel() == 0:
        return
    p, n, width, ld = place(out)
    for other, t in inputs.items():
        if t is None or t.numel() == 0:
            continue
        q, m, w, step = place(t)
        if p + (n - 1) * ld + width <= q or q + (m - 1) * step + w <= p:
            continue
        pitch = ld if n > 1 else step  # of whichever has several rows
        if (n == 1 or m == 1 or ld == step) and (q - p) % pitch >= width and (q - p) % pitch + w <= pitch:
            continue
        raise AideenError(f"{what}: {name} overlaps {other}")


_GRADS = ("x", "weight", "bias")


def _wanted(want, what: str):
    """The names of gradients to form, checked (one name may come alone)."""
    want = (want,) if isinstance(want, str) else tuple(want)
    for name in want:
        if name not in _GRADS:
            raise AideenError(f"{what}: want names 'x', 'weight' and 'bias', not {name!r}")
    return want


def _like(t, dtype=None):
    """A new contiguous tensor of t's shape (the cheapest way to allocate one)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# torch's own short cut to the same handle (2 us less per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


class _Here:
    """Stands for `torch.cuda.device` where the device is current already."""
    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_HERE = _Here()


def _on(device):
    """Context with `device` current: the library works on the current one."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _scratch(nbytes: int, like):
    return like.new_empty(nbytes, dtype=torch.uint8)  # torch's blocks start on 512 bytes; the library asks for 256


def check(device=None):
    """Wait for torch's current stream and raise if a bounded wait of an
    operator ran out on the device since the last check."""
    with torch.cuda.device(device):
        _check(load_library().aideen_operator_check(_raw_stream(torch.cuda.current_device())), "check")


# ---- embedding -------------------------------------------------------------
def _ids(ids, what: str, like, name: str = "ids"):
    _tensor(ids, what, name, like, torch.int32)
    if ids.numel() >= _COUNTS:
        raise AideenError(f"{what}: more {name} than the library counts")
    if not ids.is_contiguous():
        raise AideenError(f"{what}: {name} must be contiguous")
    return ids.data_ptr()


def embed(ids, table, scale: float = 1.0, out=None):
    """`scale * table[ids]` (ids int32, any shape; table [vocab, dim]); an id
    outside [0, vocab) gives a row of zeros.  `out` must not overlap the inputs."""
    what = "embed"
    _tensor(table, what, "table")
    if table.dim() != 2:
        raise AideenError(f"{what}: table must be [vocab, dim]")
    vocab, dim, ld = _rows(table, what, "table")
    ip = _ids(ids, what, table)
    n, old = ids.numel(), dim
    if out is None:
        out = table.new_empty((*ids.shape, dim))
    else:
        _out(out, what, "out", (*ids.shape, dim), table)
        if n:
            old = _rows(out, what, "out")[2]
            _apart(what, "out", out, table=table, ids=ids)
    a = EmbedArgs(_DTYPES[table.dtype], n, dim, vocab, scale, 0, ld, old)
    with _on(table.device):
        rc = load_library().aideen_embed(C.byref(a), ip, table.data_ptr(), out.data_ptr(), _raw_stream(table.device.index))
    if rc:
        _check(rc, what)
    return out


def embed_grad(ids, dout, vocab: int, scale: float = 1.0, into=None):
    """Gradient of `embed` by its table: [vocab, dim], or added to `into` (only
    rows that occur in `ids` are touched then) and `into` returned; `into` must
    not overlap the inputs."""
    what = "embed_grad"
    _tensor(dout, what, "dout")
    ip = _ids(ids, what, dout)
    if dout.dim() != ids.dim() + 1 or dout.shape[:-1] != ids.shape:
        raise AideenError(f"{what}: dout must have ids' shape and one more dimension")
    dim, n = dout.shape[-1], ids.numel()
    rld = _rows(dout, what, "dout")[2] if n else dim
    if not 0 < vocab < _COUNTS:
        raise AideenError(f"{what}: vocab must be in [1, 2^31)")
    if into is None:
        grad, gld = dout.new_empty((vocab, dim)), dim
    else:
        grad = _out(into, what, "into", (vocab, dim), dout)
        gld = _rows(grad, what, "into")[2]
        _apart(what, "into", grad, dout=dout, ids=ids)
    a = EmbedArgs(_DTYPES[dout.dtype], n, dim, vocab, scale, int(into is not None), gld, rld)
    lib, size, r = load_library(), C.c_size_t(), C.byref(a)
    _check(lib.aideen_embed_grad_workspace(r, C.byref(size)), what)
    ws = _scratch(size.value, dout)
    with _on(dout.device):
        rc = lib.aideen_embed_grad(r, ip, dout.data_ptr(), grad.data_ptr(), ws.data_ptr(), size.value,
                                   _raw_stream(dout.device.index))
    if rc:
        _check(rc, what)
    return grad


# ---- layer normalisation ----------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None):
    """(y, mean, rstd): each row of x (its last dimension) normalised; mean and
    rstd are float32 with x's leading shape, for `layer_norm_grad`.  `out` may be
    x itself and must not overlap the inputs otherwise."""
    what = "layer_norm"
    _tensor(x, what, "x")
    n, dim, xld = _rows(x, what, "x")
    wp, bp = _vector(weight, what, "weight", dim, x), _vector(bias, what, "bias", dim, x)
    if out is None:
        y, yld = _like(x), dim
    else:
        y = _out(out, what, "out", x.shape, x)
        yld = _rows(y, what, "out")[2]
        _apart(what, "out", y, x=None if y.data_ptr() == x.data_ptr() and yld == xld else x, weight=weight, bias=bias)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = _like(mean)
    a = LayerNormArgs(_DTYPES[x.dtype], n, dim, eps, xld, yld, 0)
    with _on(x.device):
        rc = load_library().aideen_layer_norm(C.byref(a), x.data_ptr(), wp, bp, y.data_ptr(), mean.data_ptr(),
                                              rstd.data_ptr(), _raw_stream(x.device.index))
    if rc:
        _check(rc, what)
    return y, mean, rstd


def layer_norm_grad(dy, x, weight, mean, rstd, want=("x", "weight", "bias")):
    """(dx, dweight, dbias) from the forward's x, mean and rstd; weight may be
    None (1).  `want` names the gradients to form; the others are None."""
    what = "layer_norm_grad"
    want = _wanted(want, what)
    _tensor(x, what, "x")
    _tensor(dy, what, "dy", x, x.dtype)
    if dy.shape != x.shape:
        raise AideenError(f"{what}: dy and x differ in shape")
    n, dim, xld = _rows(x, what, "x")
    yld = _rows(dy, what, "dy")[2]
    wp = _vector(weight, what, "weight", dim, x)
    mp = _vector(mean, what, "mean", n, x, torch.float32)
    rp = _vector(rstd, what, "rstd", n, x, torch.float32)
    dx = _like(x) if "x" in want else None
    dw = x.new_empty(dim) if "weight" in want else None
    db = x.new_empty(dim) if "bias" in want else None
    a = LayerNormArgs(_DTYPES[x.dtype], n, dim, 0.0, xld, yld, dim)
    lib, size, ws, r = load_library(), C.c_size_t(), None, C.byref(a)
    with _on(x.device):
        if dw is not None or db is not None:
            _check(lib.aideen_layer_norm_grad_workspace(r, C.byref(size)), what)
            ws = _scratch(size.value, x)
        rc = lib.aideen_layer_norm_grad(r, dy.data_ptr(), x.data_ptr(), wp, mp, rp,
                                        None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                                        None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(),
                                        size.value, _raw_stream(x.device.index))
    if rc:
        _check(rc, what)
    return dx, dw, db


# ---- cross entropy of a linear head -----------------------------------------
def _ce_args(what, x, weight, targets, bias, reduction):
    _tensor(x, what, "x")
    _tensor(weight, what, "weight", x, x.dtype)
    if reduction not in _REDUCTIONS:
        raise AideenError(f"{what}: reduction must be 'mean' or 'sum'")
    if x.dim() < 1:
        raise AideenError(f"{what}: x needs a last dimension of at least 1")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise AideenError(f"{what}: weight must be [vocab, {x.shape[-1]}]")
    tp = _ids(targets, what, x, "targets")
    if targets.shape != x.shape[:-1]:
        raise AideenError(f"{what}: targets must have x's leading shape")
    n, dim, xld = _rows(x, what, "x")
    if n == 0:
        xld = dim
    vocab, _, wld = _rows(weight, what, "weight")
    if x.element_size() == 2 and wld % 8 == 0 and weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)  # the library reads it in place and needs 16 bytes
        wld = dim
    bp = _vector(bias, what, "bias", vocab, x)
    return LinearCeArgs(_DTYPES[x.dtype], n, dim, vocab, _REDUCTIONS[reduction], xld, wld, dim, dim), weight, tp, bp


def linear_ce(x, weight, targets, bias=None, reduction: str = "mean"):
    """(loss [1], row_loss, lse) of the cross entropy of `x @ weight.T + bias`
    against int32 targets; the logits are not kept.  Rows whose target lies
    outside [0, vocab) are not counted (row_loss and lse 0).  A bias of -Inf
    takes an entry out, whatever its row of weight holds.

    In float32, past 8 rows, x and weight enter the products with 22 bits of a
    value; what lies below 2^-39 of its own row's largest magnitude is rounded
    off."""
    what = "linear_ce"
    a, weight, tp, bp = _ce_args(what, x, weight, targets, bias, reduction)
    lib, size, r = load_library(), C.c_size_t(), C.byref(a)
    loss = x.new_empty(1, dtype=torch.float32)
    row_loss = _like(targets, torch.float32)
    lse = _like(row_loss)
    with _on(x.device):
        _check(lib.aideen_linear_ce_workspace(r, C.byref(size), None), what)
        ws = _scratch(size.value, x)
        rc = lib.aideen_linear_ce(r, x.data_ptr(), weight.data_ptr(), bp, tp, loss.data_ptr(), row_loss.data_ptr(),
                                  lse.data_ptr(), ws.data_ptr(), size.value, _raw_stream(x.device.index))
    if rc:
        _check(rc, what)
    return loss, row_loss, lse


def linear_ce_grad(x, weight, targets, lse, bias=None, dloss=None, reduction: str = "mean",
                   want=("x", "weight", "bias")):
    """(dx, dweight, dbias) of `dloss * loss` from `linear_ce`'s lse (same bias
    and reduction); dloss is a float32 tensor of one element or None (1).
    `want` names the gradients to form; the others, and dbias without a bias,
    are None.

    In 16 bits, softmax - onehot is rounded to the type before its products with
    weight and x (not before dbias's sum).  In float32, weight and x have one scale
    each there: an entry or a row of x 2^17 times all others takes digits from
    theirs, and what lies below 2^-39 of the largest magnitude is rounded off
    (entries that a bias of -Inf masks do not count)."""
    what = "linear_ce_grad"
    want = _wanted(want, what)
    a, weight, tp, bp = _ce_args(what, x, weight, targets, bias, reduction)
    lp = _vector(lse, what, "lse", a.rows, x, torch.float32)
    gp = _vector(dloss, what, "dloss", 1, x, torch.float32)
    lib, size, r = load_library(), C.c_size_t(), C.byref(a)
    dx = _like(x) if "x" in want else None
    dw = x.new_empty((a.vocab, a.dim)) if "weight" in want else None
    db = x.new_empty(a.vocab) if "bias" in want and bias is not None else None
    with _on(x.device):
        _check(lib.aideen_linear_ce_workspace(r, None, C.byref(size)), what)
        ws = _scratch(size.value, x)
        rc = lib.aideen_linear_ce_grad(r, x.data_ptr(), weight.data_ptr(), bp, tp, lp, gp,
                                       None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                                       None if db is None else db.data_ptr(), ws.data_ptr(), size.value,
                                       _raw_stream(x.device.index))
    if rc:
        _check(rc, what)
    return dx, dw, db
