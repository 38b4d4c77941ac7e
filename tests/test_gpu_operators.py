"""Operators on caller-owned tensors against plain float64 formulas, at the sizes
and masks where they can go wrong.

Tolerances are worst-case rounding bounds, element by element, written from the
operation counts: U32 = 2^-24 is half a step of float32, U[t] of the stored
type, TINY[t] half of the smallest number it can hold, and a float32 sum of k
terms is off by at most k U32 sum |terms| (2 k U32 where the tensor cores add,
which may cut instead of round)."""
import ctypes as C
import threading

import pytest
import torch

from aideen_b200 import operators as K
from aideen_b200.backend import AideenError, EmbedArgs, LinearCeArgs, load_library

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
U32 = 2.0 ** -24
U = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def rand(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def close(got, want, bound):
    """|got - want| <= bound everywhere (float64)."""
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def strided(t, pad):
    """The same values with a row stride of `pad` more elements."""
    if pad == 0:
        return t
    big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    big[:, :t.shape[1]] = t
    return big[:, :t.shape[1]]


# ---- embedding -------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim,vocab,pad", [(1, 512, 100, 0), (0, 8, 5, 0), (7, 1, 3, 0), (65, 33, 50, 0),
                                              (300, 1024, 64, 8), (129, 264, 1000, 3)])
def test_embed(dtype, n, dim, vocab, pad):
    g = gen(n + dim)
    table = strided(rand(g, vocab, dim, dtype=dtype), pad)
    ids = torch.randint(-2, vocab + 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    out = strided(torch.zeros(n, dim, dtype=dtype, device="cuda"), pad)
    got = K.embed(ids, table, scale=2.3, out=out)
    assert got is out
    inside = (ids >= 0) & (ids < vocab)
    scale = float(torch.tensor(2.3, dtype=F32))
    want = torch.where(inside[:, None], table.double()[ids.clamp(0, vocab - 1).long()] * scale, 0.0)
    close(got, want, (U[dtype] + U32) * (1 + U[dtype]) * want.abs() + TINY[dtype])


def embed_grad_reference(ids, dout, vocab, scale):
    """(sum, sum of magnitudes, counts) per id in float64."""
    keep = ((ids >= 0) & (ids < vocab)).nonzero()[:, 0]
    at, rows = ids[keep].long(), dout.double()[keep] * scale
    zero = torch.zeros(vocab, dout.shape[1], dtype=torch.float64, device="cuda")
    count = torch.zeros(vocab, dtype=torch.float64, device="cuda")
    count.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return zero.clone().index_add_(0, at, rows), zero.clone().index_add_(0, at, rows.abs()), count


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim,vocab,kind", [
    (1, 512, 300, "any"), (0, 16, 5, "any"), (9, 1, 1, "any"), (257, 40, 7, "any"), (1000, 33, 70000, "any"),
    (4096, 64, 50257, "zipf"), (16384, 8, 3, "one"), (16385, 24, 257, "zipf"), (40001, 16, 65536, "zipf"),
    (513, 32, 256, "outside"), (32 * 8 * 32 + 5, 8, 255, "runs")])
@pytest.mark.parametrize("into", [False, True])
def test_embed_grad(dtype, n, dim, vocab, kind, into):
    g = gen(n + dim + vocab)
    if kind == "any":
        ids = torch.randint(-1, vocab + 1, (n,), generator=g, device="cuda")
    elif kind == "zipf":
        ids = ((vocab + 1.0) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).long() - 1
    elif kind == "one":
        ids = torch.full((n,), 1, device="cuda")
    elif kind == "outside":  # nothing is inside
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -1, vocab)
    else:  # runs that end exactly on tile borders
        ids = torch.arange(n, device="cuda") // 64 % vocab
    ids = ids.int()
    dout = rand(g, n, dim, dtype=dtype)
    outside = (ids < 0) | (ids >= vocab)
    dout[outside] = float("nan")  # reaches no result
    scale = 0.5
    old = rand(g, vocab, dim, dtype=dtype)
    old[vocab // 2] = float("inf")
    grad = old.clone() if into else None
    got = K.embed_grad(ids, dout, vocab, scale=scale, into=grad)
    want, mag, count = embed_grad_reference(ids, dout, vocab, scale)
    if into:
        assert got is grad
        untouched = count == 0
        assert torch.equal(got[untouched], old[untouched])
        want = torch.where(untouched[:, None], 0.0, want + old.double())
        got = torch.where(untouched[:, None], torch.zeros_like(got), got)
        live = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), live)
        want, got = torch.where(live, want, 0.0), torch.where(live, got, torch.zeros_like(got))
    sums = (count[:, None] + 2) * U32 * mag + 2 * U32 * want.abs()
    close(got, want, sums + U[dtype] * (want.abs() + sums) + TINY[dtype])
    if not into:
        assert torch.equal(got, K.embed_grad(ids, dout, vocab, scale=scale))  # the same bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim,vocab,pad", [(1, 1, 450, 0), (5, 3, 5851, 0), (2, 7, 33, 0), (40, 5, 20011, 0), (3, 1, 7, 2),
                                             (0, 3, 100, 0), (0, 6, 9, 2), (2, 12, 4097, 0), (1, 4, 1, 0), (6, 2, 900, 6)])
def test_embed_grad_writes_every_row(dtype, n, dim, vocab, pad):
    """Whatever the memory held, also where a row is shorter than 16 bytes."""
    g = gen(n + dim + vocab)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    dout = rand(g, n, dim, dtype=dtype)
    old = torch.full((vocab, dim + pad), 7.0, dtype=dtype, device="cuda")
    a, size = EmbedArgs(TYPES.index(dtype), n, dim, vocab, 1.0, 0, dim + pad, dim), C.c_size_t()
    lib = load_library()
    assert lib.aideen_embed_grad_workspace(C.byref(a), C.byref(size)) == 0
    ws = torch.empty(size.value + 256, dtype=torch.uint8, device="cuda")
    assert lib.aideen_embed_grad(C.byref(a), ids.data_ptr(), dout.data_ptr(), old.data_ptr(), ws.data_ptr(), size.value,
                                 torch.cuda.current_stream().cuda_stream) == 0
    want, mag, count = embed_grad_reference(ids, dout, vocab, 1.0)
    sums = (count[:, None] + 2) * U32 * mag
    close(old[:, :dim], want, sums + U[dtype] * (want.abs() + sums) + TINY[dtype])
    assert bool((old[:, dim:] == 7).all())


def test_embed_grad_strides_and_shapes():
    g = gen(5)
    ids = torch.randint(0, 40, (3, 50), generator=g, device="cuda", dtype=torch.int32)
    wide = rand(g, 3, 50, 48, dtype=BF16)
    dout = wide[:, :, :40]  # one row stride over both leading dimensions
    big = torch.full((40, 56), 7.0, dtype=BF16, device="cuda")
    K.embed_grad(ids, dout, 40, into=big[:, :40].zero_())
    want, mag, count = embed_grad_reference(ids.reshape(-1), dout.reshape(-1, 40), 40, 1.0)
    sums = (count[:, None] + 2) * U32 * mag
    close(big[:, :40], want, sums + U[BF16] * (want.abs() + sums) + TINY[BF16])
    assert bool((big[:, 40:] == 7).all())  # behind the rows nothing is written


# ---- layer normalisation ----------------------------------------------------
def norm_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    var = (xc * xc).mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    y = xc * rstd
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return x, mean, xc, var, rstd, y


# longest chain of additions in a row's sum: per lane, over the lanes and warps,
# and the strided sums of the longest rows
def chain(dim):
    return 64 + dim // 1024


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,pad", [(1, 512, 0), (0, 8, 0), (3, 1, 0), (33, 100, 0), (5, 128, 0), (70, 1000, 0),
                                           (9, 1024, 8), (17, 513, 3), (4, 4096, 0), (3, 8192, 0), (2, 8200, 0),
                                           (2, 20011, 0), (1025, 64, 0)])
@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm(dtype, rows, dim, pad, affine):
    g = gen(rows + dim)
    x = strided(rand(g, rows, dim, dtype=dtype, std=1.7, mean=3.0), pad)
    w = rand(g, dim, dtype=dtype, std=0.1, mean=1.0) if affine else None
    b = rand(g, dim, dtype=dtype, std=0.1) if affine else None
    eps = 1e-5
    y, mean, rstd = K.layer_norm(x, w, b, eps=eps)
    xd, m, xc, var, r, want = norm_reference(x, w, b, eps)
    c = chain(dim)
    dm = c * U32 * xd.abs().mean(1, keepdim=True) + U32 * m.abs() + 1e-30
    close(mean[:, None], m, dm)
    # the variance is taken about the computed mean: off by dm^2, and by the rounding of the differences
    dvar = (c + 4) * U32 * var + dm * dm + 2 * U32 * xc.abs().mean(1, keepdim=True) * (xd.abs().amax(1, keepdim=True) if rows else 0)
    rel_r = 0.5 * dvar / (var + eps) + 4 * U32
    close(rstd[:, None], r, r * rel_r * (1 + rel_r))
    wd = w.double().abs() if affine else 1.0
    dy = wd * (r * (dm + 2 * U32 * xc.abs()) + (xc * r).abs() * (rel_r + 2 * U32)) * 1.01 + 2 * U32 * want.abs()
    close(y, want, dy + U[dtype] * (want.abs() + dy) + TINY[dtype])


# many rows: several for every resident group of warps, at 16-byte and other strides,
# against the same rows alone
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,pad", [(8001, 512, 0), (7999, 40, 8), (9000, 1000, 0), (3001, 2056, 0),
                                           (8000, 24, 1), (2500, 4096, 0), (1001, 8192, 8)])
def test_layer_norm_many_rows(dtype, rows, dim, pad):
    g = gen(rows + dim + 2)
    x = strided(rand(g, rows, dim, dtype=dtype, std=1.7, mean=0.3), pad)
    dy = strided(rand(g, rows, dim, dtype=dtype), pad)
    w, b = rand(g, dim, dtype=dtype, std=0.1, mean=1.0), rand(g, dim, dtype=dtype, std=0.1)
    whole = K.layer_norm(x, w, b)
    grads = K.layer_norm_grad(dy, x, w, whole[1], whole[2])
    K.check(x.device)
    # every row alone is what it is among the others, up to the order of its sums
    some = torch.randint(0, rows, (64,), generator=g, device="cuda").sort().values
    some[0], some[-1] = 0, rows - 1
    few = K.layer_norm(x[some], w, b)
    fewg = K.layer_norm_grad(dy[some], x[some], w, whole[1][some], whole[2][some])
    c = chain(dim)
    xd, m, xc, var, r, want = norm_reference(x[some], w, b, 1e-5)
    for y, mean, rstd in ((whole[0][some], whole[1][some], whole[2][some]), few):
        dm = c * U32 * xd.abs().mean(1, keepdim=True) + U32 * m.abs()
        close(mean[:, None], m, dm)
        dvar = (c + 4) * U32 * var + dm * dm + 2 * U32 * xc.abs().mean(1, keepdim=True) * xd.abs().amax(1, keepdim=True)
        rel_r = 0.5 * dvar / (var + 1e-5) + 4 * U32
        close(rstd[:, None], r, r * rel_r * (1 + rel_r))
        e = w.double().abs() * (r * (dm + 2 * U32 * xc.abs()) + (xc * r).abs() * (rel_r + 2 * U32)) * 1.01 + 2 * U32 * want.abs()
        close(y, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    md, rd = whole[1].double()[:, None], whole[2].double()[:, None]
    xh = (x.double() - md) * rd
    gd = dy.double() * w.double()
    c1, c2 = gd.mean(1, keepdim=True), (gd * xh).mean(1, keepdim=True)
    want = rd * (gd - c1 - xh * c2)
    e1, e2 = (c + 4) * U32 * gd.abs().mean(1, keepdim=True), (c + 8) * U32 * (gd * xh).abs().mean(1, keepdim=True)
    e = rd * (e1 + xh.abs() * e2 + 6 * U32 * (gd.abs() + c1.abs() + (xh * c2).abs())) * 1.01
    bound = e + U[dtype] * (want.abs() + e) + TINY[dtype]
    close(grads[0], want, bound)
    close(fewg[0], want[some], bound[some])
    for got, terms in ((grads[1], dy.double() * xh), (grads[2], dy.double())):
        t = terms.sum(0)
        e = (rows + 16) * U32 * terms.abs().sum(0)
        close(got, t, e + U[dtype] * (t.abs() + e) + TINY[dtype])
    assert all(torch.equal(p, q) for p, q in zip(grads, K.layer_norm_grad(dy, x, w, whole[1], whole[2])))
    only = K.layer_norm_grad(dy, x, None, whole[1], whole[2], want=("weight", "bias"))
    assert only[0] is None and torch.equal(only[1], grads[1]) and torch.equal(only[2], grads[2])
    plain = K.layer_norm(x, None, None)[0]
    ones = K.layer_norm(x, torch.ones_like(w), torch.zeros_like(b))[0]
    assert torch.equal(plain, ones)


def test_layer_norm_constant_and_extreme_rows():
    # a constant row: variance 0, y is the bias; rows with Inf or NaN spoil only themselves
    x = torch.full((4, 96), 3.0, device="cuda")
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    b = torch.linspace(-1, 1, 96, device="cuda")
    y, mean, rstd = K.layer_norm(x, None, b)
    assert torch.equal(y[0], b) and torch.equal(y[3], b)
    assert float(mean[0]) == 3.0 and abs(float(rstd[0]) - 1e-5 ** -0.5) < 1e-4 * 1e-5 ** -0.5
    assert bool(torch.isnan(y[1:3]).all())
    # large values: squares stay in range as long as the variance does
    big = torch.tensor([[1e18, -1e18, 2e18, 0.0]], device="cuda")
    y, _, _ = K.layer_norm(big, eps=0.0)
    want = norm_reference(big, None, None, 0.0)[5]
    close(y, want, 40 * U32 * (want.abs() + 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,pad", [(1, 512, 0), (0, 8, 0), (3, 1, 0), (2, 33, 0), (257, 100, 0), (2048, 512, 0),
                                           (70, 1000, 8), (601, 1024, 0), (17, 513, 3), (40, 2048, 0), (9, 4096, 0),
                                           (5, 8192, 0), (70, 9001, 0)])
@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_grad(dtype, rows, dim, pad, affine):
    g = gen(rows + dim + 1)
    x = strided(rand(g, rows, dim, dtype=dtype, std=1.7, mean=0.3), pad)
    dy = strided(rand(g, rows, dim, dtype=dtype), pad)
    w = rand(g, dim, dtype=dtype, std=0.1, mean=1.0) if affine else None
    _, m, _, _, r, _ = norm_reference(x, None, None, 1e-5)
    mean, rstd = m[:, 0].float(), r[:, 0].float()
    dx, dw, db = K.layer_norm_grad(dy, x, w, mean, rstd)
    md, rd = mean.double()[:, None], rstd.double()[:, None]
    xh = (x.double() - md) * rd
    gd = dy.double() * (w.double() if affine else 1.0)
    c1, c2 = gd.mean(1, keepdim=True), (gd * xh).mean(1, keepdim=True)
    want = rd * (gd - c1 - xh * c2)
    c = chain(dim) + 4
    e1, e2 = c * U32 * gd.abs().mean(1, keepdim=True), (c + 4) * U32 * (gd * xh).abs().mean(1, keepdim=True)
    e = rd * (e1 + xh.abs() * e2 + 6 * U32 * (gd.abs() + c1.abs() + (xh * c2).abs())) * 1.01
    close(dx, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    for got, terms in ((dw, dy.double() * xh), (db, dy.double())):
        s = terms.sum(0)
        e = (rows + 16) * U32 * terms.abs().sum(0)
        close(got, s, e + U[dtype] * (s.abs() + e) + TINY[dtype])
    again = K.layer_norm_grad(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    # the parts alone are the same as together
    assert torch.equal(K.layer_norm_grad(dy, x, w, mean, rstd, want=("x",))[0], dx)
    only = K.layer_norm_grad(dy, x, w, mean, rstd, want=("bias",))
    assert only[0] is None and only[1] is None and torch.equal(only[2], db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,pad", [(37, 9, 0), (37, 121, 0), (2400, 121, 0), (37, 257, 3), (37, 777, 0), (37, 1001, 1),
                                           (600, 513, 0), (9, 2047, 0), (5, 5003, 0), (1, 3, 0), (2, 1, 0)])
def test_layer_norm_rows_at_any_address(dtype, rows, dim, pad):
    """Rows that start between 16-byte boundaries: the same bits wherever they start, and
    nothing outside them is written."""
    g = gen(rows * dim)
    v = 128 // torch.finfo(dtype).bits
    x, dy = rand(g, rows, dim, dtype=dtype, std=1.7), rand(g, rows, dim, dtype=dtype)
    w, b = rand(g, dim, dtype=dtype), rand(g, dim, dtype=dtype)
    ld = dim + pad

    def place(t, offset):
        big = torch.full((rows * ld + 2 * v,), 7.0, dtype=dtype, device="cuda")
        view = big[offset:offset + rows * ld].view(rows, ld)[:, :dim]
        if t is not None:
            view.copy_(t)
        return big, view

    first = None
    for offset in range(1, v):
        xv, dv = place(x, offset)[1], place(dy, (offset * 3) % v)[1]
        big, y = place(None, (offset * 5) % v)
        wv = torch.cat([w[:1]] * (offset % 3) + [w])[offset % 3:]
        _, mean, rstd = K.layer_norm(xv, wv, b, out=y)
        got = (y.clone(), mean, rstd, *K.layer_norm_grad(dv, xv, wv, mean, rstd))
        if first is None:
            first = got
        assert all(torch.equal(p, q) for p, q in zip(first, got))
        y.fill_(7.0)
        assert bool((big == 7.0).all())
    test_layer_norm(dtype, rows, dim, pad, True)
    test_layer_norm_grad(dtype, rows, dim, pad, True)


# ---- cross entropy of a linear head -----------------------------------------
def ce_reference(x, w, b, tg, reduction, dloss, dtype):
    """Results in float64 and their bounds."""
    n, d = x.shape
    v = w.shape[0]
    wd = w.double()
    keep = ((tg >= 0) & (tg < v)).nonzero()[:, 0]
    xd, t = x.double()[keep], tg[keep].long()
    z = xd @ wd.t()
    # d products and additions, the bias, the shift of the exponent
    ez = 2 * (d + 16) * U32 * (xd.abs() @ wd.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + 2 * U32 * b.double().abs()
    ez = ez + 4 * U32 * torch.where(torch.isfinite(z), z.abs(), 0.0)
    lse = torch.logsumexp(z, 1)
    # sums of exponentials: each 8 units off, a few hundred additions at most in a chain
    elz = ez.masked_fill(~torch.isfinite(z), 0.0).amax(1) + 600 * U32 + 4 * U32 * lse.abs()
    rows = lse - z.gather(1, t[:, None])[:, 0]
    erows = elz + ez.gather(1, t[:, None])[:, 0] + 4 * U32 * (lse.abs() + rows.abs())
    count = max(1, keep.numel()) if reduction == "mean" else 1
    c = dloss / count
    p = (z - lse[:, None]).exp()
    G = p.clone()
    G[torch.arange(keep.numel(), device="cuda"), t] -= 1
    eG = p * torch.expm1((ez + elz[:, None] + 8 * U32).clamp(max=10)) + 2 * U32
    if dtype != F32:
        eG = eG + U[dtype] * (G.abs() + eG) + (2.0 ** -36 if dtype == F16 else 0.0)
    full = lambda rows_, width: torch.zeros(n, *width, dtype=torch.float64, device="cuda").index_copy_(0, keep, rows_)  # noqa: E731
    dx = c * (G @ wd)
    edx = abs(c) * (eG @ wd.abs() + 2 * (v + 16) * U32 * (G.abs() @ wd.abs())) + 4 * U32 * dx.abs()
    dw = c * (G.t() @ xd)
    k = keep.numel()
    edw = abs(c) * (eG.t() @ xd.abs() + 2 * (k + 16) * U32 * (G.abs().t() @ xd.abs())) + 4 * U32 * dw.abs()
    db = c * G.sum(0)
    edb = abs(c) * (eG.sum(0) + 2 * (k + 16) * U32 * G.abs().sum(0)) + 4 * U32 * db.abs()
    loss = rows.sum() / count
    eloss = erows.sum() / count + (n + 8) * U32 * rows.abs().sum() / count
    return dict(loss=(loss.reshape(1), eloss.reshape(1)), rows=(full(rows, ()), full(erows, ())),
                lse=(full(lse, ()), full(elz, ())), dx=(full(dx, (d,)), full(edx, (d,))), dw=(dw, edw), db=(db, edb))


def ce_check(x, w, b, tg, reduction="mean", dloss=1.0):
    dtype = x.dtype
    loss, rows, lse = K.linear_ce(x, w, tg, bias=b, reduction=reduction)
    dl = None if dloss == 1.0 else torch.full((1,), dloss, device="cuda")
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse, bias=b, dloss=dl, reduction=reduction)
    K.check(x.device)
    ref = ce_reference(x, w, b, tg, reduction, dloss, dtype)
    for got, name in ((loss, "loss"), (rows, "rows"), (lse, "lse")):
        close(got, ref[name][0], ref[name][1] + 1e-30)
    for got, name in ((dx, "dx"), (dw, "dw")) + (((db, "db"),) if b is not None else ()):
        want, e = ref[name]
        close(got, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    assert (db is None) == (b is None)
    return loss, rows, lse, dx, dw, db


def ce_inputs(seed, rows, dim, vocab, dtype, bias, ignored=0.0, pad=0, spread=3.0):
    g = gen(seed)
    x = strided(rand(g, rows, dim, dtype=dtype), pad)
    w = strided(rand(g, vocab, dim, dtype=dtype, std=spread / dim ** 0.5), pad)
    b = rand(g, vocab, dtype=dtype, std=0.5) if bias else None
    tg = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if ignored:
        tg[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    return x, w, b, tg


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab,bias,ignored,pad", [
    (1, 512, 1000, True, 0.0, 0), (1, 1, 1, False, 0.0, 0), (2, 7, 2, True, 0.0, 0), (5, 16, 65, True, 0.3, 0),
    (127, 64, 255, False, 0.0, 0), (128, 128, 256, True, 0.0, 0), (129, 65, 257, True, 0.5, 0),
    (300, 250, 1030, True, 0.1, 3), (257, 96, 4999, False, 0.2, 8), (640, 512, 777, True, 0.0, 0),
    (3, 1024, 9001, True, 0.0, 0), (1025, 40, 513, True, 0.9, 0)])
def test_linear_ce(dtype, rows, dim, vocab, bias, ignored, pad):
    x, w, b, tg = ce_inputs(rows + dim, rows, dim, vocab, dtype, bias, ignored, pad)
    dloss = 512.0 if dtype == F16 else 1.0
    first = ce_check(x, w, b, tg, dloss=dloss)
    again = ce_check(x, w, b, tg, dloss=dloss)
    for p, q in zip(first, again):
        assert p is q is None or torch.equal(p, q)  # the same bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("dim,vocab,pad", [(512, 50257, 0), (1, 3, 0), (77, 1001, 3), (2056, 130, 0), (4104, 33, 0)])
def test_linear_ce_few_rows(dtype, rows, dim, vocab, pad):
    x, w, b, tg = ce_inputs(rows * dim, rows, dim, vocab, dtype, True, 0.0, pad)
    if rows > 2:
        tg[1], tg[rows - 1] = -1, vocab
        x[1] = float("nan")
    loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
    ref = ce_reference(x, w, b, tg, "mean", 1.0, dtype)
    for got, name in ((loss, "loss"), (row_loss, "rows"), (lse, "lse")):
        close(got, ref[name][0], ref[name][1] + 1e-30)
    total, _, _ = K.linear_ce(x, w, tg, bias=b, reduction="sum")
    kept = int(((tg >= 0) & (tg < vocab)).sum())
    assert abs(float(total) - float(loss) * kept) <= 4 * U32 * float(total)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_at_the_training_vocabulary(dtype):
    x, w, b, tg = ce_inputs(3, 200, 512, 50257, dtype, True, 0.1)
    ce_check(x, w, b, tg, reduction="sum", dloss=0.25 if dtype != F16 else 8.0)


@pytest.mark.parametrize("dtype,rows,dim,vocab,ignored", [
    (F32, 2048, 512, 50257, 0.0),    # 3 pieces of 68, 68 and 61 tiles of 256 entries (on 148 SMs)
    (BF16, 2048, 512, 50257, 0.0),   # 160 + 37
    (BF16, 5000, 512, 50257, 0.3),   # 3 x 54 + 35
    (F32, 4500, 136, 50257, 0.1),    # 5 x 37 + 12
    (F16, 9000, 256, 20011, 0.5),    # 2 x 36 + 7
    (F32, 4200, 520, 20011, 0.6),    # 2 x 34 + 11
    (BF16, 5000, 200, 50257, 0.93)])
def test_linear_ce_gradient_over_several_pieces(dtype, rows, dim, vocab, ignored):
    """Every piece of the vocabulary adds to dx, the shorter last one too."""
    x, w, b, tg = ce_inputs(rows + dim, rows, dim, vocab, dtype, True, ignored)
    size = C.c_size_t()
    a = LinearCeArgs(TYPES.index(dtype), rows, dim, vocab, 0, dim, dim, dim, dim)
    assert load_library().aideen_linear_ce_workspace(C.byref(a), None, C.byref(size)) == 0
    # without x's layouts, W's in float32 and three slabs of dx (there are at least that many)
    # there is not room for softmax - onehot of all entries at once
    planes, m = 2 if dtype == F32 else 1, -(-rows // 256) * 256
    others = 3 * m * dim * 4 + planes * planes * 2 * m * dim + (2 * vocab * dim * 4 if dtype == F32 else 0)
    assert size.value - others < m * -(-vocab // 256) * 256 * 2 * planes
    dloss = 1024.0 if dtype == F16 else 1.0
    _, _, lse, dx, _, _ = ce_check(x, w, b, tg, dloss=dloss)
    # that bound is tight enough to miss any tenth of the vocabulary
    want, e = ce_reference(x, w, b, tg, "mean", dloss, dtype)["dx"]
    keep = ((tg >= 0) & (tg < vocab)).nonzero()[:, 0]
    for part in torch.arange(vocab, device="cuda").split(-(-vocab // 10)):
        p = (x[keep].double() @ w[part].double().t() + b[part].double() - lse[keep].double()[:, None]).exp()
        share = dloss / keep.numel() * (p @ w[part].double())
        assert bool((share.abs() > 2 * (e[keep] + U[dtype] * (want[keep].abs() + e[keep]) + TINY[dtype])).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_rows_that_are_not_counted_reach_nothing(dtype):
    x, w, b, tg = ce_inputs(9, 150, 72, 300, dtype, True)
    tg[10:30], tg[149], tg[0] = -1, 300, -2147483648
    clean = K.linear_ce(x, w, tg, bias=b)
    grads = K.linear_ce_grad(x, w, tg, clean[2], bias=b)
    bad = x.clone()
    bad[10:20], bad[20:30], bad[149], bad[0] = float("nan"), float("inf"), float("nan"), -float("inf")
    loss, rows, lse = K.linear_ce(bad, w, tg, bias=b)
    for p, q in zip((loss, rows, lse), clean):
        assert torch.equal(p, q)
    for p, q in zip(K.linear_ce_grad(bad, w, tg, lse, bias=b), grads):
        assert torch.equal(p, q)
    out = (tg < 0) | (tg >= 300)
    assert bool((rows[out] == 0).all()) and bool((lse[out] == 0).all()) and bool((grads[0][out] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [0, 1, 130])
def test_linear_ce_without_counted_rows(dtype, rows):
    x, w, b, tg = ce_inputs(4, rows, 64, 300, dtype, True)
    tg.fill_(-1)
    x.fill_(float("nan"))
    loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse, bias=b)
    assert float(loss) == 0.0
    for t in (row_loss, lse, dx, dw, db):
        assert bool((t == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_masked_vocabulary(dtype):
    """A bias of -Inf (or the type's lowest value) takes entries out of the softmax."""
    x, w, b, tg = ce_inputs(6, 140, 64, 600, dtype, True)
    dead = torch.arange(600, device="cuda") % 3 == 1
    dead[256:512] = True  # a whole tile among them
    tg = torch.where(dead[tg.long()], torch.full_like(tg, 2), tg)
    low = -float("inf") if dtype != BF16 else torch.finfo(dtype).min
    b[dead] = low
    loss, rows, lse = K.linear_ce(x, w, tg, bias=b)
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse, bias=b)
    keep = (~dead).nonzero()[:, 0]
    back = torch.zeros(600, dtype=torch.int32, device="cuda")
    back[keep] = torch.arange(keep.numel(), device="cuda", dtype=torch.int32)
    ref = ce_reference(x, w[keep], b[keep], back[tg.long()], "mean", 1.0, dtype)
    for got, name in ((loss, "loss"), (rows, "rows"), (lse, "lse")):
        close(got, ref[name][0], ref[name][1])
    for got, name in ((dx, "dx"), (dw[keep], "dw"), (db[keep], "db")):
        want, e = ref[name]
        close(got, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    assert bool((dw[dead] == 0).all()) and bool((db[dead] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [3, 140])
def test_linear_ce_logits_near_the_ends_of_float32(dtype, rows):
    """Finite logits have a finite loss, also above 2^128 ln 2 = 2.36e38, where float32 does
    not hold them in base 2, and also where every entry is at the type's lowest value: such
    logits round to that value in float32, all alike, so the row's loss is log(vocabulary)."""
    x, w, b, tg = ce_inputs(61, rows, 64, 600, dtype, True)
    b.fill_(torch.finfo(dtype).min)
    loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
    assert bool((lse == torch.finfo(dtype).min).all())
    want = torch.full((rows,), 600.0, device="cuda", dtype=torch.float64).log()
    close(row_loss, want, 700 * U32 * want)  # 600 terms of e^0, added up and joined, and a logarithm
    close(loss, want[:1], 900 * U32 * want[:1])
    b.normal_()
    b[77], b[300] = 3e38, -3e38
    tg[0], tg[1], tg[2] = 77, 300, 5
    loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
    top = float(b[77].double())
    gone = top - torch.where(tg == 300, float(b[300].double()), 0.0)
    gone[tg == 77] = 0.0
    gone[tg == 300] = float("inf")  # 6e38: the one loss that float32 does not hold
    assert bool((lse.double() - top).abs().max() <= 2 * U32 * top)
    near = tg != 300
    close(row_loss[near], gone[near].double(), 4 * U32 * gone[near].double() + 1e-30)
    assert bool((row_loss[~near] == float("inf")).all())
    tg[tg == 300] = 5
    _, _, lse = K.linear_ce(x, w, tg, bias=b)
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse, bias=b)
    p = torch.zeros(rows, 600, device="cuda", dtype=torch.float64)
    p[:, 77] = 1.0
    p[torch.arange(rows, device="cuda"), tg.long()] -= 1.0
    p /= rows
    for got, want, mag in ((dx, p @ w.double(), p.abs() @ w.double().abs()), (dw, p.t() @ x.double(), p.abs().t() @ x.double().abs()),
                           (db, p.sum(0), p.abs().sum(0))):
        e = 2 * (rows + 600 + 32) * U32 * mag
        close(got, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 40, 300])
def test_linear_ce_masked_logits_that_overflow(dtype, rows):
    """An entry that a bias of -Inf masks has probability 0, also where its product with x is
    too large for float32 (in float16: where W holds an infinity), at either sign."""
    x, w, b, tg = ce_inputs(rows, rows, 48, 600, dtype, True)
    w[100:300:2] = torch.where(torch.rand(100, 1, device="cuda", generator=gen(1)) < 0.5, -1.0, 1.0).to(dtype)
    w[100:300:2] *= 3e38 if dtype != F16 else float("inf")
    out = torch.zeros(600, dtype=torch.bool, device="cuda")
    out[100:300:2] = True
    b[out] = -float("inf")
    tg[out[tg.long()]] = 1
    keep = (~out).nonzero()[:, 0]
    back = torch.zeros(600, dtype=torch.int32, device="cuda")
    back[keep] = torch.arange(keep.numel(), device="cuda", dtype=torch.int32)
    x = x.abs() + 0.25
    x[:, 0] *= 8
    ref = ce_reference(x, w[keep], b[keep], back[tg.long()], "mean", 1.0, dtype)
    loss, row_loss, lse = K.linear_ce(x, w, tg, b)
    _, dw, db = K.linear_ce_grad(x, w, tg, lse, b, want=("weight", "bias"))
    if dtype != F32 or rows < 9:  # W's largest magnitude is float32's scale
        for got, name in ((loss, "loss"), (row_loss, "rows"), (lse, "lse")):
            close(got, ref[name][0], ref[name][1])
        for got, name in ((dw[keep], "dw"), (db[keep], "db")) if dtype != F32 else ():
            want, e = ref[name]
            close(got, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    assert not bool(dw[out].any()) and not bool(db[out].any())
    assert bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 140])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_linear_ce_masked_entries_that_hold_no_numbers(dtype, rows, value):
    """A bias of -Inf takes an entry out of the loss, dW and dbias whatever its row of W holds."""
    x, w, b, tg = ce_inputs(rows, rows, 40, 300, dtype, True)
    b[[7, 290]] = -float("inf")
    tg[(tg == 7) | (tg == 290)] = 1
    loss, row_loss, lse = K.linear_ce(x, w, tg, b)
    _, dw, db = K.linear_ce_grad(x, w, tg, lse, b, want=("weight", "bias"))
    w[7], w[290, 3] = value, value
    for p, q in zip(K.linear_ce(x, w, tg, b), (loss, row_loss, lse)):
        assert torch.equal(p, q) and bool(torch.isfinite(p).all())
    got = K.linear_ce_grad(x, w, tg, lse, b, want=("weight", "bias"))
    assert torch.equal(got[1], dw) and torch.equal(got[2], db) and bool(torch.isfinite(dw).all())


def test_linear_ce_nonfinite_rows_spoil_only_themselves():
    x, w, b, tg = ce_inputs(8, 64, 32, 100, F32, True)
    x[5, 3], x[9, 1] = float("nan"), float("inf")
    _, rows, lse = K.linear_ce(x, w, tg, bias=b)
    dx, _, _ = K.linear_ce_grad(x, w, tg, lse, bias=b)
    spoilt = torch.zeros(64, dtype=torch.bool, device="cuda")
    spoilt[5] = spoilt[9] = True
    assert torch.equal(~torch.isfinite(rows), spoilt)
    assert torch.equal(~torch.isfinite(dx).all(1), spoilt)
    # a vocabulary with nothing in it: no probability to give
    rows = K.linear_ce(x[:4], w, tg[:4], bias=torch.full_like(b, -float("inf")))[1]
    assert not bool(torch.isfinite(rows).any())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [30, 257])
def test_linear_ce_infinite_row_of_w(dtype, rows):
    """A vocabulary entry that W puts at minus infinity has probability 0, and the rows
    that fill up the last tile do not reach its gradients."""
    x, w, b, tg = ce_inputs(5, rows, 72, 300, dtype, True)
    x = x.abs() + 0.25
    w[41] = float("-inf")
    tg[tg == 41] = 0
    _, _, lse = K.linear_ce(x, w, tg, b)
    _, dw, db = K.linear_ce_grad(x, w, tg, lse, b, want=("weight", "bias"))
    assert bool((dw[41] == 0).all()) and float(db[41]) == 0
    keep = [v for v in range(300) if v != 41]
    tg2 = torch.where(tg > 41, tg - 1, tg)
    _, _, lse2 = K.linear_ce(x, w[keep], tg2, b[keep])
    assert bool(torch.isfinite(lse).all())
    # either lse is off by its 300 terms' roundings and those of its logits, of 72 products each
    zabs = (x.double().abs() @ w[keep].double().abs().T + b[keep].double().abs()).amax(1)
    close(lse, lse2.double(), 2 * U32 * (2 * 72 * zabs + 2 * 300 + 4 * lse2.double().abs() + 16))


@pytest.mark.parametrize("rows", [30, 257])
def test_linear_ce_infinities_in_float32(rows):
    """As above in float32: an entry at minus infinity has probability 0, one at plus infinity
    all of it, and an infinite x has infinite logits."""
    x, w, b, tg = ce_inputs(5, rows, 72, 300, F32, True)
    x = x.abs() + 0.25
    tg[tg == 41] = 0
    keep = [v for v in range(300) if v != 41]
    ref = ce_reference(x, w[keep], b[keep], torch.where(tg > 41, tg - 1, tg), "mean", 1.0, F32)
    for where in (7, slice(None)):
        low = w.clone()
        low[41, where] = float("-inf")
        loss, row_loss, lse = K.linear_ce(x, low, tg, b)
        for got, name in ((loss, "loss"), (row_loss, "rows"), (lse, "lse")):
            close(got, ref[name][0], ref[name][1])
        _, dw, db = K.linear_ce_grad(x, low, tg, lse, b, want=("weight", "bias"))
        assert bool((dw[41] == 0).all()) and float(db[41]) == 0
        close(dw[keep], ref["dw"][0], ref["dw"][1] + U32 * ref["dw"][0].abs())
        close(db[keep], ref["db"][0], ref["db"][1] + U32 * ref["db"][0].abs())
    high = w.clone()
    high[41] = float("inf")
    assert not bool(torch.isfinite(K.linear_ce(x, high, tg, b)[1]).any())
    x[3, 5] = float("inf")
    w[:, 5] = w[:, 5].abs() + 0.25
    row_loss = K.linear_ce(x, w, tg, b)[1]
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[3] = True
    assert torch.equal(~torch.isfinite(row_loss), bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 40])
@pytest.mark.parametrize("power", [20, 33, 100, 126])
def test_linear_ce_masked_entry_that_dwarfs_the_others(dtype, rows, power):
    """An entry that a bias of -Inf masks takes no digits from the others, whatever its row of
    W holds: an unused entry's memory, say."""
    x, w, b, tg = ce_inputs(rows + power, rows, 512, 600, dtype, True)
    if dtype == F16:
        power = 14  # as large as it holds
    big = (w[100].float() * 2.0 ** power).to(dtype)
    assert bool(torch.isfinite(big).all())
    w[100], b[100] = big, -float("inf")
    tg[tg == 100] = 1
    keep = [v for v in range(600) if v != 100]
    ref = ce_reference(x, w[keep], b[keep], torch.where(tg > 100, tg - 1, tg), "mean", 1.0, dtype)
    loss, row_loss, lse = K.linear_ce(x, w, tg, b)
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse, b)
    for got, name in ((loss, "loss"), (row_loss, "rows"), (lse, "lse")):
        close(got, ref[name][0], ref[name][1])
    for got, name in ((dx, "dx"), (dw[keep], "dw"), (db[keep], "db")):
        want, e = ref[name]
        close(got, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])
    assert not bool(dw[100].any()) and float(db[100]) == 0


@pytest.mark.parametrize("rows", [7, 60, 300])
def test_linear_ce_in_float32_with_rows_of_any_magnitude(rows):
    """Rows of x and of W at powers of two apart keep all their digits in the logits: each
    logit's bound is made of its own row's and entry's products."""
    x, w, b, tg = ce_inputs(rows, rows, 96, 500, F32, True)
    g = gen(77)
    w *= 2.0 ** torch.randint(-40, 3, (500, 1), generator=g, device="cuda").float()
    w[3] *= 2.0 ** 60
    x *= 2.0 ** torch.randint(-30, 2, (rows, 1), generator=g, device="cuda").float()
    x[0], w[4] = 0.0, 0.0
    x[1] *= 2.0 ** 40
    loss, row_loss, lse = K.linear_ce(x, w, tg, b)
    ref = ce_reference(x, w, b, tg, "mean", 1.0, F32)
    for got, name in ((loss, "loss"), (row_loss, "rows")):
        close(got, ref[name][0], ref[name][1])
    # lse: off by the logits' bounds weighted with their probabilities, and by its sum's
    z = x.double() @ w.double().t() + b.double()
    ez = 2 * (96 + 16) * U32 * (x.double().abs() @ w.double().abs().t() + b.double().abs()) + 4 * U32 * z.abs()
    want = torch.logsumexp(z, 1)
    p = (z - want[:, None]).exp()
    close(lse, want, 2 * (p * ez.clamp(max=1e30)).sum(1) + 600 * U32 + 4 * U32 * want.abs())


def test_linear_ce_of_a_call_that_is_scaled_to_nan():
    """dx of rows that are not counted is 0 whatever dloss is."""
    for dtype in TYPES:
        x, w, b, tg = ce_inputs(6, 40, 24, 100, dtype, False)
        tg[::3] = -1
        _, _, lse = K.linear_ce(x, w, tg)
        dx, _, _ = K.linear_ce_grad(x, w, tg, lse, dloss=torch.tensor([float("nan")], device="cuda"))
        assert bool((dx[::3] == 0).all()) and bool(torch.isnan(dx[1::3]).all())


def test_linear_ce_in_float32_at_the_ends_of_the_range():
    """x times a power of two and W divided by it change no logit, so not a bit of the
    loss, and dW by that power alone (W stays normal: its smallest value is 1/2)."""
    g = gen(7)
    x, w = rand(g, 60, 64, std=0.3), torch.rand(200, 64, generator=g, device="cuda") / 2 + 0.5
    tg = torch.randint(0, 200, (60,), generator=g, device="cuda", dtype=torch.int32)
    far = 2.0 ** 120
    loss, row, lse = K.linear_ce(x, w, tg)
    loss2, row2, lse2 = K.linear_ce(x * far, w / far, tg)
    assert torch.equal(loss, loss2) and torch.equal(row, row2) and torch.equal(lse, lse2)
    _, dw, _ = K.linear_ce_grad(x, w, tg, lse, want=("weight",))
    _, dw2, _ = K.linear_ce_grad(x * far, w / far, tg, lse, want=("weight",))
    assert torch.equal(dw * far, dw2)


@pytest.mark.parametrize("power", [-108, 108])
@pytest.mark.parametrize("dloss", [1.0, 2.0 ** 20, 2.0 ** -20])
def test_linear_ce_gradients_in_float32_at_the_ends_of_the_range(power, dloss):
    """As above, for both gradients: they scale by that power, bit by bit (what becomes
    subnormal is rounded once more, in the kernel as here)."""
    g = gen(8)
    x, w = rand(g, 60, 64, std=0.3), torch.rand(200, 64, generator=g, device="cuda") / 2 + 0.5
    tg = torch.randint(0, 200, (60,), generator=g, device="cuda", dtype=torch.int32)
    far, c = 2.0 ** power, torch.tensor([dloss], device="cuda")
    _, _, lse = K.linear_ce(x, w, tg)
    dx, dw, _ = K.linear_ce_grad(x, w, tg, lse, dloss=c)
    dx2, dw2, _ = K.linear_ce_grad(x * far, w / far, tg, lse, dloss=c)
    assert torch.equal(dw * far, dw2) and torch.equal(dx / far, dx2)


@pytest.mark.parametrize("rows,dim", [(40, 16384), (300, 16390), (513, 4097), (300, 577), (9, 513)])
def test_linear_ce_of_deep_rows_in_float32(rows, dim):
    """Logits of positive terms, where every cut of the tensor cores has the same sign: over 512
    of dim 32 steps of 2 U32 each at most, 12 U32 for 22-bit operands and their two smaller
    products, and one rounding for each 512 of dim.  No term grows with dim but the last."""
    g = gen(dim)
    x = rand(g, rows, dim).abs()
    w = rand(g, 300, dim, std=157.0 / dim).abs()  # logits about 100
    tg = torch.randint(0, 300, (rows,), generator=g, device="cuda", dtype=torch.int32)
    _, row_loss, lse = K.linear_ce(x, w, tg)
    z = x.double() @ w.double().t()
    eps = (64 + 12 + dim // 512 + 1) * U32
    want = torch.logsumexp(z, 1)
    elz = eps * z.amax(1) + 600 * U32 + 4 * U32 * want
    close(lse, want, elz)
    zt = z.gather(1, tg.long()[:, None])[:, 0]
    close(row_loss, want - zt, elz + (dim // 32 + 16) * U32 * zt)  # the target's logit: a float32 sum by 32 lanes
    dx, dw, _ = K.linear_ce_grad(x, w, tg, lse)
    G = (z - lse.double()[:, None]).exp()  # by the lse that it gets
    eG = G * torch.expm1(eps * z + 2 * U32 * z + 16 * U32) + 2 * U32
    G[torch.arange(rows, device="cuda"), tg.long()] -= 1
    G, eG = G / rows, eG / rows
    for got, p, e, m in ((dx, G, eG, w.double()), (dw, G.t(), eG.t(), x.double())):
        close(got, p @ m, e @ m + (64 + 12 + 8 + p.shape[1] // 512) * U32 * (p.abs() @ m) + TINY[F32])


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_peaked_rows(dtype):
    """Large logits: the softmax is all but one-hot, the loss near zero or large."""
    x, w, b, tg = ce_inputs(12, 100, 64, 700, dtype, False, spread=40.0)
    tg[::2] = (x[::2].double() @ w.double().t()).argmax(1).int()
    ce_check(x, w, b, tg, dloss=64.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_at_odd_addresses(dtype):
    """Views that start between 16-byte boundaries, with row strides that are and
    are not multiples of 16 bytes."""
    for pad in (1, 8):
        x, w, b, tg = ce_inputs(14, 40, 63, 301, dtype, True, 0.1)
        bx = torch.zeros(40, 63 + pad, dtype=dtype, device="cuda")
        bw = torch.zeros(301, 63 + pad, dtype=dtype, device="cuda")
        bx[:, 1:64], bw[:, 1:64] = x, w
        bb = torch.zeros(302, dtype=dtype, device="cuda")
        bb[1:] = b
        ce_check(bx[:, 1:64], bw[:, 1:64], bb[1:], tg, dloss=16.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,pad_x,pad_w", [(250, 0, 0), (64, 2, 0), (64, 0, 2), (66, 1, 0), (66, 0, 2), (64, 4, 8)])
def test_linear_ce_row_widths(dtype, dim, pad_x, pad_w):
    """Rows that move by 16 bytes, by pairs of 16-bit elements or one by one, x and W
    alike or not."""
    x, w, b, tg = ce_inputs(15, 300, dim, 1030, dtype, True, 0.1)
    ce_check(strided(x, pad_x), strided(w, pad_w), b, tg, dloss=16.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(300, 64, 700), (33, 520, 300), (1, 24, 40), (1100, 32, 257)])
def test_linear_ce_bias_gradient_is_summed_in_float32(dtype, rows, dim, vocab):
    """softmax - onehot enters dbias unrounded: the bound has float32's steps, and the type's
    one for the result alone."""
    x, w, b, tg = ce_inputs(rows + vocab, rows, dim, vocab, dtype, True, 0.1)
    if rows > 1:
        tg[:rows // 2] = 3  # a target that comes often: its sum is all but cancelled rounding
    tg[0] = 1
    _, _, lse = K.linear_ce(x, w, tg, bias=b)
    db = K.linear_ce_grad(x, w, tg, lse, bias=b, want=("bias",))[2]
    want, e = ce_reference(x, w, b, tg, "mean", 1.0, F32)["db"]
    close(db, want, e + U[dtype] * (want.abs() + e) + TINY[dtype])


def test_linear_ce_parts_alone():
    x, w, b, tg = ce_inputs(2, 70, 48, 333, BF16, True, 0.2)
    _, _, lse = K.linear_ce(x, w, tg, bias=b)
    whole = K.linear_ce_grad(x, w, tg, lse, bias=b)
    for i, name in enumerate(("x", "weight", "bias")):
        part = K.linear_ce_grad(x, w, tg, lse, bias=b, want=(name,))
        assert torch.equal(part[i], whole[i]) and sum(p is not None for p in part) == 1


# ---- streams, graphs, devices ------------------------------------------------
def model(ids, tg, table, lw, lb, hb):
    """Embedding, norm and tied head; loss and the gradients of every leaf."""
    s = table.shape[1] ** 0.5
    e = K.embed(ids, table, scale=s)
    y, mean, rstd = K.layer_norm(e, lw, lb)
    loss, _, lse = K.linear_ce(y, table, tg, bias=hb)
    dy, dtable, dhb = K.linear_ce_grad(y, table, tg, lse, bias=hb)
    de, dlw, dlb = K.layer_norm_grad(dy, e, lw, mean, rstd)
    K.embed_grad(ids, de, table.shape[0], scale=s, into=dtable)
    return loss, dtable, dlw, dlb, dhb


def model_inputs(seed, dtype, n=192, dim=72, vocab=530):
    g = gen(seed)
    ids = torch.randint(0, vocab, (2, n // 2), generator=g, device="cuda", dtype=torch.int32)
    tg = torch.randint(0, vocab, (2, n // 2), generator=g, device="cuda", dtype=torch.int32)
    tg[0, :7] = -1
    return (ids, tg, rand(g, vocab, dim, dtype=dtype, std=0.25), rand(g, dim, dtype=dtype, std=0.1, mean=1.0),
            rand(g, dim, dtype=dtype, std=0.1), rand(g, vocab, dtype=dtype, std=0.3))


def model_reference(ids, tg, table, lw, lb, hb):
    leaves = [t.double().requires_grad_() for t in (table, lw, lb, hb)]
    t, w, b, h = leaves
    e = t[ids.long()] * t.shape[1] ** 0.5
    y = (e - e.mean(-1, keepdim=True)) / (e.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b
    z = (y @ t.t() + h).log_softmax(-1)
    keep = tg >= 0
    loss = -(z.gather(-1, tg.clamp(min=0).long()[..., None])[..., 0] * keep).sum() / keep.sum()
    return loss, torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_model_of_them_together(dtype):
    """Each of the five stages rounds its output once, and each gradient passes
    at most eight roundings of relative size U on the way to its leaf; in the
    2-norm they add as independent errors at worst linearly, doubled for the
    reuse of the rounded values in the products' other operand."""
    inputs = model_inputs(1, dtype)
    got = model(*inputs)
    loss, want = model_reference(*inputs)
    tol = 16 * U[dtype] + 1000 * U32
    assert abs(float(got[0]) - float(loss)) <= tol * float(loss)
    for g, w in zip(got[1:], want):
        assert float((g.double() - w).norm()) <= tol * float(w.norm())


def test_the_models_gradient_against_differences():
    """Central differences of the float64 loss along random directions, at a step
    of 1e-4: off by h^2 times a third derivative of a few times the loss, far
    below the float32 results' 1e-4 relative."""
    inputs = model_inputs(2, F32)
    grads = model(*inputs)[1:]
    g = gen(3)
    for i, grad in enumerate(grads):
        d = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4

        def at(step):
            moved = [t.double() for t in inputs[2:]]
            moved[i] = moved[i] + step * d
            return float(model_reference(inputs[0], inputs[1], *moved)[0])
        want = (at(h) - at(-h)) / (2 * h)
        got = float((grad.double() * d).sum())
        assert abs(got - want) <= 1e-4 * float(grad.double().norm() * d.norm()), (i, got, want)


def test_streams_and_captured_graphs():
    """The same bits on a side stream and from graphs replayed side by side, with
    inputs that change between replays."""
    sets = [model_inputs(s, BF16) for s in (11, 12, 13)]
    want = [model(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = model(*sets[1])
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
    graphs, outs, ins = [], [], []
    for k in range(2):
        s = [t.clone() for t in sets[k]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = model(*s)
        graphs.append(graph), outs.append(o), ins.append(s)
    for k in range(2):  # other inputs than at capture
        for dst, src in zip(ins[k], sets[k + 1]):
            dst.copy_(src)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    K.check()
    for k in range(2):
        assert all(torch.equal(p, q) for p, q in zip(outs[k], want[k + 1]))


@pytest.mark.parametrize("dim", [72, 640])
def test_captured_loss_and_gradient_in_float32(dim):
    """Replayed with inputs of another magnitude and another outlying masked row than at capture
    (the scales are found anew), the same bits as called."""
    sets = [ce_inputs(50 + k, 300, dim, 700, F32, True, 0.2) for k in range(3)]
    for k, (x, w, b, tg) in enumerate(sets):
        x.mul_(4.0 ** k), w.mul_(0.25 ** k)
        w[10 * k] *= 1e20
        b[10 * k] = -float("inf")
        tg[tg == 10 * k] = 5

    def work(x, w, b, tg):
        loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
        return (loss, row_loss, lse) + K.linear_ce_grad(x, w, tg, lse, bias=b)
    want = [work(*s) for s in sets]
    live = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(*live)
    for k in (1, 2, 0):
        for dst, src in zip(live, sets[k]):
            dst.copy_(src)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want[k]))
        assert bool(torch.isfinite(want[k][0]))
    K.check()


def test_calls_of_several_host_threads():
    """Threads that call at once, each on its own stream and at its own sizes (so with other
    amounts of shared memory), get what they get alone."""
    jobs = [ce_inputs(40 + i, rows, dim, 600, BF16, True) for i, (rows, dim) in
            enumerate([(200, 64), (200, 512), (1, 512), (1, 2048), (7, 64), (8, 2048)])]

    def work(x, w, b, tg):
        loss, row_loss, lse = K.linear_ce(x, w, tg, bias=b)
        return (loss, row_loss, lse) + K.linear_ce_grad(x, w, tg, lse, bias=b)
    want = [work(*job) for job in jobs]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(jobs)), []

    def caller(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for _ in range(400):
                try:
                    got = work(*jobs[k])
                except AideenError as e:
                    wrong.append((k, str(e)))
                    return
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(p, q) for p, q in zip(got, want[k])):
                wrong.append((k, "other bits"))
    threads = [threading.Thread(target=caller, args=(k,)) for k in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    K.check()


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: their last rows are what those rows alone give."""
    n, dim, k = 2_150_000, 1001, 70
    g = gen(31)
    big = torch.zeros(n, dim, dtype=F16, device="cuda")
    big[-k:] = rand(g, k, dim, dtype=F16)
    last = big[-k:].clone()
    ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    ids[-k:] = torch.randint(0, 5, (k,), generator=g, device="cuda", dtype=torch.int32)
    assert torch.equal(K.embed(n - k + torch.arange(k, device="cuda", dtype=torch.int32), big, 2.0), last * 2)
    out = K.embed(ids, last, 1.5)
    assert torch.equal(out[-k:], K.embed(ids[-k:], last, 1.5)) and not bool(out[:-k:9999].any())
    got = K.embed_grad(ids, big, 5)
    for v in range(5):
        terms = last[ids[-k:] == v].double()
        e = (k + 2) * U32 * terms.abs().sum(0)
        close(got[v], terms.sum(0), e + U[F16] * (terms.sum(0).abs() + e) + TINY[F16])
    y, mean, rstd = K.layer_norm(big, out=out)
    y1, mean1, rstd1 = K.layer_norm(last)
    assert torch.equal(y[-k:], y1) and torch.equal(mean[-k:], mean1) and torch.equal(rstd[-k:], rstd1)
    dx = K.layer_norm_grad(big, big, None, mean, rstd, want=("x",))[0]
    assert torch.equal(dx[-k:], K.layer_norm_grad(last, last, None, mean1, rstd1, want=("x",))[0])


def test_linear_ce_over_a_vocabulary_past_32_bits():
    """All entries but the last 1000 masked: the statistics and gradients are theirs alone."""
    vocab, dim, rows, k = (1 << 22) + 1000, 512, 130, 1000
    g = gen(32)
    x, w1 = rand(g, rows, dim, dtype=BF16), rand(g, k, dim, dtype=BF16, std=0.1)
    w = torch.zeros(vocab, dim, dtype=BF16, device="cuda")
    w[-k:] = w1
    b = torch.full((vocab,), float("-inf"), dtype=BF16, device="cuda")
    b[-k:] = rand(g, k, dtype=BF16)
    tg1 = torch.randint(0, k, (rows,), generator=g, device="cuda", dtype=torch.int32)
    tg = tg1 + (vocab - k)
    _, _, lse = K.linear_ce(x, w, tg, b)
    _, _, lse1 = K.linear_ce(x, w1, tg1, b[-k:].clone())
    # either is a sum of 1000 terms, whose exponents are off by a rounding each
    close(lse, lse1.double(), 2 * (k + 64) * U32 * (1 + lse1.double().abs()))
    dx, dw, db = K.linear_ce_grad(x, w, tg, lse1, b)
    dx1, dw1, db1 = K.linear_ce_grad(x, w1, tg1, lse1, b[-k:].clone())
    # the same lse, so the same softmax - onehot bit by bit; dx adds it up in other parts
    assert torch.equal(dw[-k:], dw1) and torch.equal(db[-k:], db1)
    assert not bool(dw[:-k].any()) and not bool(db[:-k].any())
    p = torch.softmax(x.double() @ w1.double().T + b[-k:].double(), 1)
    p[torch.arange(rows, device="cuda"), tg1.long()] -= 1
    terms = (p.abs() / rows) @ w1.double().abs()
    close(dx, dx1.double(), 2 * U[BF16] * dx1.double().abs() + 4 * (k + 64) * U32 * terms + 2 * TINY[BF16])


def test_python_refusals():
    t = torch.zeros(4, 8, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [lambda: K.embed(i.long(), t), lambda: K.embed(i, t.double()), lambda: K.embed(i, t.t()),
           lambda: K.embed(i, t, out=torch.zeros(4, 9, device="cuda")), lambda: K.embed(i.cpu(), t),
           lambda: K.embed_grad(i[:3], t, 5), lambda: K.embed_grad(i, t, 0),
           lambda: K.embed_grad(i, t, 5, into=torch.zeros(5, 8, device="cuda", dtype=BF16)),
           lambda: K.layer_norm(t, torch.zeros(7, device="cuda")), lambda: K.layer_norm(t, t[:, 0]),
           lambda: K.layer_norm(t, eps=-1.0), lambda: K.layer_norm(t.half(), torch.zeros(8, device="cuda")),
           lambda: K.layer_norm(torch.zeros(2, 4, 8, device="cuda").transpose(0, 1)),
           lambda: K.layer_norm_grad(t, t, None, i, i), lambda: K.layer_norm_grad(t[:2], t, None, t[:, 0], t[:, 0]),
           lambda: K.layer_norm_grad(t, t, None, t[0, :4], t[0, :4], want=()),
           lambda: K.linear_ce(t, torch.zeros(5, 7, device="cuda"), i), lambda: K.linear_ce(t, t, i[:2]),
           lambda: K.linear_ce(t, t, i, reduction="none"), lambda: K.linear_ce(t, t.half(), i),
           lambda: K.linear_ce_grad(t, t, i, t[:, 0]), lambda: K.linear_ce_grad(t, t, i, t[0, :4], want=())]
    for call in bad:
        with pytest.raises(AideenError):
            call()


def test_python_refusals_of_strided_vectors_and_counts():
    t = torch.zeros(4, 8, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: K.layer_norm(t[0, ::2]), lambda: K.linear_ce(t[0, ::2], t[:, :4], i[0]),
                 lambda: K.embed_grad(i, t, -1), lambda: K.embed_grad(i, t, 1 << 32)):
        with pytest.raises(AideenError):
            call()
    y, mean, rstd = K.layer_norm(t[0] + torch.arange(8, device="cuda"))
    assert y.shape == (8,) and mean.shape == rstd.shape == () and float(mean) == 3.5


def test_python_refuses_outputs_over_inputs():
    t, i = torch.zeros(6, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: K.embed(i, t[:5], out=t[2:]), lambda: K.embed(t[3].view(torch.int32)[2:4], t[:2], out=t[3:5]),
                 lambda: K.embed_grad(i, t[:4], 3, into=t[3:]), lambda: K.layer_norm(t[1:], out=t[:5]),
                 lambda: K.layer_norm(t[:2], t[3], out=t[2:4])):
        with pytest.raises(AideenError, match="overlap"):
            call()
    assert not bool(t.any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 512), (700, 1024), (301, 777), (33, 24), (5, 20011), (3000, 96)])
def test_layer_norm_in_place(dtype, rows, dim):
    g = gen(rows + dim)
    x, w, b = rand(g, rows, dim, dtype=dtype, mean=2.0), rand(g, dim, dtype=dtype), rand(g, dim, dtype=dtype)
    want = K.layer_norm(x, w, b)
    got = K.layer_norm(x, w, b, out=x)
    assert got[0] is x and all(torch.equal(p, q) for p, q in zip(got, want))


def test_linear_ce_refuses_a_number_for_x():
    x, w, i = torch.tensor(1.0, device="cuda"), torch.zeros(4, 1, device="cuda"), torch.tensor(0, device="cuda").int()
    for call in (lambda: K.linear_ce(x, w, i), lambda: K.linear_ce_grad(x, w, i, x)):
        with pytest.raises(AideenError, match="dimension"):
            call()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current_one():
    a = model_inputs(21, BF16)
    want = model(*a)
    with torch.cuda.device(0):
        got = model(*[t.to("cuda:1") for t in a])
    assert all(torch.equal(p, q.to("cuda:0")) for p, q in zip(want, got))
