"""Refusals of the operators on caller-owned tensors: every bad argument is
turned down on the host, with a reason, before anything is launched (no GPU is
needed, and the addresses below are never touched)."""
import ctypes as C

import pytest
import torch

from aideen_b200 import backend, operators
from aideen_b200.backend import AideenError, EmbedArgs, LayerNormArgs, LinearCeArgs

OK, INVALID = 0, 1
P = 1 << 20  # an aligned address that stands for a device pointer


@pytest.fixture(scope="module")
def lib():
    return backend.load_library()


def embed_args(**kw):
    a = dict(dtype=0, n_tokens=4, dim=8, vocab=10, scale=1.0, accumulate=0, table_ld=8, rows_ld=8)
    a.update(kw)
    return EmbedArgs(**a)


def norm_args(**kw):
    a = dict(dtype=0, rows=4, dim=8, eps=1e-5, x_ld=8, y_ld=8, dx_ld=8)
    a.update(kw)
    return LayerNormArgs(**a)


def ce_args(**kw):
    a = dict(dtype=0, rows=4, dim=8, vocab=10, reduction=0, x_ld=8, w_ld=8, dx_ld=8, dw_ld=8)
    a.update(kw)
    return LinearCeArgs(**a)


def refused(lib, rc, word):
    assert rc == INVALID
    why = lib.aideen_operator_error().decode()
    assert word in why, why


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=3), "dtype"), (dict(dim=0), "dim"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 31), "vocab"),
    (dict(n_tokens=(1 << 30) + 1), "tokens"), (dict(accumulate=2), "accumulate"), (dict(table_ld=7), "stride"),
    (dict(rows_ld=-8), "stride")])
def test_embed_refuses_bad_arguments(lib, bad, word):
    a = embed_args(**bad)
    n = C.c_size_t()
    refused(lib, lib.aideen_embed(C.byref(a), P, P, P, None), word)
    refused(lib, lib.aideen_embed_grad_workspace(C.byref(a), C.byref(n)), word)
    refused(lib, lib.aideen_embed_grad(C.byref(a), P, P, P, P, 1 << 20, None), word)


def test_embed_refuses_bad_pointers(lib):
    a, n = embed_args(), C.c_size_t()
    refused(lib, lib.aideen_embed(None, P, P, P, None), "null")
    refused(lib, lib.aideen_embed(C.byref(a), None, P, P, None), "null")
    refused(lib, lib.aideen_embed(C.byref(a), P, P + 2, P, None), "aligned")
    refused(lib, lib.aideen_embed(C.byref(a), P + 1, P, P, None), "aligned")
    assert lib.aideen_embed_grad_workspace(C.byref(a), C.byref(n)) == OK and n.value > 0
    refused(lib, lib.aideen_embed_grad(C.byref(a), P, P, None, P, n.value, None), "null")
    refused(lib, lib.aideen_embed_grad(C.byref(a), P, P, P, P, n.value - 1, None), "workspace")
    refused(lib, lib.aideen_embed_grad(C.byref(a), P, P, P, P + 16, n.value, None), "workspace")
    refused(lib, lib.aideen_embed_grad(C.byref(a), P, P, P, None, 0, None), "workspace")


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=9), "dtype"), (dict(dim=0), "dim"), (dict(rows=(1 << 30) + 1), "rows"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x_ld=7), "stride"), (dict(y_ld=0), "stride")])
def test_layer_norm_refuses_bad_arguments(lib, bad, word):
    a, n = norm_args(**bad), C.c_size_t()
    refused(lib, lib.aideen_layer_norm(C.byref(a), P, P, P, P, P, P, None), word)
    refused(lib, lib.aideen_layer_norm_grad_workspace(C.byref(a), C.byref(n)), word)
    refused(lib, lib.aideen_layer_norm_grad(C.byref(a), P, P, P, P, P, P, P, P, P, 1 << 20, None), word)


def test_layer_norm_refuses_bad_pointers(lib):
    a, n = norm_args(), C.c_size_t()
    refused(lib, lib.aideen_layer_norm(C.byref(a), None, P, P, P, P, P, None), "null")
    refused(lib, lib.aideen_layer_norm(C.byref(a), P, P + 1, P, P, P, P, None), "aligned")
    assert lib.aideen_layer_norm_grad_workspace(C.byref(a), C.byref(n)) == OK and n.value > 0
    grad = lib.aideen_layer_norm_grad
    refused(lib, grad(C.byref(a), P, P, P, P, P, None, None, None, P, n.value, None), "no output")
    refused(lib, grad(C.byref(a), P, P, P, None, P, P, P, P, P, n.value, None), "null")
    refused(lib, grad(C.byref(a), P, P, P, P, P, P, P, P, P, n.value - 1, None), "workspace")
    refused(lib, grad(C.byref(norm_args(dx_ld=3)), P, P, P, P, P, P, P, P, P, n.value, None), "stride")


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=3), "dtype"), (dict(dim=0), "dim"), (dict(vocab=0), "vocab"), (dict(rows=(1 << 24) + 1), "rows"),
    (dict(reduction=2), "reduction"), (dict(x_ld=7), "stride"), (dict(w_ld=7), "stride")])
def test_linear_ce_refuses_bad_arguments(lib, bad, word):
    a, n, m = ce_args(**bad), C.c_size_t(), C.c_size_t()
    refused(lib, lib.aideen_linear_ce_workspace(C.byref(a), C.byref(n), C.byref(m)), word)
    refused(lib, lib.aideen_linear_ce(C.byref(a), P, P, P, P, P, P, P, P, 1 << 30, None), word)
    refused(lib, lib.aideen_linear_ce_grad(C.byref(a), P, P, P, P, P, P, P, P, P, P, 1 << 30, None), word)


def test_linear_ce_refuses_bad_pointers(lib):
    a, n, m = ce_args(), C.c_size_t(), C.c_size_t()
    assert lib.aideen_linear_ce_workspace(C.byref(a), C.byref(n), C.byref(m)) == OK and n.value and m.value
    loss, grad = lib.aideen_linear_ce, lib.aideen_linear_ce_grad
    refused(lib, loss(C.byref(a), P, P, P, P, None, None, None, P, n.value, None), "no output")
    refused(lib, loss(C.byref(a), P, None, P, P, P, P, P, P, n.value, None), "null")
    refused(lib, loss(C.byref(a), P, P + 2, P, P, P, P, P, P, n.value, None), "aligned")
    refused(lib, loss(C.byref(a), P, P, P, P, P, P, P, P, n.value - 1, None), "workspace")
    refused(lib, grad(C.byref(a), P, P, P, P, P, P, None, None, None, P, m.value, None), "no output")
    refused(lib, grad(C.byref(a), P, P, P, P, None, P, P, P, P, P, m.value, None), "null")
    refused(lib, grad(C.byref(a), P, P, P, P, P, P, P, P, P, P, m.value - 1, None), "workspace")
    refused(lib, grad(C.byref(ce_args(dw_ld=7)), P, P, P, P, P, P, P, P, P, P, m.value, None), "stride")
    refused(lib, grad(C.byref(ce_args(dx_ld=7)), P, P, P, P, P, P, P, P, P, P, m.value, None), "stride")


def test_linear_ce_refuses_a_16_bit_weight_that_tma_cannot_read(lib):
    a, n, m = ce_args(dtype=1), C.c_size_t(), C.c_size_t()
    assert lib.aideen_linear_ce_workspace(C.byref(a), C.byref(n), C.byref(m)) == OK
    refused(lib, lib.aideen_linear_ce(C.byref(a), P, P + 8, P, P, P, P, P, P, n.value, None), "16-byte")
    refused(lib, lib.aideen_linear_ce_grad(C.byref(a), P, P + 2, P, P, P, P, P, P, P, P, m.value, None), "16-byte")


def test_workspaces_grow_with_the_sizes_and_stay_below_the_logits(lib):
    """The point of the pieces: at the training shard's size the gradient's
    workspace is a fraction of the float32 logits, and it stops growing with the
    vocabulary."""
    def grad_bytes(vocab, rows=16384):
        m = C.c_size_t()
        a = ce_args(dtype=1, rows=rows, dim=512, vocab=vocab, x_ld=512, w_ld=512)
        assert lib.aideen_linear_ce_workspace(C.byref(a), None, C.byref(m)) == OK
        return m.value
    assert grad_bytes(50257) < 16384 * 50257 * 4 / 4
    assert grad_bytes(200000) < 1.5 * grad_bytes(50257)


@pytest.mark.parametrize("rows,dim,most", [(1, 512, 1 << 14), (8, 2048, 1 << 16), (8, 2049, None), (9, 512, None)])
def test_workspace_of_a_few_scored_rows(lib, rows, dim, most):
    """The loss of up to 8 rows reads W where it is; more rows of float32 have it laid out."""
    n, both, m = C.c_size_t(), C.c_size_t(), C.c_size_t()
    a = ce_args(rows=rows, dim=dim, vocab=50257, x_ld=dim, w_ld=dim)
    assert lib.aideen_linear_ce_workspace(C.byref(a), C.byref(n), None) == OK
    assert lib.aideen_linear_ce_workspace(C.byref(a), C.byref(both), C.byref(m)) == OK
    assert both.value == n.value and m.value >= 4 * dim * 50257
    assert n.value <= most if most else n.value >= 4 * dim * 50257


def test_rows_of_a_matrix():
    x = torch.zeros(4, 6, 10)
    assert operators._rows(x, "f", "x") == (24, 10, 10)
    assert operators._rows(x[..., :8], "f", "x") == (24, 8, 10)
    assert operators._rows(x[0, 0], "f", "x") == (1, 10, 10)
    assert operators._rows(x[:0], "f", "x") == (0, 10, 10)
    for bad, word in [(x[..., ::2], "contiguous"), (x[0, 0, ::2], "contiguous"), (x[:, :5, :], "row stride"),
                      (x[0, :1].expand(3, 10), "overlap"), (torch.tensor(1.0), "dimension"), (x[..., :0], "dimension"),
                      (torch.zeros(1).expand(1 << 32, 1), "counts"), (torch.zeros(1).expand(2, 1 << 31), "counts")]:
        with pytest.raises(AideenError, match=word):
            operators._rows(bad, "f", "x")


@pytest.mark.parametrize("call", [
    lambda t, i: operators.embed(i, t),
    lambda t, i: operators.embed_grad(i, t, 4),
    lambda t, i: operators.layer_norm(t),
    lambda t, i: operators.layer_norm_grad(t, t, None, t, t),
    lambda t, i: operators.linear_ce(t, t, i),
    lambda t, i: operators.linear_ce_grad(t, t, i, t)])
def test_host_tensors_are_refused(call):
    with pytest.raises(AideenError, match="CUDA tensor"):
        call(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32))


def test_wanted_gradients_are_named_rightly():
    t, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for bad in (("weigth",), ("x", "w"), "dx", ["weight", None]):
        with pytest.raises(AideenError, match="want"):
            operators.layer_norm_grad(t, t, None, t, t, want=bad)
        with pytest.raises(AideenError, match="want"):
            operators.linear_ce_grad(t, t, i, t, want=bad)
    assert tuple(operators._wanted("weight", "f")) == ("weight",)
    assert tuple(operators._wanted(["bias", "x"], "f")) == ("bias", "x")


def test_outputs_must_not_overlap_inputs():
    buf = torch.zeros(40, 24)
    for out, t in [(buf[:, :8], buf[:, 8:]), (buf[:, 16:], buf[:, :16]), (buf[:20], buf[20:]), (buf[:, :8], buf[3, 8:20]),
                   (buf[5, 20:], buf[:, 4:20]), (buf[1, :4], buf[1, 4:]), (buf[:, :8], None), (buf[:0], buf),
                   (buf, buf[:0]), (buf[:8, :6], buf[10:, :6]), (buf[:, 0:1], buf[:, 1:2])]:
        operators._apart("f", "out", out, x=t)
        if t is not None:
            operators._apart("f", "out", t, x=out)
    for out, t in [(buf, buf), (buf[:, :8], buf[:, 7:]), (buf[:21], buf[20:]), (buf[:, :8], buf[3, 7:20]),
                   (buf[:, 16:], buf.view(-1)[24 * 4 + 10:24 * 4 + 17]), (buf[1, :5], buf[1, 4:]),
                   (buf, buf.view(-1)[960 - 1:]), (buf.view(20, 48)[:, :8], buf[:, :8]), (buf[:, :8], buf[0, 0])]:
        for a, b in ((out, t), (t, out)):
            with pytest.raises(AideenError, match="overlaps x"):
                operators._apart("f", "out", a, x=b)
