"""Workloads of the token-side operators: the scaled embedding lookup and its
gradient, layer normalisation and its gradient, and the linear cross entropy
over the vocabulary (loss and gradients without keeping the logits).

`own` selects who computes: False, elementary torch operations in 32 bits;
True, `aideen_b200.operators`.  Sizes are this repository's training shard
(8 x 256 tokens, d 512, vocabulary 50257), its wide configuration (d 1024), its
small test shapes, single tokens, and odd sizes between them.
"""
import math

import torch

own = False

V_FULL = 50257
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
#: the most work a drawn linear cross entropy may have: rows * dim * vocab of the largest listed one
MOST = 8192 * 512 * V_FULL


def listed():
    return [
        # one generated token enters the model: only latency counts
        dict(name="embed_one", op="embed", rows=1, dim=512, vocab=V_FULL, dtype="f32"),
        # a long batch at the wide configuration
        dict(name="embed_large", op="embed", rows=32768, dim=1024, vocab=V_FULL, dtype="bf16"),
        # the training shard: 8 x 256 Zipf tokens, a dense gradient of the whole table
        dict(name="embed_grad_shard", op="embed_grad", rows=2048, dim=512, vocab=V_FULL, dtype="f32"),
        # many tokens (an odd number), so that the frequent ids have thousands of rows each
        dict(name="embed_grad_large", op="embed_grad", rows=65521, dim=512, vocab=V_FULL, dtype="bf16"),
        # one generated token is normalised
        dict(name="layer_norm_one", op="layer_norm", rows=1, dim=512, dtype="f32"),
        # a long batch at the wide configuration
        dict(name="layer_norm_large", op="layer_norm", rows=32768, dim=1024, dtype="bf16"),
        # the training shard's backward pass with the weight's and bias's gradients
        dict(name="layer_norm_grad_shard", op="layer_norm_grad", rows=2048, dim=512, dtype="f32"),
        # odd sizes, many rows: the reduction of the weight's gradient over them
        dict(name="layer_norm_grad_odd", op="layer_norm_grad", rows=32749, dim=1000, dtype="f16"),
        # one token is scored against the whole vocabulary
        dict(name="linear_ce_one", op="linear_ce", rows=1, dim=512, vocab=V_FULL, dtype="bf16", bias=True, ignored=0.0),
        # a small vocabulary with odd sizes in 16 bits, loss and gradients under a loss scale
        dict(name="linear_ce_odd", op="linear_ce_train", rows=1021, dim=250, vocab=4999, dtype="f16", bias=True, ignored=0.2),
        # the training shard in the framework's own type: loss and every gradient
        dict(name="linear_ce_shard", op="linear_ce_train", rows=2048, dim=512, vocab=V_FULL, dtype="f32", bias=True, ignored=0.0),
        # a large 16-bit batch, a tenth of it padding
        dict(name="linear_ce_large", op="linear_ce_train", rows=8192, dim=512, vocab=V_FULL, dtype="bf16", bias=False, ignored=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng):
    """The framework's widths, or any number in their range."""
    return rng.choice([128, 256, 512, 1024]) if rng.random() < 0.5 else _log_int(rng, 96, 1024)


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "layer_norm", "layer_norm_grad", "linear_ce", "linear_ce_train", "linear_ce_train"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), dim=_dim(rng))
    if op in ("embed", "embed_grad"):
        case.update(rows=_log_int(rng, 1, 65536), vocab=_log_int(rng, 65, V_FULL))
    elif op in ("layer_norm", "layer_norm_grad"):
        case.update(rows=_log_int(rng, 1, 32768))
    else:
        vocab = V_FULL if rng.random() < 0.3 else _log_int(rng, 65, V_FULL)
        most = max(1, min(16384, MOST // (vocab * case["dim"])))
        case.update(rows=_log_int(rng, 1, most), vocab=vocab, bias=rng.random() < 0.5, ignored=rng.choice([0.0, 0.1, 0.6]))
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, n, d = DTYPES[case["dtype"]], case["rows"], case["dim"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)

    s = dict(case=case)
    if "vocab" in case:
        # Zipf-like ids: uniform in the logarithm of the rank, ranks in a fixed shuffled order
        v = case["vocab"]
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = ((v + 1.0) ** u).long().sub_(1).clamp_(0, v - 1)
        ids = ((rank * 7919 + 13) % v if v % 7919 else rank).int()
    if case["op"] == "embed":
        s.update(ids=ids, table=normal(v, d, std=0.02), scale=math.sqrt(d))
    elif case["op"] == "embed_grad":
        s.update(ids=ids, dout=normal(n, d, std=0.05), scale=math.sqrt(d))
    elif case["op"] == "layer_norm":
        s.update(x=normal(n, d, std=1.7, mean=0.3), weight=normal(d, std=0.1, mean=1.0), bias=normal(d, std=0.1))
    elif case["op"] == "layer_norm_grad":
        x = normal(n, d, std=1.7, mean=0.3)
        xf = x.double()
        mean = xf.mean(1)
        rstd = torch.rsqrt((xf - mean[:, None]).square().mean(1) + 1e-5)
        s.update(x=x, weight=normal(d, std=0.1, mean=1.0), dy=normal(n, d, std=0.05), mean=mean.float(), rstd=rstd.float())
    else:
        if case["ignored"]:
            drop = torch.rand(n, generator=g, device="cuda") < case["ignored"]
            drop[0] = False  # one counted row at least
            ids = torch.where(drop, torch.full_like(ids, -1), ids)
        # normalised hidden rows against weights that spread the logits by about 3
        s.update(x=normal(n, d), weight=normal(v, d, std=3.0 / math.sqrt(d)), targets=ids,
                 bias=normal(v, std=0.5) if case["bias"] else None,
                 dloss=torch.full((1,), 1024.0 if case["dtype"] == "f16" else 1.0, device="cuda"))
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from aideen_b200 import operators as K
    op = s["case"]["op"]
    if op == "embed":
        return K.embed(s["ids"], s["table"], scale=s["scale"])
    if op == "embed_grad":
        return K.embed_grad(s["ids"], s["dout"], s["case"]["vocab"], scale=s["scale"])
    if op == "layer_norm":
        return K.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
    if op == "layer_norm_grad":
        return K.layer_norm_grad(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
    loss, row_loss, lse = K.linear_ce(s["x"], s["weight"], s["targets"], bias=s["bias"])
    if op == "linear_ce":
        return loss, row_loss
    dx, dw, db = K.linear_ce_grad(s["x"], s["weight"], s["targets"], lse, bias=s["bias"], dloss=s["dloss"])
    return [loss, row_loss, dx, dw] + ([db] if s["bias"] is not None else [])


def _run_plain(s):
    op = s["case"]["op"]
    if op == "embed":
        ids, table = s["ids"], s["table"]
        inside = (ids >= 0) & (ids < table.shape[0])
        rows = table[ids.clamp(0, table.shape[0] - 1)].float() * s["scale"]
        return torch.where(inside[:, None], rows, torch.zeros_like(rows)).to(table.dtype)
    if op == "embed_grad":
        ids, dout, v = s["ids"], s["dout"], s["case"]["vocab"]
        inside = (ids >= 0) & (ids < v)
        rows = torch.where(inside[:, None], dout.float() * s["scale"], torch.zeros((), device="cuda"))
        grad = torch.zeros(v, dout.shape[1], device="cuda")
        grad.index_add_(0, ids.clamp(0, v - 1), rows)
        return grad.to(dout.dtype)
    if op == "layer_norm":
        x = s["x"].float()
        mean = x.mean(1)
        xc = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((xc * xc).mean(1) + 1e-5)
        y = xc * rstd[:, None] * s["weight"].float() + s["bias"].float()
        return y.to(s["x"].dtype), mean, rstd
    if op == "layer_norm_grad":
        x, dy = s["x"].float(), s["dy"].float()
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["weight"].float()
        dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        t = s["x"].dtype
        return dx.to(t), (dy * xhat).sum(0).to(t), dy.sum(0).to(t)
    x, w, tg = s["x"].float(), s["weight"].float(), s["targets"]
    counted = (tg >= 0) & (tg < w.shape[0])
    at = tg.clamp(0, w.shape[0] - 1).long()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    picked = z.gather(1, at[:, None])[:, 0]
    row_loss = torch.where(counted, lse - picked, torch.zeros_like(lse))
    n = counted.sum().clamp(min=1).float()
    loss = (row_loss.sum() / n).reshape(1)
    if op == "linear_ce":
        return loss, row_loss
    dz = e / total
    dz[torch.arange(dz.shape[0], device="cuda"), at] -= 1.0
    dz = torch.where(counted[:, None], dz, torch.zeros_like(dz)) * (s["dloss"] / n)
    t = s["x"].dtype
    out = [loss, row_loss, (dz @ w).to(t), (dz.t() @ x).to(t)]
    return out + [dz.sum(0).to(t)] if s["bias"] is not None else out


def work(case):
    n, d, b = case["rows"], case["dim"], BYTES[case["dtype"]]
    op = case["op"]
    if op == "embed":
        # each gathered row is read (a repeated id reads the same row: at most the table) and each output row written
        return dict(bytes=4 * n + min(n, case["vocab"]) * d * b + n * d * b, flops=n * d)
    if op == "embed_grad":
        return dict(bytes=4 * n + n * d * b + case["vocab"] * d * b, flops=2 * n * d)
    if op == "layer_norm":
        return dict(bytes=2 * n * d * b + 2 * d * b + 8 * n, flops=8 * n * d)
    if op == "layer_norm_grad":
        return dict(bytes=3 * n * d * b + 3 * d * b + 8 * n, flops=13 * n * d)
    v = case["vocab"]
    counted = max(1, round(n * (1.0 - case["ignored"])))
    bias = v * b if case["bias"] else 0
    if op == "linear_ce":
        return dict(bytes=counted * d * b + v * d * b + bias + 12 * n + 4, flops=2 * counted * d * v)
    # three products of this size are the formula's own: the logits, x's gradient and the weight's
    return dict(bytes=2 * (counted * d * b + v * d * b + bias) + 12 * n + 4, flops=6 * counted * d * v)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
        inside = ((s["ids"] >= 0) & (s["ids"] < case["vocab"])).nonzero()[:, 0]
        out[inside] = s["table"].double().index_select(0, s["ids"][inside]) * s["scale"]
        return out
    if op == "embed_grad":
        n, v = case["rows"], case["vocab"]
        inside = ((s["ids"] >= 0) & (s["ids"] < v)).nonzero()[:, 0]
        out = torch.zeros(v, case["dim"], dtype=torch.float64, device="cuda")
        out.index_put_((s["ids"][inside].long(),), s["dout"][inside].double(), accumulate=True)
        return out * s["scale"]
    if op == "layer_norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + 1e-5).rsqrt()
        xhat = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1)
        return torch.addcmul(s["bias"].double(), xhat, s["weight"].double()), mean, rstd
    if op == "layer_norm_grad":
        d = case["dim"]
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        r = s["rstd"].double().unsqueeze(1)
        xhat = (x - s["mean"].double().unsqueeze(1)) * r
        c1 = dy @ w / d
        c2 = (dy * xhat) @ w / d
        return r * (dy * w - c1[:, None] - c2[:, None] * xhat), torch.einsum("nd,nd->d", dy, xhat), dy.sum(0)
    n, v, d = case["rows"], case["vocab"], case["dim"]
    w, tg = s["weight"].double(), s["targets"].long()
    b = s["bias"].double() if case["bias"] else torch.zeros(v, dtype=torch.float64, device="cuda")
    keep = ((tg >= 0) & (tg < v)).nonzero()[:, 0]
    scale = float(s["dloss"]) / max(1, keep.numel())
    row_loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    dx = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    dw = torch.zeros(v, d, dtype=torch.float64, device="cuda")
    db = torch.zeros(v, dtype=torch.float64, device="cuda")
    for part in keep.split(1024):
        x = s["x"][part].double()
        logp = torch.log_softmax(torch.addmm(b, x, w.t()), dim=1)
        row_loss[part] = -logp.gather(1, tg[part, None])[:, 0]
        if op == "linear_ce_train":
            g = logp.exp_().scatter_add_(1, tg[part, None], torch.full((part.numel(), 1), -1.0, dtype=torch.float64, device="cuda"))
            g *= scale
            dx[part] = g @ w
            dw.addmm_(g.t(), x)
            db += g.sum(0)
    loss = (row_loss.sum() / max(1, keep.numel())).reshape(1)
    if op == "linear_ce":
        return loss, row_loss
    return [loss, row_loss, dx, dw] + ([db] if case["bias"] else [])
