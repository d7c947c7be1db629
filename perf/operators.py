"""Cases of the fixed-point linear operators and of the distillation loss: their inputs, their plain forms in elementary
torch operations, their definitions in 64 bits, and the calls that a user makes of ``geo_b200.functional``.

Three kinds of case:

* ``norm``: root-mean-square norm of ``x`` (plus a residual stream) into 8-bit integers with one scale per row, and the
  integers read back as the values that they stand for;
* ``product``: 8-bit matrix product with a scale per token (row of ``x``) and per output channel (row of ``w``);
* ``distill``: loss of a student's logits against a teacher's top logits, forward alone or with its gradient.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def listed():
    return [
        # one token of a decoding step between two layers: latency
        dict(name="norm_token", kind="norm", rows=1, cols=4096, dtype="bf16", residual=True),
        # the tokens of a prompt at an ordinary width
        dict(name="norm_prompt", kind="norm", rows=4096, cols=4096, dtype="bf16", residual=True),
        # first norm of a network (nothing to add), odd sizes, the framework's own fp32
        dict(name="norm_odd", kind="norm", rows=1023, cols=2047, dtype="fp32", residual=False),
        # a long batch at a wide layer
        dict(name="norm_long", kind="norm", rows=16384, cols=8192, dtype="fp16", residual=True),
        # one token through the 1024 -> 4096 linear layer that the layer benchmark has: reads the weights once
        dict(name="product_token", kind="product", m=1, n=4096, k=1024, dtype="bf16", bias=False),
        # the 512 -> 512 classifier layer of the VGG-11-style network at its batch of 256, in fp32
        dict(name="product_batch", kind="product", m=256, n=512, k=512, dtype="fp32", bias=True),
        # a ragged batch, odd sizes on every side
        dict(name="product_odd", kind="product", m=333, n=1001, k=2047, dtype="fp16", bias=True),
        # a long prompt through a wide layer: bound by the matrix instructions
        dict(name="product_large", kind="product", m=8192, n=8192, k=8192, dtype="bf16", bias=False),
        # the 10-class networks of this repository at their batch of 256, a training step's loss
        dict(name="distill_classes", kind="distill", rows=256, vocab=10, top=3, dtype="fp32", temperature=4.0, backward=True,
             reduction="batchmean", masked=False),
        # a training step over a vocabulary
        dict(name="distill_step", kind="distill", rows=4096, vocab=32768, top=64, dtype="bf16", temperature=2.0, backward=True,
             reduction="batchmean", masked=False),
        # few rows of a large odd vocabulary, weighted rows, some without any entry; the caller weighs the rows' losses
        dict(name="distill_few", kind="distill", rows=8, vocab=131071, top=100, dtype="bf16", temperature=1.0, backward=True,
             reduction="none", masked=True),
        # scoring a student on held-out rows: the loss alone
        dict(name="distill_score", kind="distill", rows=2048, vocab=65537, top=32, dtype="fp16", temperature=1.5, backward=False,
             reduction="none", masked=True),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "product", "distill"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "norm":
        cols = _between(rng, 16, 16384)
        if rng.random() < 0.6:   # layers' widths are mostly multiples of a power of two
            cols = max(16, cols // 16 * 16)
        rows = min(_between(rng, 1, 16384), max(1, (1 << 26) // cols))
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7)
    if kind == "product":
        n, k = _between(rng, 16, 8192), _between(rng, 16, 8192)
        if rng.random() < 0.6:
            n, k = max(16, n // 16 * 16), max(16, k // 16 * 16)
        return dict(kind=kind, m=_between(rng, 1, 8192), n=n, k=k, dtype=dtype, bias=rng.random() < 0.5)
    vocab = _between(rng, 10, 131072)
    rows = min(_between(rng, 1, 8192), max(1, (1 << 26) // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, top=min(vocab, _between(rng, 1, 256)), dtype=dtype,
                temperature=round(rng.uniform(0.5, 5.0), 2), backward=rng.random() < 0.75,
                reduction=rng.choice(["batchmean", "none"]), masked=rng.random() < 0.5)


def _int8_rows(rows, cols, g, dev):
    """Random integers of a quantiser, rows 16 bytes apart as the framework's quantisers leave them."""
    t = torch.randint(-127, 128, (rows, (cols + 15) // 16 * 16), generator=g, device=dev, dtype=torch.int8)
    return t[:, :cols]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = (normal(rows, cols) * 1.5).to(dtype)
        s["residual_in"] = (normal(rows, cols) * 4).to(dtype) if case["residual"] else None
        s["weight"] = 1 + 0.25 * normal(cols)
    elif case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["xq"], s["wq"] = _int8_rows(m, k, g, dev), _int8_rows(n, k, g, dev)
        s["xs"] = torch.rand(m, generator=g, device=dev) * 0.03 + 0.01
        s["ws"] = (torch.rand(n, generator=g, device=dev) + 0.5) / (127 * math.sqrt(k))
        s["b"] = normal(n) if case["bias"] else None
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = (normal(rows, vocab) * 2.5).to(dtype).requires_grad_(case["backward"])
        values, indices = torch.topk(s["logits"].detach().float() * 0.8 + normal(rows, vocab) * 1.5, top)
        s["row_weight"] = None
        if case["masked"]:
            have = torch.randint(0, top + 1, (rows, 1), generator=g, device=dev)   # entries that a row has: none, at times
            indices = torch.where(torch.arange(top, device=dev) < have, indices, -1)
            s["row_weight"] = (torch.rand(rows, generator=g, device=dev) + 0.5) * (torch.rand(rows, generator=g, device=dev) > 0.1)
        s["indices"], s["teacher"] = indices, values.to(dtype)
        s["upstream"] = normal(rows) if case["reduction"] == "none" else None
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from geo_b200 import functional as F

    if s["kind"] == "norm":
        if s["residual_in"] is None:
            q, scale = F.rms_norm_int8(s["x"], s["weight"], eps=EPS)
            return {"y": F.dequantize_int8(q, scale, s["x"].dtype), "scale": scale}
        q, scale, total = F.rms_norm_int8(s["x"], s["weight"], residual=s["residual_in"], eps=EPS)
        return {"y": F.dequantize_int8(q, scale, s["x"].dtype), "scale": scale, "total": total}
    if s["kind"] == "product":
        return F.linear_int8(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["b"], dtype=DTYPES[s["dtype"]])
    loss = F.distillation_loss(s["logits"], s["indices"], s["teacher"], temperature=s["temperature"], weight=s["row_weight"],
                               reduction=s["reduction"])
    if not s["backward"]:
        return {"loss": loss}
    (grad,) = torch.autograd.grad(loss, s["logits"], s["upstream"])
    return {"loss": loss.detach(), "grad": grad}


def _plain(s):
    if s["kind"] == "norm":
        return _plain_norm(s)
    if s["kind"] == "product":
        return _plain_product(s)
    return _plain_distill(s)


def _plain_norm(s):
    x, dtype = s["x"], s["x"].dtype
    total = x
    if s["residual_in"] is not None:
        total = (x.float() + s["residual_in"].float()).to(dtype)
    r = total.float()
    rstd = 1 / torch.sqrt((r * r).sum(-1) / r.shape[-1] + EPS)
    p = r * s["weight"]
    top = p.abs().amax(-1)
    # the integers are of p over its row's largest value alone (the norm's factor cancels); 64 bits, because a quotient
    # next to a border between two integers would otherwise fall on either side
    q = torch.round(p.double() * 127 / top.double()[:, None])
    scale = top * rstd / 127
    out = {"y": (q.float() * scale[:, None]).to(dtype), "scale": scale}
    if s["residual_in"] is not None:
        out["total"] = total
    return out


def _plain_product(s):
    y = torch.matmul(s["xq"].float(), s["wq"].float().t()) * s["xs"][:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["dtype"]])


def _plain_distill(s):
    T, w, idx = s["temperature"], s["row_weight"], s["indices"]
    logits = s["logits"].detach()
    z = logits.float() / T
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    valid = idx >= 0
    at = idx.clamp(min=0)
    t = torch.where(valid, s["teacher"].float() / T, -math.inf)
    t_top = t.amax(-1, keepdim=True)
    live = t_top > -math.inf
    if w is not None:
        live = live & (w != 0)[:, None]
    t = t - torch.where(live, t_top, 0.0)
    pe = torch.exp(t)
    p_total = torch.where(live, pe.sum(-1, keepdim=True), 1.0)
    p = torch.where(live, pe / p_total, 0.0)
    log_ratio = (t - torch.log(p_total)) - (z.gather(-1, at) - top - torch.log(total))
    row = torch.where(p > 0, p * log_ratio, 0.0).sum(-1) * (T * T)
    if w is not None:
        row = row * w
    row = torch.where(live[:, 0], row, 0.0)
    loss = row if s["reduction"] == "none" else row.sum() / row.shape[0]
    if not s["backward"]:
        return {"loss": loss}
    factor = torch.full_like(row, 1 / row.shape[0]) if s["upstream"] is None else s["upstream"]
    if w is not None:
        factor = factor * w
    grad = (e / total).scatter_add(-1, at, torch.where(valid, -p, 0.0)) * (T * factor)[:, None]
    return {"loss": loss, "grad": torch.where(live, grad, 0.0).to(logits.dtype)}


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        streams = 4 if case["residual"] else 2   # x, residual, their sum, the values; or x and the values
        return {"bytes": n * size * streams + 4 * case["cols"] + 4 * case["rows"], "flops": 8 * n}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size + 4 * (m + n) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    n = case["rows"] * case["vocab"]
    small = case["rows"] * case["top"] * (8 + size) + 12 * case["rows"]
    return {"bytes": n * size * (2 if case["backward"] else 1) + small, "flops": n * (8 if case["backward"] else 5)}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "norm":
        total = s["x"]
        if s["residual_in"] is not None:
            total = (s["x"].double() + s["residual_in"].double()).to(s["x"].dtype)   # the sum is kept in the stream's type
        normed = total.double()
        # of the 32-bit product with the weight, by definition
        normed = (normed.float() * s["weight"]).double().div_(normed.square().mean(-1, keepdim=True).add_(EPS).sqrt_())
        scale = normed.abs().amax(-1, keepdim=True) / 127
        y = (normed / scale).round_().mul_(scale)
        out = {"y": y, "scale": scale[:, 0]}
        if s["residual_in"] is not None:
            out["total"] = total
        return out
    if case["kind"] == "product":
        y = (s["xq"].double() @ s["wq"].double().T).mul_(s["xs"].double().unsqueeze(1)).mul_(s["ws"].double())
        return y if s["b"] is None else y.add_(s["b"].double())
    T = float(case["temperature"])
    log_q = torch.log_softmax(s["logits"].detach().double() / T, -1)
    teacher = s["teacher"].double() / T
    teacher[s["indices"] < 0] = -math.inf
    live = (teacher > -math.inf).any(-1)
    if s["row_weight"] is not None:
        live &= s["row_weight"] != 0
    log_p = torch.log_softmax(torch.where(live[:, None], teacher, 0.0), -1)
    p = log_p.exp() * live[:, None]
    place = s["indices"].clamp(min=0)
    kl = torch.where(p > 0, p * (log_p - log_q.gather(-1, place)), 0.0).sum(-1) * T**2
    w = live.double() if s["row_weight"] is None else s["row_weight"].double() * live
    loss = w * kl if case["reduction"] == "none" else (w * kl).mean()
    if not case["backward"]:
        return {"loss": loss}
    up = s["upstream"].double() if s["upstream"] is not None else torch.ones_like(w) / case["rows"]
    target = torch.zeros_like(log_q)
    target.scatter_add_(-1, place, p)
    return {"loss": loss, "grad": log_q.exp_().sub_(target).mul_((T * up * w)[:, None])}
