"""Operators of language-model training as timed cases: token embeddings, block norms, distillation.

  embedding             rows of a table picked by token ids, times a scale
  embedding_backward    the table's gradient: the rows of one token summed, the rows of absent tokens zero
  block_norm            what stands between two blocks of a residual network: norm of a block's result, its
                        gate and scales, the sum with the residual stream, the norm in front of the next block
  block_norm_backward   gradients of all of it
  distill               distillation from a teacher's top logits (with a share of cross-entropy on labels),
                        losses and the logits' gradient in one call
  distill_loss          the losses alone
  distill_backward      the logits' gradient alone, from losses' gradients that are known only then

`run` computes a case in its plain form, or, where `own` is set, by the calls of `vkml_b200.Backend`.
"""
import math

import torch

own = False

_TYPE = {"f32": torch.float32, "f16": torch.float16}
_SIZE = {"f32": 4, "f16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _embedding(name, kind, batch, length, vocab, width, table, rows, scale=1.0, padded=0.0):
    return {"name": name, "kind": kind, "batch": batch, "length": length, "vocab": vocab, "width": width, "table": table,
            "rows": rows, "scale": scale, "padded": padded}


def _norm(name, kind, batch, length, width, residual, branch, norm="rms", weights="f32", gates=1, bias=False):
    return {"name": name, "kind": kind, "batch": batch, "length": length, "width": width, "residual": residual,
            "branch": branch, "norm": norm, "weights": weights, "gates": gates, "bias": bias}


def _distill(name, kind, rows, vocab, top, logits, temperature, hard):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "top": top, "logits": logits,
            "temperature": temperature, "hard": hard}


def listed():
    return [
        # a few short sequences through a small table: one call, its latency
        _embedding("embedding 4x8 of 1000", "embedding", 4, 8, 1000, 64, "f32", "f32", 8.0),
        # the tokens of a training step out of a table kept in F32, rows in the blocks' F16
        _embedding("embedding 8x2048 of 50000", "embedding", 8, 2048, 50000, 1024, "f32", "f16", 32.0),
        # its gradient: most of the table's rows have no token; a tenth of the tokens fills up short sequences
        _embedding("embedding grad 8x2048 of 50000", "embedding_backward", 8, 2048, 50000, 1024, "f32", "f16", 32.0, 0.1),
        # many more tokens than the table has rows, frequent ones by the thousand
        _embedding("embedding grad 16x8192 of 32000", "embedding_backward", 16, 8192, 32000, 1024, "f32", "f32"),
        # single tokens of a few sequences: latency
        _norm("block norm 4x1x512", "block_norm", 4, 1, 512, "f16", "f16", weights="f16"),
        # a training step's tokens, the residual stream in F32 between blocks in F16
        _norm("block norm 8x2048x4096", "block_norm", 8, 2048, 4096, "f32", "f16"),
        # the gradients with everything in F16
        _norm("block norm grad 8x2048x4096", "block_norm_backward", 8, 2048, 4096, "f16", "f16", weights="f16"),
        # LayerNorm in F32, a gate of its own for each sequence, odd sizes
        _norm("block norm grad 5x1025x1000", "block_norm_backward", 5, 1025, 1000, "f32", "f32", "layer", "f32", 5, True),
        # a small vocabulary, a few rows: latency
        _distill("distill 16x1000", "distill", 16, 1000, 8, "f32", 1.0, 0.5),
        # a training step: losses and gradient at once, the gradient scaled for F16
        _distill("distill 4096x32000", "distill", 4096, 32000, 64, "f16", 2.0, 0.0),
        # a validation step over a large vocabulary, labels beside the teacher, a last row missing
        _distill("distill loss 2047x128000", "distill_loss", 2047, 128000, 32, "f32", 1.5, 0.25),
        # the gradient when the losses' weights come later; rows that start at odd addresses
        _distill("distill grad 2048x50001", "distill_backward", 2048, 50001, 100, "f16", 2.0, 0.1),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm uniform."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _width(rng, low, high):
    """Widths as models have them, and odd ones."""
    w = _spread(rng, low, high)
    return w if rng.random() < 0.35 else max(low, w // 8 * 8) if w < 256 else w // 64 * 64


def draw(rng):
    what = rng.choice(["embedding", "embedding_backward", "block_norm", "block_norm_backward", "distill", "distill_loss",
                       "distill_backward"])
    if what.startswith("embedding"):
        batch, length, vocab, width = _spread(rng, 1, 16), _spread(rng, 1, 8192), _spread(rng, 50, 50000), _width(rng, 8, 2048)
        length = max(1, min(length, (1 << 26) // (batch * width)))
        c = _embedding("", what, batch, length, vocab, width, rng.choice(["f32", "f32", "f16"]), rng.choice(["f32", "f16"]),
                       rng.choice([1.0, round(math.sqrt(width), 3)]), rng.choice([0.0, 0.25]))
    elif what.startswith("block_norm"):
        batch, length, width = _spread(rng, 1, 16), _spread(rng, 1, 4096), _width(rng, 8, 8192)
        length = max(1, min(length, (1 << 25) // (batch * width)))
        residual, branch = rng.choice([("f32", "f32"), ("f16", "f16"), ("f32", "f16")])
        norm = rng.choice(["rms", "layer"])
        c = _norm("", what, batch, length, width, residual, branch, norm, rng.choice(["f32", branch]),
                  rng.choice([0, 1, batch]), norm == "layer")
    else:
        rows, vocab = _spread(rng, 1, 4096), _spread(rng, 10, 128000)
        rows = max(1, min(rows, (1 << 26) // vocab))
        c = _distill("", what, rows, vocab, min(vocab, _spread(rng, 1, 256)), rng.choice(["f32", "f16"]),
                     rng.choice([1.0, 1.5, 2.0, 4.0]), rng.choice([0.0, 0.1, 0.5]))
    del c["name"]
    return c


def _distinct(count, vocab):
    """How many different tokens `count` draws of _tokens have, on average (a token's share falls with its rank)."""
    edges = [min(vocab, 1.05 ** i) for i in range(int(math.log(vocab) / math.log(1.05)) + 2)]
    total = 0.0
    for a, b in zip(edges[:-1], edges[1:]):
        if b > a:
            share = math.log(b / a) / math.log(vocab) / (b - a)
            total += (b - a) * -math.expm1(-count * share)
    return min(total, count, vocab)


def work(case):
    c = case
    if c["kind"].startswith("embedding"):
        count = c["batch"] * c["length"]
        distinct = _distinct(count, c["vocab"])
        if c["kind"] == "embedding":
            return {"bytes": 8.0 * count + (distinct * _SIZE[c["table"]] + count * _SIZE[c["rows"]]) * c["width"],
                    "flops": float(count * c["width"])}
        kept = count * (1 - c["padded"])
        return {"bytes": 8.0 * count + (kept * _SIZE[c["rows"]] + c["vocab"] * _SIZE[c["table"]]) * c["width"],
                "flops": 2.0 * kept * c["width"]}
    if c["kind"].startswith("block_norm"):
        rows = c["batch"] * c["length"]
        elements = float(rows * c["width"])
        h, y, w = _SIZE[c["residual"]], _SIZE[c["branch"]], _SIZE[c["weights"]]
        vectors = (4 if c["bias"] else 2) + c["gates"]
        if c["kind"] == "block_norm":
            return {"bytes": elements * (2 * h + 2 * y) + vectors * c["width"] * w + 16.0 * rows, "flops": 12 * elements}
        return {"bytes": elements * (3 * h + 3 * y) + vectors * c["width"] * (w + 4) + 16.0 * rows, "flops": 30 * elements}
    elements = float(c["rows"] * c["vocab"])
    passes = 2 if c["kind"] != "distill_loss" else 1
    small = c["rows"] * (12.0 * c["top"] + 24)
    return {"bytes": elements * _SIZE[c["logits"]] * passes + small, "flops": elements * (4 if c["kind"] == "distill_loss" else 8)}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------

def _tokens(g, shape, vocab):
    """Token ids whose frequency falls with their rank, as those of text."""
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    return ((vocab + 1.0) ** u - 1.0).to(torch.int64).clamp_(0, vocab - 1)


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean).to(dtype)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    s = {"case": c}
    if c["kind"].startswith("embedding"):
        batch, length, vocab, width = c["batch"], c["length"], c["vocab"], c["width"]
        ids = _tokens(g, (batch, length), vocab)
        s["padding"] = vocab - 1 if c["padded"] else None
        if c["padded"]:  # every sequence ends in padding
            ids[:, length - int(length * c["padded"]):] = vocab - 1
        s["ids"] = ids
        if c["kind"] == "embedding":
            s["table"] = normal(vocab, width, scale=0.02, dtype=_TYPE[c["table"]])
            s["out"] = empty(batch, length, width, dtype=_TYPE[c["rows"]])
        else:
            s["grad"] = normal(batch, length, width, scale=0.01, dtype=_TYPE[c["rows"]])
            s["table_grad"] = empty(vocab, width, dtype=_TYPE[c["table"]])
        return s
    if c["kind"].startswith("block_norm"):
        shape, width = (c["batch"], c["length"], c["width"]), c["width"]
        th, ty, tw = _TYPE[c["residual"]], _TYPE[c["branch"]], _TYPE[c["weights"]]
        s["residual"], s["branch"] = normal(*shape, scale=2.0, dtype=th), normal(*shape, scale=0.7, dtype=ty)
        s["post_weight"], s["pre_weight"] = (normal(width, scale=0.1, mean=1.0, dtype=tw) for _ in range(2))
        s["post_bias"], s["pre_bias"] = (normal(width, scale=0.1, dtype=tw) if c["bias"] else None for _ in range(2))
        s["gate"] = normal(c["gates"], width, scale=0.3, mean=0.5, dtype=tw) if c["gates"] else None
        s["scales"] = (1.0, 0.5)
        s["out"], s["normed"] = empty(*shape, dtype=th), empty(*shape, dtype=ty)
        s["stats"] = empty(shape[0] * shape[1], 4)
        if c["kind"] == "block_norm_backward":  # the forward pass left these
            s["out"], s["normed"], s["stats"] = _norm_plain(s)
            del s["residual"]
            s["out_grad"], s["normed_grad"] = normal(*shape, dtype=th), normal(*shape, dtype=ty)
            s["residual_grad"], s["branch_grad"] = empty(*shape, dtype=th), empty(*shape, dtype=ty)
            for name in ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias"):
                s[name + "_grad"] = empty(*s[name].shape) if s[name] is not None else None
        return s
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    teacher = normal(rows, vocab, scale=2.0, dtype=torch.float32)
    s["logits"] = (teacher * 0.7 + normal(rows, vocab, scale=1.2)).to(_TYPE[c["logits"]])
    values, ids = teacher.topk(top, dim=1)
    s["teacher_logits"], s["teacher_ids"] = values.to(_TYPE[c["logits"]]), ids.to(torch.int32)
    s["labels"] = ids[:, 0].contiguous() if c["hard"] else None
    s["losses"], s["stats"] = empty(rows), empty(rows, 4)
    s["grad"] = empty(rows, vocab, dtype=_TYPE[c["logits"]])
    s["losses_grad"] = torch.rand(rows, generator=g, device="cuda").mul_(64.0)  # a loss scaled for F16
    s["losses_grad"][rows - rows // 16:] = 0.0                                   # rows of padding
    if c["kind"] == "distill_backward":
        s["stats"] = _stats_plain(s)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _standardised(x, c):
    mean = x.mean(-1, keepdim=True) if c["norm"] == "layer" else torch.zeros_like(x[..., :1])
    x = x - mean
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    return x * rstd, mean, rstd


def _affine(x, weight, bias):
    x = x * weight.float()
    return x if bias is None else x + bias.float()


def _gate_rows(s):
    """The gate of every row, or nothing: one for all, or one for each sequence."""
    return None if s["gate"] is None else s["gate"].float()[:, None, :]


def _norm_plain(s):
    c = s["case"]
    a, b = s["scales"]
    u, post_mean, post_rstd = _standardised(s["branch"].float(), c)
    u = _affine(u, s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        u = u * _gate_rows(s)
    h = s["residual"].float() * a + u * b
    n, pre_mean, pre_rstd = _standardised(h, c)
    stats = torch.cat([post_mean, post_rstd, pre_mean, pre_rstd], -1).reshape(-1, 4)
    return h.to(s["out"].dtype), _affine(n, s["pre_weight"], s["pre_bias"]).to(s["normed"].dtype), stats


def _norm_input_grad(g, hat, rstd, c):
    m = (g * hat).mean(-1, keepdim=True)
    if c["norm"] == "layer":
        return rstd * (g - g.mean(-1, keepdim=True) - hat * m)
    return rstd * (g - hat * m)


def _norm_backward_plain(s):
    c = s["case"]
    a, b = s["scales"]
    width = c["width"]
    post_mean, post_rstd, pre_mean, pre_rstd = (x.reshape(c["batch"], c["length"], 1) for x in s["stats"].unbind(1))
    hat, dn = (s["out"].float() - pre_mean) * pre_rstd, s["normed_grad"].float()
    r = {"pre_weight": (dn * hat).reshape(-1, width).sum(0), "pre_bias": dn.reshape(-1, width).sum(0)}
    ds = s["out_grad"].float() + _norm_input_grad(dn * s["pre_weight"].float(), hat, pre_rstd, c)
    hat = (s["branch"].float() - post_mean) * post_rstd
    du = ds * b
    if s["gate"] is not None:
        dgate = du * _affine(hat, s["post_weight"], s["post_bias"])
        r["gate"] = dgate.sum((0, 1), keepdim=True)[0] if c["gates"] == 1 else dgate.sum(1)
        du = du * _gate_rows(s)
    r["post_weight"], r["post_bias"] = (du * hat).reshape(-1, width).sum(0), du.reshape(-1, width).sum(0)
    dy = _norm_input_grad(du * s["post_weight"].float(), hat, post_rstd, c)
    if not c["bias"]:
        del r["pre_bias"], r["post_bias"]
    return {"residual": (ds * a).to(s["residual_grad"].dtype), "branch": dy.to(s["branch_grad"].dtype), **r}


def _embedding_plain(s):
    return (s["table"][s["ids"]].float() * s["case"]["scale"]).to(s["out"].dtype)


def _embedding_backward_plain(s):
    c = s["case"]
    ids, g = s["ids"].reshape(-1), s["grad"].reshape(-1, c["width"]).float()
    if s["padding"] is not None:
        g = g * (ids != s["padding"])[:, None]
    total = torch.zeros(c["vocab"], c["width"], device="cuda").index_add_(0, ids, g)
    return (total * c["scale"]).to(s["table_grad"].dtype)


def _logsumexp(x):
    top = x.amax(-1, keepdim=True)
    return top.squeeze(-1) + torch.log(torch.exp(x - top).sum(-1))


def _stats_plain(s):
    """A row's maximum, its log sum exp beside that over the temperature, and without the temperature where labels need it (0 where not)."""
    z, c = s["logits"].float(), s["case"]
    top = z.amax(-1, keepdim=True)
    z = z - top
    soft = torch.log(torch.exp(z / c["temperature"]).sum(-1))
    hard = torch.log(torch.exp(z).sum(-1)) if c["hard"] else torch.zeros_like(soft)
    return torch.stack([top.squeeze(-1), soft, hard, torch.zeros_like(soft)], 1)


def _teacher(s):
    t = s["teacher_logits"].float() / s["case"]["temperature"]
    log_p = t - _logsumexp(t)[:, None]
    return torch.exp(log_p), log_p


def _distill_plain(s):
    c = s["case"]
    temperature, hard = c["temperature"], c["hard"]
    ids = s["teacher_ids"].long()
    stats = s["stats"] if c["kind"] == "distill_backward" else _stats_plain(s)
    z = s["logits"].float() - stats[:, :1]
    p, log_p = _teacher(s)
    r = {}
    if c["kind"] != "distill_backward":
        log_q = z.gather(1, ids) / temperature - stats[:, 1:2]
        losses = (1 - hard) * temperature ** 2 * (p * (log_p - log_q)).sum(1)
        if hard:
            losses = losses + hard * (stats[:, 2] - z.gather(1, s["labels"][:, None])[:, 0])
        r = {"losses": losses, "stats": stats}
    if c["kind"] != "distill_loss":
        weight = s["losses_grad"][:, None]
        g = torch.exp(z / temperature - stats[:, 1:2]).scatter_add_(1, ids, -p) * ((1 - hard) * temperature)
        if hard:
            q = torch.exp(z - stats[:, 2:3])
            g = g + hard * q.scatter_add_(1, s["labels"][:, None], torch.full_like(weight, -1.0))
        r["grad"] = (g * weight).to(s["grad"].dtype)
    return r


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

_backend = None


def _gpu():
    global _backend
    if _backend is None:
        from vkml_b200 import Backend
        _backend = Backend(0)
    return _backend


def _view(t):
    """A torch tensor as the framework describes one: its address, extents, byte strides and type."""
    if t is None:
        return None
    from vkml_b200 import DType, TensorDesc
    kind = {torch.float32: DType.F32, torch.float16: DType.F16, torch.int32: DType.I32, torch.int64: DType.I64}[t.dtype]
    size = t.element_size()
    return TensorDesc(t.data_ptr(), tuple(t.shape), tuple(size * x for x in t.stride()), kind)


def _views(s):
    """The descriptions of a state's tensors, which a program makes once for a buffer and keeps with it."""
    if "views" not in s:
        s["views"] = {k: _view(t) for k, t in s.items() if t is None or isinstance(t, torch.Tensor)}
    return s["views"]


def _own(s):
    c, gpu, v = s["case"], _gpu(), _views(s)
    kind = c["kind"]
    if kind == "embedding":
        gpu.embedding(v["table"], v["ids"], v["out"], scale=c["scale"])
        return s["out"]
    if kind == "embedding_backward":
        gpu.embedding_backward(v["grad"], v["ids"], v["table_grad"], scale=c["scale"], padding_id=s["padding"])
        return s["table_grad"]
    if kind == "block_norm":
        gpu.block_norm(v["residual"], v["branch"], out=v["out"], normed=v["normed"], stats=v["stats"],
                       post_weight=v["post_weight"], post_bias=v["post_bias"], gate=v["gate"], pre_weight=v["pre_weight"],
                       pre_bias=v["pre_bias"], residual_scale=s["scales"][0], branch_scale=s["scales"][1], kind=c["norm"],
                       eps=1e-5)
        return s["out"], s["normed"], s["stats"]
    if kind == "block_norm_backward":
        gpu.block_norm_backward(v["out"], v["branch"], v["stats"], out_grad=v["out_grad"], normed_grad=v["normed_grad"],
                                residual_grad=v["residual_grad"], branch_grad=v["branch_grad"],
                                post_weight=v["post_weight"], post_bias=v["post_bias"], gate=v["gate"],
                                pre_weight=v["pre_weight"], post_weight_grad=v["post_weight_grad"],
                                post_bias_grad=v["post_bias_grad"], gate_grad=v["gate_grad"],
                                pre_weight_grad=v["pre_weight_grad"], pre_bias_grad=v["pre_bias_grad"],
                                residual_scale=s["scales"][0], branch_scale=s["scales"][1], kind=c["norm"])
        r = {"residual": s["residual_grad"], "branch": s["branch_grad"]}
        for name in ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias"):
            if s[name] is not None:
                r[name] = s[name + "_grad"]
        return r
    options = {"labels": v["labels"], "temperature": c["temperature"], "hard_weight": c["hard"]}
    if kind == "distill_backward":
        gpu.distill_loss_backward(v["logits"], v["teacher_ids"], v["teacher_logits"], v["stats"], v["grad"],
                                  losses_grad=v["losses_grad"], **options)
        return {"grad": s["grad"]}
    if kind == "distill_loss":
        gpu.distill_loss(v["logits"], v["teacher_ids"], v["teacher_logits"], v["losses"], stats=v["stats"], **options)
        return {"losses": s["losses"], "stats": s["stats"]}
    gpu.distill_loss(v["logits"], v["teacher_ids"], v["teacher_logits"], v["losses"], stats=v["stats"], grad=v["grad"],
                     losses_grad=v["losses_grad"], **options)
    return {"losses": s["losses"], "stats": s["stats"], "grad": s["grad"]}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "embedding":
        return _embedding_plain(state)
    if kind == "embedding_backward":
        return _embedding_backward_plain(state)
    if kind == "block_norm":
        return _norm_plain(state)
    if kind == "block_norm_backward":
        return _norm_backward_plain(state)
    return _distill_plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_embedding(s, c):
    if c["kind"] == "embedding":
        return torch.nn.functional.embedding(s["ids"], s["table"].double()) * c["scale"]
    # sorted tokens: a token's sum is a difference of running sums, a block of columns at a time
    ids = s["ids"].flatten()
    if s["padding"] is not None:
        ids = torch.where(ids == s["padding"], c["vocab"], ids)
    ids, order = torch.sort(ids)
    ends = torch.searchsorted(ids, torch.arange(c["vocab"], device="cuda"), right=True)
    g = s["grad"].reshape(-1, c["width"])
    parts = []
    for lo in range(0, c["width"], 256):
        upto = torch.cumsum(g[order, lo:lo + 256].double(), 0)
        upto = torch.cat([torch.zeros_like(upto[:1]), upto])[ends]
        parts.append(torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1])))
    return torch.cat(parts, 1) * c["scale"]


def _exact_norm_forward(h, y, p, c, scales):
    """(out, normed) from leaves in 64 bits."""
    def norm(x, weight, bias):
        if c["norm"] == "layer":
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            x = (x - mean) * torch.rsqrt(var + 1e-5)
        else:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        return torch.addcmul(bias, x, weight) if bias is not None else x * weight

    u = norm(y, p["post_weight"], p["post_bias"])
    if p["gate"] is not None:
        u = u * p["gate"].unsqueeze(1)
    out = h if y is None else scales[0] * h + scales[1] * u
    return out, norm(out, p["pre_weight"], p["pre_bias"])


def _exact_norm(s, c):
    names = ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias")
    p = {k: None if s[k] is None else s[k].double() for k in names}
    y = s["branch"].double()
    if c["kind"] == "block_norm":
        out, normed = _exact_norm_forward(s["residual"].double(), y, p, c, s["scales"])
        return out, normed, None
    # The same function differentiated; the residual that gives the stored sum: out = a h + b gate u.
    a, b = s["scales"]
    for k in names:
        if p[k] is not None:
            p[k].requires_grad_()
    y.requires_grad_()
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    with torch.no_grad():
        h = (s["out"].double() - _exact_norm_forward(zero, y, p, c, (a, b))[0]) / a
    h.requires_grad_()
    out, normed = _exact_norm_forward(h, y, p, c, (a, b))
    leaves = {"residual": h, "branch": y, **{k: v for k, v in p.items() if v is not None}}
    grads = torch.autograd.grad([out, normed], list(leaves.values()), [s["out_grad"].double(), s["normed_grad"].double()])
    return dict(zip(leaves, grads))


def _exact_distill(s, c):
    temperature, hard = c["temperature"], c["hard"]
    z = s["logits"].double()
    p = torch.softmax(s["teacher_logits"].double() / temperature, 1)
    soft, plain = torch.log_softmax(z / temperature, 1), torch.log_softmax(z, 1) if hard else None
    ids = s["teacher_ids"].long()
    r = {}
    if c["kind"] != "distill_backward":
        losses = (1 - hard) * temperature ** 2 * (torch.special.xlogy(p, p) - p * torch.take_along_dim(soft, ids, 1)).sum(1)
        if hard:
            losses = losses - hard * torch.take_along_dim(plain, s["labels"][:, None], 1).squeeze(1)
        r["losses"] = losses
        top = z.amax(1)
        r["stats"] = torch.stack([top, torch.logsumexp(z / temperature, 1) - top / temperature,
                                  (torch.logsumexp(z, 1) - top) * (hard > 0), torch.zeros_like(top)], 1)
    if c["kind"] != "distill_loss":
        wanted = torch.zeros_like(z).scatter_(1, ids, p)
        g = (1 - hard) * temperature * (soft.exp_() - wanted)
        if hard:
            g += hard * plain.exp_()
            g[torch.arange(c["rows"], device="cuda"), s["labels"]] -= hard
        r["grad"] = g * s["losses_grad"].double()[:, None]
    return r


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("embedding"):
        return _exact_embedding(s, case)
    if case["kind"].startswith("block_norm"):
        return _exact_norm(s, case)
    return _exact_distill(s, case)
