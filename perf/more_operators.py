"""Operators of language-model training as timed cases: gated recurrence, token log probabilities, AdamW.

  recurrence            h = a h + b along a sequence, a and b from gates and inputs: what mixes a block's tokens
  recurrence_backward   the gradients of gates, inputs and the state in front
  logprobs              log probabilities of given tokens, the distribution's entropy, the likeliest alternatives
  logprobs_backward     the logits' gradient from those of log probabilities and entropies
  adamw                 an optimiser's step over all of a model's tensors, its states in 32 bits or in 8

`run` computes a case in its plain form, or, where `own` is set, by the calls of `vkml_b200.Backend`.
"""
import math

import torch

own = False

_TYPE = {"f32": torch.float32, "f16": torch.float16}
_SIZE = {"f32": 4, "f16": 2}
_CHUNK = 16    # steps between two states that a forward recurrence leaves for its backward
_BLOCK = 256   # elements that share a scale of 8-bit states
_RATE, _BETA1, _BETA2, _EPS, _DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.1
_SEED = 12345


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _recurrence(name, kind, batch, length, width, inputs, gates, form="sigmoid", ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "length": length, "width": width, "inputs": inputs, "gates": gates,
            "form": form, "ragged": ragged}


def _logprobs(name, kind, rows, vocab, logits, top=0, temperature=1.0, banned=0.0):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "logits": logits, "top": top, "temperature": temperature,
            "banned": banned}


def _adamw(name, vocab, widths, bits, grads, copies=False, step=100):
    return {"name": name, "kind": "adamw", "vocab": vocab, "widths": widths, "bits": bits, "grads": grads, "copies": copies,
            "step": step}


def listed():
    return [
        # a token of each of many sequences that are being continued, the state updated in place: latency
        _recurrence("recurrence 64x1x2048", "recurrence", 64, 1, 2048, "f16", "f16"),
        # a training step's blocks
        _recurrence("recurrence 8x4096x2048", "recurrence", 8, 4096, 2048, "f16", "f16"),
        # one long document, a width that is no power of two: few channels, many steps
        _recurrence("recurrence 1x50000x1000", "recurrence", 1, 50000, 1000, "f32", "f32", "exp"),
        # a training step's gradients
        _recurrence("recurrence grad 8x4096x2048", "recurrence_backward", 8, 4096, 2048, "f16", "f16"),
        # sequences of different lengths in an odd batch, rows at odd addresses, gates kept in F32
        _recurrence("recurrence grad 3x5001x333", "recurrence_backward", 3, 5001, 333, "f16", "f32", "exp", True),
        # the tokens that a few sequences have sampled, with what else was likely: latency
        _logprobs("logprobs 16x1000 top 5", "logprobs", 16, 1000, "f32", 5),
        # log probabilities of sampled sequences and a teacher's top logits, a validation step over a large vocabulary
        _logprobs("logprobs 4096x32000 top 20", "logprobs", 4096, 32000, "f16", 20),
        _logprobs("logprobs 2047x128000", "logprobs", 2047, 128000, "f32", 0, 0.7, 0.1),
        # a policy's gradient, with a bonus for entropy; rows that start at odd addresses
        _logprobs("logprobs grad 2048x50001", "logprobs_backward", 2048, 50001, "f16", 0, 1.0),
        # a small model's tensors: latency
        _adamw("adamw 1000x64 and 4 layers", 1000, "64-256-64-256-64", 32, "f32"),
        # the wide perceptron of the benchmark
        _adamw("adamw 4096-8192x3-1000", 0, "4096-8192-8192-8192-1000", 32, "f32"),
        # a language model trained in mixed precision with states in 8 bits, weights in F16 beside the master's
        _adamw("adamw 50000x1024 and 16, 8 bits", 50000, "-".join(["1024-4096"] * 8 + ["1024"]), 8, "f16", True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm uniform."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _width(rng, low, high):
    """Widths as models have them, and odd ones."""
    w = _spread(rng, low, high)
    return w if rng.random() < 0.35 else max(low, w // 8 * 8) if w < 256 else w // 64 * 64


def draw(rng):
    what = rng.choice(["recurrence", "recurrence", "recurrence_backward", "logprobs", "logprobs", "logprobs_backward", "adamw"])
    if what.startswith("recurrence"):
        batch, length, width = _spread(rng, 1, 64), _spread(rng, 1, 50000), _width(rng, 8, 4096)
        length = max(1, min(length, (1 << 25) // (batch * width)))
        inputs, gates = rng.choice([("f32", "f32"), ("f16", "f16"), ("f16", "f32")])
        c = _recurrence("", what, batch, length, width, inputs, gates, rng.choice(["sigmoid", "exp"]), rng.random() < 0.3)
    elif what.startswith("logprobs"):
        rows, vocab = _spread(rng, 1, 4096), _spread(rng, 10, 128000)
        rows = max(1, min(rows, (1 << 26) // vocab))
        top = min(vocab, rng.choice([0, 1, _spread(rng, 2, 128)])) if what == "logprobs" else 0
        c = _logprobs("", what, rows, vocab, rng.choice(["f32", "f16"]), top, rng.choice([0.7, 1.0, 1.5]), rng.choice([0.0, 0.0, 0.3]))
    else:
        layers, width, hidden = _spread(rng, 1, 24), _width(rng, 8, 1024), _width(rng, 8, 4096)
        layers = max(1, min(layers, (1 << 25) // (2 * width * hidden)))
        c = _adamw("", rng.choice([0, _spread(rng, 50, 30000)]), "-".join([f"{width}-{hidden}"] * layers + [str(width)]),
                   rng.choice([32, 8]), rng.choice(["f32", "f16"]), rng.random() < 0.5, _spread(rng, 1, 10000))
    del c["name"]
    return c


def _shapes(case):
    """A model's tensors: a table, then each layer's weight and bias."""
    w = [int(x) for x in case["widths"].split("-")]
    table = [(case["vocab"], w[0])] if case["vocab"] else []
    return table + [s for a, b in zip(w[:-1], w[1:]) for s in ((b, a), (b,))]


def work(case):
    c = case
    if c["kind"].startswith("recurrence"):
        rows, x, g = float(c["batch"] * c["length"]), _SIZE[c["inputs"]], _SIZE[c["gates"]]
        states = 4.0 * c["batch"] * c["width"] * math.ceil(c["length"] / _CHUNK)
        ends = 8.0 * c["batch"] * c["width"]
        if c["kind"] == "recurrence":
            return {"bytes": rows * c["width"] * (2 * x + g) + (states if c["length"] > 1 else 0) + ends, "flops": 8 * rows * c["width"]}
        return {"bytes": rows * c["width"] * (3 * x + 2 * g) + states + ends, "flops": 16 * rows * c["width"]}
    if c["kind"].startswith("logprobs"):
        elements, size = float(c["rows"] * c["vocab"]), _SIZE[c["logits"]]
        if c["kind"] == "logprobs":
            return {"bytes": elements * size + c["rows"] * (32.0 + 8 * c["top"]), "flops": 6 * elements}
        return {"bytes": 2 * elements * size + 32.0 * c["rows"], "flops": 8 * elements}
    n = float(sum(math.prod(s) for s in _shapes(c)))
    states = 16.0 if c["bits"] == 32 else 4 + 16.0 / _BLOCK
    return {"bytes": n * (8 + _SIZE[c["grads"]] + (2 if c["copies"] else 0) + states), "flops": 16 * n}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------

def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    s = {"case": c}
    if c["kind"].startswith("recurrence"):
        batch, length, width = c["batch"], c["length"], c["width"]
        shape, tx, tg = (batch, length, width), _TYPE[c["inputs"]], _TYPE[c["gates"]]
        s["x"] = normal(*shape, dtype=tx)
        means = normal(width, scale=1.5)  # channels that remember for longer than others
        if c["form"] == "sigmoid":
            s["gate"] = (normal(*shape) + means + 2.0).to(tg)
        else:
            s["gate"] = (-torch.exp(normal(*shape, scale=0.5) + means - 3.0)).to(tg)
        s["state"] = normal(batch, width)
        s["lengths"] = (uniform(batch).mul(length + 1).long().clamp_(max=length)) if c["ragged"] else None
        chunks = -(-length // _CHUNK)
        if c["kind"] == "recurrence":
            s["out"], s["states"] = empty(*shape, dtype=tx), empty(batch, chunks, width) if length > 1 else None
            s["final"] = s["state"] if length == 1 else empty(batch, width)
        else:  # the forward pass left these
            s["states"] = _recurrence_states(s, _recurrence_scan(s)[0])
            s["out_grad"], s["final_grad"] = normal(*shape, dtype=tx), normal(batch, width)
            s["x_grad"], s["gate_grad"], s["state_grad"] = empty(*shape, dtype=tx), empty(*shape, dtype=tg), empty(batch, width)
        return s
    if c["kind"].startswith("logprobs"):
        rows, vocab, top = c["rows"], c["vocab"], c["top"]
        z = normal(rows, vocab, scale=2.5)
        if c["banned"]:
            z[:, torch.randperm(vocab, generator=g, device="cuda")[:int(vocab * c["banned"])]] = -math.inf
        s["tokens"] = (z + normal(rows, vocab)).argmax(1)
        s["tokens"][rows - rows // 16:] = -1  # rows of padding
        s["logits"] = z.to(_TYPE[c["logits"]])
        s["logprobs"], s["entropies"], s["stats"] = empty(rows), empty(rows), empty(rows, 4)
        s["top_ids"] = empty(rows, top, dtype=torch.int32) if top else None
        s["top_logprobs"] = empty(rows, top) if top else None
        if c["kind"] == "logprobs_backward":
            s["stats"] = _logprobs_stats(s)
            s["logprobs_grad"] = normal(rows, scale=64.0)   # advantages, a loss scaled for F16
            s["entropies_grad"] = torch.full((rows,), 0.64, device="cuda")
            s["logprobs_grad"][rows - rows // 16:] = 0.0
            s["entropies_grad"][rows - rows // 16:] = 0.0
            s["grad"] = empty(rows, vocab, dtype=_TYPE[c["logits"]])
        return s
    # the tensors of a model in one buffer, as programs hold them, each from a multiple of a block on
    shapes = _shapes(c)
    blocks = [-(-math.prod(x) // _BLOCK) for x in shapes]
    starts = [sum(blocks[:i]) for i in range(len(blocks))]
    n = sum(blocks) * _BLOCK
    s["shapes"], s["starts"] = shapes, starts
    each = torch.tensor(blocks, device="cuda")
    spread = torch.exp(normal(len(shapes), scale=1.0) - 6.0).repeat_interleave(each)[:, None]  # gradients' sizes differ from tensor to tensor
    real = (torch.arange(_BLOCK, device="cuda")[None] + _BLOCK * _block_in_tensor(starts, blocks)[:, None]) < \
        torch.tensor([math.prod(x) for x in shapes], device="cuda").repeat_interleave(each)[:, None]
    s["params"] = (normal(n // _BLOCK, _BLOCK, scale=0.02) * real).reshape(-1)
    s["grads"] = (normal(n // _BLOCK, _BLOCK) * spread * 8.0 * real).to(_TYPE[c["grads"]]).reshape(-1)
    first, root = normal(n // _BLOCK, _BLOCK, scale=0.3) * spread * real, (normal(n // _BLOCK, _BLOCK, scale=0.3).abs_() + 0.7) * spread * real
    s["grad_scale"] = 0.125
    s["decay"] = torch.tensor([_DECAY if len(x) > 1 else 0.0 for x in shapes], device="cuda").repeat_interleave(each)[:, None]
    s["numbers"] = torch.arange(len(shapes), device="cuda").repeat_interleave(each)[:, None]
    s["elements"] = (torch.arange(_BLOCK, device="cuda")[None] + _BLOCK * _block_in_tensor(starts, blocks)[:, None]) if c["bits"] == 8 else None
    s["copy"] = s["params"].to(torch.float16) if c["copies"] else None
    if c["bits"] == 32:
        s["first"], s["second"], s["scales"] = first.reshape(-1), (root * root).reshape(-1), None
    else:
        half = torch.full((n // _BLOCK, _BLOCK), 1 << 15, device="cuda")
        a, sa = _encode(first, half, False)
        b, sb = _encode(root, half, True)
        s["first"], s["second"] = a.reshape(-1).view(torch.int32), b.reshape(-1).view(torch.int32)
        s["scales"] = torch.cat([sa, sb], 1).contiguous()  # [blocks, 2]
    return s


def _block_in_tensor(starts, blocks):
    each = torch.tensor(blocks, device="cuda")
    return torch.arange(sum(blocks), device="cuda") - torch.tensor(starts, device="cuda").repeat_interleave(each)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _coefficients(s):
    """a, b and 1 - a of every step; behind a sequence's end a = 1, b = 0.  (In 64 bits: a channel that remembers for thousands of steps
    multiplies as many decays just below 1.)"""
    c, gate, x = s["case"], s["gate"].double(), s["x"].double()
    if c["form"] == "sigmoid":
        a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
        b = rest * x
    else:
        a, rest, b = torch.exp(gate), None, x
    inside = _inside(s)
    if inside is not None:
        a, b = torch.where(inside, a, torch.ones_like(a)), torch.where(inside, b, torch.zeros_like(b))
    return a, b, rest


def _inside(s):
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["length"], device="cuda")[None] < s["lengths"][:, None])[..., None]


def _scan(a, b):
    """Running values of h = a h + b along axis 1, by doubling."""
    a, b = a.clone(), b.clone()
    step = 1
    while step < a.shape[1]:
        b[:, step:] += a[:, step:] * b[:, :-step]
        a[:, step:] *= a[:, :-step].clone()
        step *= 2
    return b


def _recurrence_scan(s):
    """(h of every step, a, 1 - a)"""
    a, b, rest = _coefficients(s)
    first = s["states"][:, 0] if s["case"]["kind"] == "recurrence_backward" and "states" in s else s["state"]
    b[:, 0] += a[:, 0] * first
    return _scan(a, b), a, rest


def _recurrence_states(s, h):
    """The state in front of every chunk of steps."""
    return torch.cat([s["state"][:, None], h[:, _CHUNK - 1:-1:_CHUNK].float()], 1)


def _recurrence_plain(s):
    h, _, _ = _recurrence_scan(s)
    states = _recurrence_states(s, h) if s["states"] is not None else None
    out, inside = h.to(s["out"].dtype), _inside(s)
    s["final"].copy_(h[:, -1])
    r = {"out": out if inside is None else out * inside, "final": s["final"]}
    if states is not None:
        r["states"] = states
    return r


def _recurrence_backward_plain(s):
    c, inside = s["case"], _inside(s)
    h, a, rest = _recurrence_scan(s)
    before = torch.cat([s["states"][:, :1], h[:, :-1]], 1)
    x, d = s["x"].double(), s["out_grad"].double()
    if inside is not None:
        d = d * inside
    # D = d + (a D of the step behind): the same scan from the end
    d[:, -1] += s["final_grad"]
    behind = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    d = _scan(behind.flip(1), d.flip(1)).flip(1)
    if c["form"] == "sigmoid":
        dx, dgate = rest * d, a * rest * (before - x) * d
    else:
        dx, dgate = d, a * before * d
    if inside is not None:
        dx, dgate = dx * inside, dgate * inside
    return {"x": dx.to(s["x_grad"].dtype), "gate": dgate.to(s["gate_grad"].dtype), "state": (a[:, 0] * d[:, 0]).float()}


def _logprobs_stats(s):
    """A row's maximum, log sum exp((z - max) / T), entropy, 0."""
    z = s["logits"].float()
    top = z.amax(1, keepdim=True)
    u = (z - top) / s["case"]["temperature"]
    e = torch.exp(u)
    total = e.sum(1)
    entropy = torch.log(total) - (e * torch.where(e > 0, u, torch.zeros_like(u))).sum(1) / total
    return torch.stack([top[:, 0], torch.log(total), entropy, torch.zeros_like(total)], 1)


def _ordered(z):
    """Whole numbers in the order of the logits, each row's equal ones in that of their columns reversed: no two alike."""
    bits = (z + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return bits * (1 << 31) + (z.shape[1] - 1 - torch.arange(z.shape[1], device="cuda"))


def _logprobs_plain(s):
    c, stats, z = s["case"], _logprobs_stats(s), s["logits"].float()

    def at(ids):
        return (z.gather(1, ids) - stats[:, :1]) / c["temperature"] - stats[:, 1:2]

    counts = s["tokens"] >= 0
    r = {"logprobs": torch.where(counts, at(s["tokens"].clamp(min=0)[:, None])[:, 0], torch.zeros_like(stats[:, 0])),
         "entropies": stats[:, 2].contiguous(), "stats": stats}
    if c["top"]:
        ids = torch.topk(_ordered(z), c["top"], 1).indices
        r["top_ids"], r["top_logprobs"] = ids.to(torch.int32), at(ids)
    return r


def _logprobs_backward_plain(s):
    c, stats = s["case"], s["stats"]
    lq = (s["logits"].float() - stats[:, :1]) / c["temperature"] - stats[:, 1:2]
    q = torch.exp(lq)
    counts = (s["tokens"] >= 0)[:, None]  # a row without a token has no log probability to change
    glp, gh = s["logprobs_grad"][:, None] * counts, s["entropies_grad"][:, None]
    g = -q * (glp + gh * (torch.where(q > 0, lq, torch.zeros_like(lq)) + stats[:, 2:3]))
    g = g.scatter_add_(1, s["tokens"].clamp(min=0)[:, None], glp)
    return {"grad": (g / c["temperature"]).to(s["grad"].dtype)}


def _mix(x):
    """Bits of a whole number below 2^32 spread over all of them."""
    x = (x ^ (x >> 16)) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x3C6EF373 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits(s):
    """32 random bits for every element of the tensors."""
    key = _mix(torch.tensor(_SEED, device="cuda"))
    key = _mix(_mix((key + s["case"]["step"]) & 0xFFFFFFFF) + s["numbers"] & 0xFFFFFFFF)
    return _mix((key + s["elements"] * 0x9E3779B9) & 0xFFFFFFFF)


def _encode(values, bits, positive):
    """Blocks [n, 256] as (bytes of 4 exponent and 3 mantissa bits, scales [n, 1]): values over the scale, up or down by 16 random bits."""
    size = values.abs()
    most = size.amax(1, keepdim=True)
    some = most >= 2.0 ** -100
    safe = torch.where(some, most, torch.ones_like(most))
    x = size * torch.where(some, 448.0 / safe, torch.zeros_like(most))
    whole = (x * 2.0 ** -120).view(torch.int32)
    code = ((whole + ((bits << 4) | 8).to(torch.int32)) >> 20).clamp(max=126)
    if positive:  # a root that is not 0 stays so
        code = torch.where((size > 0) & some, code.clamp(min=1), code)
    code = torch.where(values < 0, code + 128, code)
    return code.to(torch.uint8), torch.where(some, most * (1 / 448), torch.zeros_like(most))


def _decode(words, scales):
    code = words.view(torch.uint8).reshape(-1, _BLOCK).to(torch.int32)
    size = ((code & 127) << 20).view(torch.float32) * 2.0 ** 120
    return torch.where(code > 127, -size, size) * scales


def _adamw_plain(s):
    c, block = s["case"], (-1, _BLOCK)
    p = s["params"].view(block)
    g = s["grads"].view(block).float() * s["grad_scale"]
    if c["bits"] == 32:
        m, v = s["first"].view(block), s["second"].view(block)
    else:
        m = _decode(s["first"], s["scales"][:, :1])
        v = _decode(s["second"], s["scales"][:, 1:]) ** 2
    m = m * _BETA1 + g * (1 - _BETA1)
    v = v * _BETA2 + g * g * (1 - _BETA2)
    root = torch.sqrt(v)
    change = m / (root / math.sqrt(1 - _BETA2 ** c["step"]) + _EPS)
    p.copy_(p * (1 - _RATE * s["decay"]) - change * (_RATE / (1 - _BETA1 ** c["step"])))
    if c["copies"]:
        s["copy"].copy_(s["params"])
    if c["bits"] == 32:
        s["first"].view(block).copy_(m)
        s["second"].view(block).copy_(v)
    else:
        bits = _bits(s)
        a, sa = _encode(m, bits & 0xFFFF, False)
        b, sb = _encode(root, bits >> 16, True)
        s["first"].view(torch.uint8).copy_(a.reshape(-1))
        s["second"].view(torch.uint8).copy_(b.reshape(-1))
        s["scales"].copy_(torch.cat([sa, sb], 1))
    return _adamw_state(s)


def _adamw_state(s):
    r = {"params": s["params"]}
    if s["copy"] is not None:
        r["copy"] = s["copy"]
    if s["case"]["bits"] == 32:
        return {**r, "first": s["first"], "second": s["second"]}
    # the bytes are 8-bit floats: their values, and the scales that they are times
    return {**r, "first": s["first"].view(torch.float8_e4m3fn), "second": s["second"].view(torch.float8_e4m3fn), "scales": s["scales"]}


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
        if s["case"]["kind"] == "adamw":
            s["views"] = _table(s)
        else:
            s["views"] = {k: _view(t) for k, t in s.items() if t is None or isinstance(t, torch.Tensor)}
    return s["views"]


def _table(s):
    """The optimiser's tensors, described once."""
    from vkml_b200 import AdamWTensor, adamw_table
    tensors = []
    for shape, start in zip(s["shapes"], s["starts"]):
        at, n = start * _BLOCK, math.prod(shape)
        eight = s["scales"] is not None
        first, second = (s[k][at // 4:at // 4 + -(-n // 4)] if eight else s[k][at:at + n].view(shape) for k in ("first", "second"))
        tensors.append(AdamWTensor(
            _view(s["params"][at:at + n].view(shape)), _view(s["grads"][at:at + n].view(shape)), _view(first), _view(second),
            scales=_view(s["scales"][start:start + -(-n // _BLOCK)]) if eight else None,
            copy=_view(s["copy"][at:at + n].view(shape)) if s["copy"] is not None else None,
            weight_decay=_DECAY if len(shape) > 1 else 0.0))
    return adamw_table(tensors)


def _own(s):
    c, gpu, v = s["case"], _gpu(), _views(s)
    kind = c["kind"]
    if kind == "recurrence":
        gpu.gated_recurrence(v["x"], v["gate"], v["out"], initial=v["state"], final=v["final"], states=v["states"],
                             lengths=v["lengths"], kind=c["form"])
        r = {"out": s["out"], "final": s["final"]}
        if s["states"] is not None:
            r["states"] = s["states"]
        return r
    if kind == "recurrence_backward":
        gpu.gated_recurrence_backward(v["x"], v["gate"], v["states"], out_grad=v["out_grad"], final_grad=v["final_grad"],
                                      x_grad=v["x_grad"], gate_grad=v["gate_grad"], initial_grad=v["state_grad"],
                                      lengths=v["lengths"], kind=c["form"])
        return {"x": s["x_grad"], "gate": s["gate_grad"], "state": s["state_grad"]}
    if kind == "logprobs":
        gpu.token_logprobs(v["logits"], v["tokens"], v["logprobs"], entropies=v["entropies"], stats=v["stats"],
                           top_ids=v["top_ids"], top_logprobs=v["top_logprobs"], temperature=c["temperature"])
        r = {"logprobs": s["logprobs"], "entropies": s["entropies"], "stats": s["stats"]}
        if c["top"]:
            r["top_ids"], r["top_logprobs"] = s["top_ids"], s["top_logprobs"]
        return r
    if kind == "logprobs_backward":
        gpu.token_logprobs_backward(v["logits"], v["tokens"], v["stats"], v["grad"], logprobs_grad=v["logprobs_grad"],
                                    entropies_grad=v["entropies_grad"], temperature=c["temperature"])
        return {"grad": s["grad"]}
    gpu.adamw(v, lr=_RATE, step=c["step"], beta1=_BETA1, beta2=_BETA2, eps=_EPS, grad_scale=s["grad_scale"], seed=_SEED)
    return _adamw_state(s)


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "recurrence":
        return _recurrence_plain(state)
    if kind == "recurrence_backward":
        return _recurrence_backward_plain(state)
    if kind == "logprobs":
        return _logprobs_plain(state)
    if kind == "logprobs_backward":
        return _logprobs_backward_plain(state)
    return _adamw_plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_recurrence(s, c):
    """Step by step, and differentiated."""
    x, gate, grad = s["x"].double(), s["gate"].double(), c["kind"] == "recurrence_backward"
    h = (s["states"][:, 0] if grad else s["state"]).double()
    leaves = [x, gate, h]
    if grad:
        for t in leaves:
            t.requires_grad_()
    a = torch.sigmoid(gate) if c["form"] == "sigmoid" else gate.exp()
    b = torch.sigmoid(-gate) * x if c["form"] == "sigmoid" else x
    if s["lengths"] is not None:
        gone = torch.arange(c["length"], device="cuda").expand(c["batch"], -1).ge(s["lengths"].unsqueeze(1)).unsqueeze(2)
        a, b = a.masked_fill(gone, 1.0), b.masked_fill(gone, 0.0)
    steps, states = [], []
    for t, (at, bt) in enumerate(zip(a.unbind(1), b.unbind(1))):
        if t % _CHUNK == 0 and not grad:
            states.append(h)
        h = torch.addcmul(bt, at, h)
        steps.append(h)
    out = torch.stack(steps, 1)
    if s["lengths"] is not None:
        out = out.masked_fill(gone, 0.0)
    if not grad:
        r = {"out": out, "final": h}
        return {**r, "states": torch.stack(states, 1)} if s["states"] is not None else r
    got = torch.autograd.grad([out, h], leaves, [s["out_grad"].double(), s["final_grad"].double()])
    return dict(zip(("x", "gate", "state"), got))


def _exact_logprobs(s, c):
    # a block of rows at a time
    parts = []
    for lo in range(0, c["rows"], 1024):
        rows = slice(lo, min(lo + 1024, c["rows"]))
        z, tokens = s["logits"][rows].double(), s["tokens"][rows]
        scaled = z / c["temperature"]
        log_q = torch.log_softmax(scaled, 1)
        entropy = torch.special.entr(log_q.exp()).sum(1)
        taken = torch.take_along_dim(log_q, tokens.clamp(min=0)[:, None], 1)[:, 0].masked_fill(tokens < 0, 0.0)
        if c["kind"] == "logprobs":
            top = z.max(1).values
            r = {"logprobs": taken, "entropies": entropy,
                 "stats": torch.stack([top, torch.logsumexp(scaled, 1) - top / c["temperature"], entropy, torch.zeros_like(top)], 1)}
            if c["top"]:
                values, ids = torch.sort(z, dim=1, descending=True, stable=True)
                r["top_ids"], r["top_logprobs"] = ids[:, :c["top"]].to(torch.int32), torch.take_along_dim(log_q, ids[:, :c["top"]], 1)
        else:
            q = log_q.exp()
            one = torch.zeros_like(q)
            at = tokens.ge(0).nonzero()[:, 0]
            one[at, tokens[at]] = 1.0
            g = (s["logprobs_grad"][rows].double() * tokens.ge(0))[:, None] * (one - q)
            g -= s["entropies_grad"][rows].double()[:, None] * (q * entropy[:, None] - torch.special.entr(q))
            r = {"grad": g / c["temperature"]}
        parts.append(r)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_codes(values, draw, floor):
    """(values over the scale on the grid of 8-bit floats, scales): a part `draw` of the way up is rounded up."""
    most = values.abs().amax(1, keepdim=True)
    x = torch.where(most > 0, values.abs() * 448 / most, torch.zeros_like(values))
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    up = torch.floor(x / step + draw) * step
    if floor:
        up = torch.where(x > 0, up.clamp(min=2.0 ** -9), up)
    return up.clamp(max=448.0) * torch.sign(values), most / 448


def _exact_adamw(s, c):
    def doubled(words, scales):
        return words.view(torch.float8_e4m3fn).to(torch.float64).view(-1, _BLOCK) * scales.double()

    g = s["grads"].double().view(-1, _BLOCK) * s["grad_scale"]
    if c["bits"] == 32:
        m, v = s["first"].double().view(-1, _BLOCK), s["second"].double().view(-1, _BLOCK)
    else:
        m, v = doubled(s["first"], s["scales"][:, 0:1]), doubled(s["second"], s["scales"][:, 1:2]).square()
    m = torch.lerp(g, m, _BETA1)
    v = torch.lerp(g.square(), v, _BETA2)
    t = c["step"]
    denominator = (v / (1 - _BETA2 ** t)).sqrt() + _EPS
    p = s["params"].double().view(-1, _BLOCK)
    p = p - _RATE * (s["decay"].double() * p + m / (1 - _BETA1 ** t) / denominator)
    r = {"params": p.flatten()}
    if c["copies"]:
        r["copy"] = r["params"]
    if c["bits"] == 32:
        return {**r, "first": m.flatten(), "second": v.flatten()}
    bits = _bits(s)
    a, sa = _exact_codes(m, ((bits % 65536) * 16 + 8).double() / 2 ** 20, False)
    b, sb = _exact_codes(v.sqrt(), ((bits // 65536) * 16 + 8).double() / 2 ** 20, True)
    return {**r, "first": a.flatten(), "second": b.flatten(), "scales": torch.cat([sa, sb], 1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("recurrence"):
        return _exact_recurrence(s, case)
    if case["kind"].startswith("logprobs"):
        return _exact_logprobs(s, case)
    return _exact_adamw(s, case)
