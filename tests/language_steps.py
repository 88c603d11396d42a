"""Gated recurrences, token log probabilities and AdamW steps in 64 bits, with bounds on what the kernels' 32-bit arithmetic may be off by.

EPS is half a step of F32, relative.
"""
import numpy as np

from language import EPS

CHUNK = 16


# ---------------------------------------------------------------------------
# gated recurrence
# ---------------------------------------------------------------------------
#
# A step h' = a h + b, as h + (b - d h) or as a h + b, rounds twice: at most 2 EPS (|h'| + |h|).  Its coefficients come from an exponential and a
# reciprocal: an argument's two roundings, |gate| EPS each, and 2^-21 = 8 EPS for the functions themselves, which make the smaller one of a and 1 - a (and b) off by
# K EPS = (16 + 4 |gate|) EPS relative; where a itself is rounded (a growing state, a below a half) that is 2 EPS a |h|.  A step's error decays as its state
# does.  A kernel that divides a sequence goes through a stretch of steps three times in effect: for the stretch's own product and sum, which are rounded like
# states, and from the state in front of it: THRICE what one pass gives holds it.

THRICE = 3.0


def gates(gate, kind):
    """a, 1 - a, and b / x of every step."""
    g = gate.astype(np.float64)
    with np.errstate(over="ignore"):
        if kind == "sigmoid":
            a, d = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
            return a, d, d
        return np.exp(g), -np.expm1(g), np.ones_like(g)


def spread(gate):
    g = np.abs(np.where(np.isfinite(gate), gate, 0.0)).astype(np.float64)
    return 16 + 4 * g


def inside(lengths, shape):
    if lengths is None:
        return np.ones(shape[:2] + (1,), bool)
    return (np.arange(shape[1])[None] < np.asarray(lengths).reshape(-1, 1))[..., None]


def recurrence(x, gate, initial, lengths, kind):
    """{out, final, states, before}: (values, bounds), of [B, L, D]."""
    batch, length, width = x.shape
    valid = inside(lengths, x.shape)
    gate = np.where(valid, gate, 0)  # (behind an end it may be anything)
    a, d, scale = gates(gate, kind)
    b = scale * np.where(valid, x, 0).astype(np.float64)
    k = spread(gate)
    h = np.zeros((batch, width)) if initial is None else initial.astype(np.float64)
    e = np.zeros_like(h)
    out, error, before, before_error = (np.zeros(x.shape) for _ in range(4))
    for t in range(length):
        before[:, t], before_error[:, t] = h, e
        new = a[:, t] * h + b[:, t]
        local = (2 * np.abs(new) + 2 * np.abs(h) + 2 * a[:, t] * np.abs(h) + k[:, t] * (np.minimum(a[:, t], np.abs(d[:, t])) * np.abs(h) + np.abs(b[:, t]))) * EPS
        on = valid[:, t]
        e = np.where(on, a[:, t] * e + THRICE * local, e)
        h = np.where(on, new, h)
        out[:, t], error[:, t] = np.where(on, h, 0), np.where(on, e, 0)
    return {"out": (out, error), "final": (h, e), "states": (before[:, ::CHUNK], before_error[:, ::CHUNK]), "before": (before, before_error)}


def recurrence_backward(x, gate, initial, lengths, kind, dout, dfinal):
    """{x, gate, initial}: (gradients, bounds).  Everything is computed again from x, gate and initial: the states' errors are in the bounds."""
    batch, length, width = x.shape
    valid = inside(lengths, x.shape)
    gate = np.where(valid, gate, 0)
    a, d, scale = gates(gate, kind)
    k = spread(gate)
    before, before_error = recurrence(x, gate, initial, lengths, kind)["before"]
    x = np.where(valid, x, 0).astype(np.float64)
    dout = np.zeros(x.shape) if dout is None else np.where(valid, dout, 0).astype(np.float64)
    later = np.zeros((batch, width)) if dfinal is None else dfinal.astype(np.float64)
    e = np.zeros_like(later)
    r = {n: (np.zeros(x.shape), np.zeros(x.shape)) for n in ("x", "gate")}
    for t in range(length - 1, -1, -1):
        on = valid[:, t]
        D = dout[:, t] + later
        De = e + EPS * np.abs(D)
        dx = scale[:, t] * D
        if kind == "sigmoid":
            slope, w, we = a[:, t] * d[:, t], before[:, t] - x[:, t], before_error[:, t] + EPS * (np.abs(before[:, t]) + np.abs(x[:, t]))
        else:
            slope, w, we = a[:, t], before[:, t], before_error[:, t]
        dg = slope * w * D
        r["x"][0][:, t], r["x"][1][:, t] = np.where(on, dx, 0), np.where(on, scale[:, t] * De + k[:, t] * EPS * np.abs(dx), 0)
        r["gate"][0][:, t] = np.where(on, dg, 0)
        # (an exponential's slope that is rounded as 1 - (1 - a) is off by an EPS of 1, not of itself: it is above a half there)
        r["gate"][1][:, t] = np.where(on, slope * (we * np.abs(D) + np.abs(w) * De) + (k[:, t] + 6) * EPS * np.abs(dg), 0)
        new = a[:, t] * D
        local = (2 * np.abs(new) + 2 * np.abs(D) + 2 * a[:, t] * np.abs(D) + k[:, t] * np.minimum(a[:, t], np.abs(d[:, t])) * np.abs(D)) * EPS
        later, e = np.where(on, new, later), np.where(on, a[:, t] * De + THRICE * local, e)
    r["initial"] = (later, e)
    return r


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
#
# Exponents are differences rounded once, times a constant, rounded twice: an exponential is off by (4 |u| + 8) EPS relative (its function's 2^-22 and a
# shift's to a later maximum included), and counts in a row's sum by its share, where |u| e^u is below 1.  A sum of n terms takes n / 512 + 32 roundings, as many as a
# thread has terms and a tree.  The entropy's sum of e^u u is off by the same shares of the sum of its terms' sizes.

def _rounds(vocab):
    return vocab / 64 + 64


def logprobs(z, tokens, temperature, top=0):
    """{logprobs, entropies, stats, top_ids, top_logprobs} of rows z and their bounds (of ids: none)."""
    rows, vocab = z.shape
    z = z.astype(np.float64)
    r = {k: (np.zeros(s), np.zeros(s)) for k, s in (("logprobs", rows), ("entropies", rows), ("stats", (rows, 4)), ("top_logprobs", (rows, top)))}
    ids = np.zeros((rows, top), np.int64)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        for i in range(rows):
            most = z[i].max()  # (no number, where one is none)
            u = (z[i] - (most if most > -np.inf or most != most else 0.0)) / temperature
            p = np.exp(u)
            total = p.sum()
            log = np.log(total) if total > 0 or total != total else 0.0
            q, uu = p / total, np.where(p > 0, u, 0.0)
            turned = (q * uu).sum() if total > 0 or total != total else 0.0
            entropy = log - turned
            sum_error = (_rounds(vocab) * EPS + (q * (4 * np.abs(uu) + 8)).sum() * EPS) if total > 0 else 0.0
            # (each term of the entropy's sum: its exponential's error, its own rounding, the sum's; and the division and the difference)
            entropy_error = sum_error * (1 + np.abs(turned)) + ((q * np.abs(uu) * (4 * np.abs(uu) + 16)).sum() + _rounds(vocab) * (q * np.abs(uu)).sum() + 4 * (np.abs(turned) + log)) * EPS if total > 0 else 0.0
            log_error = sum_error + 2 * EPS * np.abs(log)
            log_q = (z[i] - (most if most > -np.inf or most != most else 0.0)) / temperature - log
            error = log_error + 4 * EPS * (np.abs(np.where(np.isfinite(u), u, 0)) + np.abs(np.where(np.isfinite(log_q), log_q, 0)))
            t = int(tokens[i]) if tokens is not None else -1
            if 0 <= t < vocab:
                r["logprobs"][0][i], r["logprobs"][1][i] = log_q[t], error[t]
            r["entropies"][0][i], r["entropies"][1][i] = entropy, entropy_error
            r["stats"][0][i], r["stats"][1][i] = [most, log, entropy, 0.0], [0.0, log_error, entropy_error, 0.0]
            order = np.lexsort((np.arange(vocab), np.where(np.isnan(z[i]), -np.inf, -z[i])))[:top]
            # (what is no number in front of +inf: their keys are alike, so set apart)
            if np.isnan(z[i]).any():
                rest = np.where(np.isnan(z[i]), 0, 1)
                order = np.lexsort((np.arange(vocab), -np.where(np.isnan(z[i]), 0, z[i]), rest))[:top]
            ids[i] = order
            r["top_logprobs"][0][i], r["top_logprobs"][1][i] = log_q[order], error[order]
    r["top_ids"] = ids
    return r


def logprobs_backward(z, tokens, stats, ulp, uh, temperature, scale):
    """(gradient, bound) by a forward call's stats (rounded to F32)."""
    rows, vocab = z.shape
    z, s = z.astype(np.float64), stats.astype(np.float64)
    g, e = np.zeros((rows, vocab)), np.zeros((rows, vocab))
    for i in range(rows):
        t = int(tokens[i]) if tokens is not None else -1
        t = t if 0 <= t < vocab else -1
        a = float(ulp[i]) if ulp is not None and t >= 0 else 0.0
        w = float(uh[i]) if uh is not None else 0.0
        if (a == 0 and w == 0) or s[i, 0] == -np.inf:
            continue
        u = (z[i] - s[i, 0]) / temperature
        log_q = u - s[i, 1]
        q = np.exp(log_q)
        lq = np.where(q > 0, log_q, 0.0)
        k = scale / temperature
        g[i] = -k * q * (a + w * (lq + s[i, 2]))
        size = np.abs(k) * q * (np.abs(a) + np.abs(w) * (np.abs(lq) + np.abs(s[i, 2])))
        # log q: the difference's rounding, the product's and the sum's; as an exponent, twice more; and the value's own few
        # (a q below 2^-126 is flushed to 0, with what it is times)
        e[i] = 2.0 ** -126 * np.abs(k) * (np.abs(a) + np.abs(w) * (np.abs(lq) + np.abs(s[i, 2]))) + size * (8 + 4 * np.where(q > 0, np.abs(np.where(np.isfinite(u), u, 0)), 0) + 4 * np.abs(lq)) * EPS + np.abs(k * w) * q * 4 * np.abs(lq) * EPS
        if t >= 0:
            g[i, t] += k * a
            e[i, t] += 4 * EPS * np.abs(k * a)
    return g, e + 2.0 ** -126 * (1 + np.abs(scale))


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

def mix(x):
    x = np.asarray(x, np.uint64)
    low = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x6A09E667)) & low
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x3C6EF373)) & low
    return x ^ (x >> np.uint64(16))


def random_bits(seed, step, number, count):
    low = np.uint64(0xFFFFFFFF)
    add = lambda x, y: (x + np.uint64(y & 0xFFFFFFFF)) & low  # noqa: E731
    key = mix(add(mix(add(mix(seed & 0xFFFFFFFF), step)), number))
    return mix((key + (np.arange(count, dtype=np.uint64) & low) * np.uint64(0x9E3779B9)) & low)


def byte_values():
    """What the 256 bytes of 8-bit states stand for."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where(c & 127 == 127, np.nan, v)
    return np.where(c > 127, -v, v)


def decode(words, scales, count):
    """Values of 8-bit states: bytes of I32 words times their block's scale."""
    return byte_values()[words.view(np.uint8)[:count]] * np.repeat(scales.astype(np.float64), 256)[:count]


def moments(g, m, v, beta1, beta2):
    """m and v after a step, and bounds: a product and a sum each round, and a coefficient is rounded."""
    g, m, v = (t.astype(np.float64) for t in (g, m, v))
    m1, v1 = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    return (m1, 6 * EPS * (np.abs(beta1 * m) + np.abs((1 - beta1) * g)) + 2.0 ** -148), (v1, 8 * EPS * v1 + 2.0 ** -147)


def update(p, m, v, lr, decay, step, beta1, beta2, eps):
    """param after a step of (values, bounds) m and v."""
    (m, me), (v, ve) = m, v
    root = np.sqrt(v)
    with np.errstate(divide="ignore", invalid="ignore"):
        root_error = np.where(v > 0, np.minimum(ve / np.maximum(root, 1e-300), np.sqrt(ve)), np.sqrt(ve)) + 2 * EPS * root
    scale = 1 / np.sqrt(1 - beta2 ** step)
    below = root * scale + eps
    below_error = root_error * scale + 4 * EPS * below
    change = lr / (1 - beta1 ** step) * m / below
    # (the host's corrections rounded to F32, the device's by expm1 of a rounded product: 1e-6 holds both)
    change_error = lr / (1 - beta1 ** step) * me / below + np.abs(change) * (below_error / below + 12 * EPS + 1e-6)
    p = p.astype(np.float64)
    new = p * (1 - lr * decay) - change
    return new, change_error + 4 * EPS * (np.abs(p) + np.abs(change))
