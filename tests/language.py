"""What the tests of the language-model operators share: device copies of strided numpy views, and the operators in 64 bits with
bounds on what 32-bit arithmetic in the kernels' order may be off by.

EPS is half a step of F32, relative.  A sum over a row is a thread's up to 16 terms and a tree over at most 1024 threads: 32 roundings at most,
64 with what its terms were computed from; so a quantity summed over a row is off by at most ROW * (the sum of its terms' sizes).
"""
import numpy as np

from vkml_b200 import TensorDesc
from vkml_b200.graph import DType

EPS = 2.0 ** -24
ROW = 64 * EPS


def half_step(dtype, value):
    """A result's own rounding (F16: half a step of its least normal's binade below that)."""
    if dtype == np.float32:
        return EPS * np.abs(value) + 2.0 ** -149
    return 2.0 ** -11 * np.abs(value) + 2.0 ** -25


def root_of(a):
    while isinstance(a.base, np.ndarray):
        a = a.base
    return a


class Space:
    """Device copies of the buffers that numpy views lie in: a view's strides and offset are kept, and what is read back shows the
    whole buffer, so that bytes outside a result can be seen to be left alone."""

    def __init__(self, backend):
        self.backend = backend
        self.buffers = {}

    def put(self, view):
        if view is None:
            return None
        root = root_of(view)
        assert root.flags["C_CONTIGUOUS"]
        if id(root) not in self.buffers:
            storage = self.backend.allocate(max(root.nbytes, 1))
            if root.nbytes:
                self.backend.copy_from_host(storage, 0, root)
            self.buffers[id(root)] = (storage, root)
        storage, _ = self.buffers[id(root)]
        offset = view.ctypes.data - root.ctypes.data if view.size else 0
        return TensorDesc(storage.data + offset, view.shape, view.strides, DType.of(view.dtype))

    def get(self, view):
        """The view's elements on the device, and whether the rest of its buffer is as it was put there."""
        storage, root = self.buffers[id(root_of(view))]
        now = np.empty_like(root)
        if root.nbytes:
            self.backend.copy_to_host(now, storage, 0)
        offset = view.ctypes.data - root.ctypes.data
        got = np.ndarray(view.shape, view.dtype, now.data, offset if view.size else 0, view.strides)
        result = got.copy()
        got[...] = view  # what was there before; the rest has to be equal then
        same = np.array_equal(now.view(np.uint8).reshape(-1), root.view(np.uint8).reshape(-1)) if root.nbytes else True
        return result, same


def rows_view(shape, dtype, layout, fill=np.nan):
    """An empty buffer's view of `shape`: dense; `pitch`: rows apart; `offset`: from an odd element; `swapped`: the leading axes' order
    in memory exchanged (rank 3)."""
    fill = np.array(fill if np.issubdtype(dtype, np.floating) else 0).astype(dtype)
    width = shape[-1]
    if layout == "dense":
        return np.full(shape, fill, dtype)
    if layout == "pitch":
        return np.full(shape[:-1] + (width + 8,), fill, dtype)[..., :width]
    if layout == "offset":
        return np.full(int(np.prod(shape)) + 3, fill, dtype)[3:].reshape(shape)
    if layout == "odd":
        return np.full(shape[:-1] + (width + 3,), fill, dtype)[..., 1:1 + width]
    if layout == "backwards":
        return np.full(shape, fill, dtype)[::-1]
    assert layout == "swapped" and len(shape) == 3
    return np.full((shape[1], shape[0], width), fill, dtype).transpose(1, 0, 2)


def placed(values, layout):
    view = rows_view(values.shape, values.dtype, layout)
    view[...] = values
    return view


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------

def embedding_backward(ids, grad, vocab, scale, padding, before):
    """(table gradient, its bound): a sum of n terms is off by at most (n + 8) roundings of its terms' sizes."""
    ids = ids.reshape(-1)
    g = grad.reshape(len(ids), grad.shape[-1]).astype(np.float64)
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    total, size = np.zeros((vocab, g.shape[1])), np.zeros((vocab, g.shape[1]))
    np.add.at(total, ids[keep], g[keep])
    np.add.at(size, ids[keep], np.abs(g[keep]))
    count = np.bincount(ids[keep], minlength=vocab)[:, None]
    base = 0.0 if before is None else before.astype(np.float64)
    return total * scale + base, (count + 8) * EPS * (size * abs(scale) + np.abs(base)), count[:, 0] > 0


# ---------------------------------------------------------------------------
# block norm
# ---------------------------------------------------------------------------

def _norm(x, layer, eps):
    mean = x.mean(-1, keepdims=True) if layer else np.zeros(x.shape[:-1] + (1,))
    r = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    return (x - mean) * r, mean, r


def block_norm(h, y, p, a, b, layer, eps, post):
    """{out, normed, stats} and bounds.  p: post_weight, post_bias, gate (of every row), pre_weight, pre_bias or None."""
    def weight(name):
        return 1.0 if p.get(name) is None else p[name].astype(np.float64)

    def bias(name):
        return 0.0 if p.get(name) is None else p[name].astype(np.float64)

    some = (h if h is not None else y).astype(np.float64)
    out, size = np.zeros_like(some), np.zeros_like(some)
    stats = np.zeros(some.shape[:-1] + (4,))
    if h is not None:
        out = a * h.astype(np.float64)
        size = np.abs(out)
    if y is not None:
        u = y.astype(np.float64)
        au = np.abs(u)
        if post:
            u, mean, r = _norm(u, layer, eps)
            stats[..., 0:1], stats[..., 1:2] = mean, r
            au = (np.abs(u) + r * np.abs(y.astype(np.float64)).mean(-1, keepdims=True)) * np.abs(weight("post_weight")) + np.abs(bias("post_bias"))
            u = u * weight("post_weight") + bias("post_bias")
        out = out + b * weight("gate") * u
        size = size + np.abs(b * weight("gate")) * au
    error = ROW * size
    hat, mean, r = _norm(out, layer, eps)
    stats[..., 2:3], stats[..., 3:4] = mean, r
    hat_error = (r * (error + error.mean(-1, keepdims=True)) + np.abs(hat) * (np.abs(hat) * r * error).mean(-1, keepdims=True) +
                 ROW * (np.abs(hat) + r * np.abs(out).mean(-1, keepdims=True)))
    normed = hat * weight("pre_weight") + bias("pre_bias")
    normed_error = hat_error * np.abs(weight("pre_weight")) + 4 * EPS * (np.abs(normed) + np.abs(bias("pre_bias")))
    return {"out": (out, error), "normed": (normed, normed_error), "stats": stats}


def block_norm_backward(out, y, stats, dout, dn, p, a, b, layer, post, shape):
    """Gradients and their bounds, from the stored sum and the forward pass's statistics; `gate` stands for its gradient in every row."""
    def weight(name):
        return 1.0 if p.get(name) is None else p[name].astype(np.float64)

    def mean(x):
        return x.mean(-1, keepdims=True)

    def through(g, g_error, hat, r):
        k0, k1 = mean(g) if layer else 0.0, mean(g * hat)
        d = r * (g - k0 - hat * k1)
        error = r * (g_error + mean(g_error) + np.abs(hat) * mean(g_error * np.abs(hat)) + ROW * (np.abs(g) + mean(np.abs(g)) + np.abs(hat) * mean(np.abs(g * hat))))
        return d, error

    m2, r2, m1, r1 = (stats.astype(np.float64).reshape(shape[:-1] + (4,))[..., i:i + 1] for i in range(4))
    got = {}
    ds, error = np.zeros(shape), np.zeros(shape)
    if dout is not None:
        ds = dout.astype(np.float64)
    if dn is not None:
        hat, g = (out.astype(np.float64) - m1) * r1, dn.astype(np.float64)
        got["pre_weight"] = (g * hat, 4 * EPS * np.abs(g * hat))
        got["pre_bias"] = (g, np.zeros(shape))
        d, error = through(g * weight("pre_weight"), 2 * EPS * np.abs(g * weight("pre_weight")), hat, r1)
        ds = ds + d
        error = error + EPS * np.abs(ds)
    got["residual"] = (a * ds, abs(a) * error + EPS * np.abs(a * ds))
    if y is not None:
        u = y.astype(np.float64)
        hat = (u - m2) * r2 if post else u
        u = hat * weight("post_weight") + (p["post_bias"].astype(np.float64) if p.get("post_bias") is not None else 0.0)
        du, du_error = b * ds, abs(b) * error + EPS * np.abs(b * ds)
        u_size = np.abs(hat * weight("post_weight")) + np.abs(u - hat * weight("post_weight"))
        got["gate"] = (du * u, du_error * np.abs(u) + 8 * EPS * np.abs(du) * u_size)
        du, du_error = du * weight("gate"), (du_error + EPS * np.abs(du)) * np.abs(weight("gate"))
        got["post_bias"] = (du, du_error)
        got["post_weight"] = (du * hat, du_error * np.abs(hat) + 4 * EPS * np.abs(du * hat))
        if post:
            q = du * weight("post_weight")
            du, du_error = through(q, (du_error + 2 * EPS * np.abs(du)) * np.abs(weight("post_weight")), hat, r2)
        got["branch"] = (du, du_error)
    return got


def column_sum(term, axes):
    """A sum over rows and its bound: as many roundings as terms at most, and a few for the partial sums."""
    value, error = term
    n = np.prod([value.shape[i] for i in axes]) if value.size else 0
    return value.sum(axes), (error.sum(axes) + (n + 16) * EPS * np.abs(value).sum(axes))


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------

def distill(z, ids, t, labels, weights, temperature, hard, scale, stats=None):
    """{losses, stats, grad} and bounds, a row at a time.  stats: the gradient goes by these (a forward call's, rounded to F32)."""
    rows, vocab = z.shape
    c, T = hard, temperature
    terms = vocab / 512 + 32   # additions in a row's sum of exponentials, one thread's and the tree's
    sum_error = terms * EPS + 2.0 ** -21   # and the exponentials' own error, their argument's included
    out = {k: (np.zeros(s), np.zeros(s)) for k, s in (("losses", (rows,)), ("stats", (rows, 4)), ("grad", (rows, vocab)))}
    z, t = z.astype(np.float64), t.astype(np.float64)

    def put(name, at, value, error):
        out[name][0][at], out[name][1][at] = value, error

    def split(x):
        """The maximum (0 where it is -inf) and the logarithm of the sum beside it: a row of one low value keeps its logarithm."""
        top = x.max() if len(x) else -np.inf
        top = top if top > -np.inf else 0.0
        return top, np.log(np.exp(x - top).sum())

    def log_softmax(x, top, log):
        return (x - top) - (log if log > -np.inf else 0.0)

    def sized(x):
        return np.where(np.isfinite(x), np.abs(x), 0)

    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        for r in range(rows):
            keep = (ids[r] >= 0) & (ids[r] < vocab)
            tk, kk = t[r][keep] / T, ids[r][keep]
            taught = c < 1 and len(tk) > 0 and tk.max() > -np.inf
            label = int(labels[r]) if labels is not None and c > 0 and 0 <= labels[r] < vocab else -1
            (top_soft, log_soft), (top, log_hard) = split(z[r] / T), split(z[r])
            put("stats", r, [z[r].max(), log_soft if c < 1 else 0.0, log_hard if c > 0 else 0.0, 0.0],
                [0.0, sum_error + 4 * EPS * abs(log_soft), sum_error + 4 * EPS * abs(log_hard), 0.0])
            q_soft, q_hard = log_softmax(z[r] / T, top_soft, log_soft), log_softmax(z[r], top, log_hard)
            loss = error = 0.0
            if taught:
                log_p = log_softmax(tk, *split(tk))
                p = np.exp(log_p)
                on = p > 0
                log_q = q_soft[kk]
                loss += (1 - c) * T * T * (p[on] * (log_p[on] - log_q[on])).sum()
                size = (p[on] * (np.abs(log_p[on]) + sized(log_q[on]) + 1)).sum() + np.abs(tk[on] - tk[on].max()).max()
                error += (1 - c) * T * T * (sum_error + (len(tk) + 32) * EPS * size)
            if label >= 0:
                loss -= c * q_hard[label]
                error += c * (sum_error + 8 * EPS * (sized(q_hard[label]) + 2 * sized(log_hard)))
            put("losses", r, loss, error)
            w = scale * (1.0 if weights is None else float(weights[r]))
            g, e = np.zeros(vocab), np.zeros(vocab)
            if w != 0:
                if stats is not None:
                    s = stats[r].astype(np.float64)
                    top = s[0] if s[0] > -np.inf else 0.0
                    q_soft, q_hard = log_softmax(z[r] / T, top / T, s[1]), log_softmax(z[r], top, s[2])
                if taught:
                    q = np.exp(q_soft)
                    g += w * (1 - c) * T * q
                    e += np.abs(w * (1 - c) * T) * q * (sum_error + 8 * EPS * (sized(q_soft) + 2 * sized(log_soft) + 4))
                    np.add.at(g, kk, -w * (1 - c) * T * p)
                    np.add.at(e, kk, np.abs(w * (1 - c) * T) * p * (8 + 8 * np.abs(np.where(on, log_p, 0)) + len(tk)) * EPS * 4)
                if label >= 0:
                    q = np.exp(q_hard)
                    g += w * c * q
                    e += np.abs(w * c) * q * (sum_error + 8 * EPS * (sized(q_hard) + 2 * sized(log_hard) + 4))
                    g[label] -= w * c
                    e[label] += 4 * EPS * abs(w * c)
            put("grad", r, g, e + 4 * EPS * np.abs(g) + 2.0 ** -126 * abs(w))
    return out


def check(got, want, bound, dtype, what):
    """Every element within its bound and its result's own rounding; not-finite ones alike."""
    got = got.astype(np.float64)
    want = np.broadcast_to(want, got.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine), what
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    limit = np.broadcast_to(bound, got.shape)[fine] + half_step(dtype, np.abs(want[fine]) + np.broadcast_to(bound, got.shape)[fine])
    off = np.abs(got[fine] - want[fine])
    worst = np.argmax(off - limit) if off.size else 0
    assert off.size == 0 or np.all(off <= limit), (what, off[worst], limit[worst], want[fine][worst])
