"""Norms in front of and behind a block, gate, residual scale, and their gradients, against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import EPS, Space, block_norm, block_norm_backward, check, column_sum, placed, rows_view

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16
SIDES = [(F32, F32), (F16, F16), (F32, F16)]
WEIGHTS = ("post_weight", "post_bias", "pre_weight", "pre_bias")
SHAPES = [((1, 1), "dense"), ((40,), "dense"), ((4, 1, 512), "dense"), ((3, 5, 33), "odd"), ((2, 7, 256), "pitch"), ((6, 3, 264), "swapped"), ((37, 1000), "dense"),
          ((5, 1024), "offset"), ((3, 2, 2048), "backwards"), ((3, 2056), "dense"), ((2, 3, 4096), "pitch"), ((7, 4104), "dense"), ((2, 5001), "odd"),
          ((3, 8192), "dense"), ((2, 2, 16384), "dense"), ((1, 16383), "dense")]


def parameters(rng, width, dtype, rows, gates, bias):
    p = {n: (rng.standard_normal(width) * 0.3 + (1.0 if n.endswith("weight") else 0.0)).astype(dtype) for n in WEIGHTS}
    if not bias:
        p["post_bias"] = p["pre_bias"] = None
    p["gate"] = None if gates == 0 else (rng.standard_normal((gates, width)) * 0.5 + 0.5).astype(dtype)
    return p


def of_rows(p, shape):
    """The gate in every row."""
    q = dict(p)
    if p["gate"] is not None:
        rows = int(np.prod(shape[:-1]))
        q["gate"] = np.repeat(p["gate"].reshape(-1, shape[-1]), rows // len(p["gate"].reshape(-1, shape[-1])), 0).reshape(shape)
    return q


@pytest.mark.parametrize("th,ty", SIDES)
@pytest.mark.parametrize("shape,layout", SHAPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_forward_and_backward(backend, th, ty, shape, layout, kind):
    rng = np.random.default_rng(shape[-1] + 3 * len(shape))
    layer, width, rows = kind == "layer", shape[-1], int(np.prod(shape[:-1]))
    wt = ty if layout in ("dense", "odd") else F32
    gates = {"dense": min(1, len(shape) - 1), "odd": shape[0], "pitch": rows, "swapped": shape[0], "offset": 0, "backwards": shape[0]}[layout]
    p = parameters(rng, width, wt, rows, gates, layer)
    h = placed((rng.standard_normal(shape) * 2 + 0.5).astype(th), layout)
    y = placed((rng.standard_normal(shape) + 0.25).astype(ty), layout)
    out, normed = rows_view(shape, th, layout), rows_view(shape, ty, layout)
    stats = np.full((rows, 4), np.nan, F32)
    space = Space(backend)
    put = space.put
    backend.block_norm(put(h), put(y), out=put(out), normed=put(normed), stats=put(stats), residual_scale=0.9, branch_scale=0.6, kind=kind, eps=1e-3,
                       **{k: put(v) for k, v in p.items()})
    want = block_norm(h, y, of_rows(p, shape), 0.9, 0.6, layer, 1e-3, True)
    got_out, rest = space.get(out)
    assert rest
    check(got_out, *want["out"], th, "out")
    got, rest = space.get(normed)
    assert rest
    check(got, *want["normed"], ty, "normed")
    got_stats = space.get(stats)[0]
    # means by the sums' bound; 1 / sqrt by half of it and two roundings, which is less than the sums'
    size = np.concatenate([np.abs(y.astype(np.float64)).mean(-1).reshape(-1, 1), want["stats"][..., 1:2].reshape(-1, 1),
                           np.abs(want["out"][0]).mean(-1).reshape(-1, 1), want["stats"][..., 3:4].reshape(-1, 1)], 1)
    assert np.all(np.abs(got_stats - want["stats"].reshape(-1, 4)) <= 4 * 64 * EPS * size)

    # backward, from what forward left
    stored = placed(got_out, layout)
    dout, dn = (placed(rng.standard_normal(shape).astype(t), layout) for t in (th, ty))
    grads = {"residual": rows_view(shape, th, layout), "branch": rows_view(shape, ty, layout)}
    grads.update({k: None if v is None else np.full(v.shape, np.nan, F32 if layout != "odd" else wt) for k, v in p.items()})
    space = Space(backend)
    put = space.put
    options = {k: put(p[k]) for k in ("post_weight", "post_bias", "gate", "pre_weight")}
    options.update({k + "_grad": put(v) for k, v in grads.items()})
    call = dict(out_grad=put(dout), normed_grad=put(dn), residual_scale=0.9, branch_scale=0.6, kind=kind, **options)
    args = put(stored), put(y), put(got_stats)
    backend.block_norm_backward(*args, **call)
    want = block_norm_backward(stored, y, got_stats, dout, dn, of_rows(p, shape), 0.9, 0.6, layer, True, shape)
    axes = tuple(range(len(shape) - 1))
    first = {}
    for name, buffer in grads.items():
        if buffer is None:
            continue
        got, rest = space.get(buffer)
        first[name] = got
        assert rest, name
        if name in ("residual", "branch"):
            value, error = want[name]
        elif name == "gate":
            per = tuple(x.reshape(len(buffer), -1, width) for x in want[name])
            value, error = column_sum(per, (1,))
        else:
            value, error = column_sum(want[name], axes)
        check(got, value, error, buffer.dtype.type, name)
    # the same bits again, in a workspace of the caller's
    ws = backend.allocate(max(1, backend.block_norm_backward_workspace(*args, **call)))
    backend.block_norm_backward(*args, workspace=ws, **call)
    for name, got in first.items():
        assert np.array_equal(space.get(grads[name])[0], got), name


@pytest.mark.parametrize("rows,gates,width", [(1000, 1, 96), (1500, 5, 200), (2222, 1111, 48), (900, 900, 512), (3001, 1, 1024), (640, 4, 4096), (600, 300, 264)])
def test_long_sums(backend, rows, gates, width):
    """Many rows, and gates whose rows are divided among blocks or not."""
    rng = np.random.default_rng(rows)
    p = parameters(rng, width, F32, rows, gates, True)
    out, y, dout, dn = (rng.standard_normal((rows, width)).astype(F32) for _ in range(4))
    stats = np.abs(rng.standard_normal((rows, 4))).astype(F32) + F32(0.5)
    grads = {k: np.full(v.shape, np.nan, F32) for k, v in p.items()}
    space = Space(backend)
    put = space.put
    backend.block_norm_backward(put(out), put(y), put(stats), out_grad=put(dout), normed_grad=put(dn), kind="layer",
                                **{k: put(p[k]) for k in ("post_weight", "post_bias", "gate", "pre_weight")}, **{k + "_grad": put(v) for k, v in grads.items()})
    want = block_norm_backward(out, y, stats, dout, dn, of_rows(p, (rows, width)), 1.0, 1.0, True, True, (rows, width))
    for name, buffer in grads.items():
        value, error = column_sum(tuple(x.reshape(gates, -1, width) for x in want[name]), (1,)) if name == "gate" else column_sum(want[name], (0,))
        check(space.get(buffer)[0], value, error, F32, name)


@pytest.mark.parametrize("ty", [F32, F16])
def test_parts_alone(backend, ty):
    """A norm in front alone, a branch without a norm, a branch without a residual, one result without the other."""
    rng = np.random.default_rng(3)
    shape = (5, 9, 200)
    h, y = (rng.standard_normal(shape).astype(ty) for _ in range(2))
    p = parameters(rng, 200, ty, 45, 1, False)
    for case in ("front", "plain branch", "no residual", "sum alone", "norm alone"):
        q = dict.fromkeys(p)
        args = [h, y]
        out, normed = np.full(shape, np.nan, ty), np.full(shape, np.nan, ty)
        post = True
        if case == "front":
            args, out = [h, None], None
            q["pre_weight"] = p["pre_weight"]
        elif case == "plain branch":
            post = False
            q["gate"] = p["gate"]
        elif case == "no residual":
            args = [None, y]
            q["post_weight"] = p["post_weight"]
        elif case == "sum alone":
            normed = None
        else:
            out = None
        space = Space(backend)
        put = space.put
        backend.block_norm(put(args[0]), put(args[1]), out=put(out), normed=put(normed), post_norm=post, residual_scale=0.5, branch_scale=2.0,
                           **{k: put(v) for k, v in q.items()})
        want = block_norm(args[0], args[1], of_rows(q, shape), 0.5, 2.0, False, 1e-5, post and args[1] is not None)
        if out is not None:
            check(space.get(out)[0], *want["out"], ty, case)
        if normed is not None:
            check(space.get(normed)[0], *want["normed"], ty, case)
        # its gradients
        o = want["out"][0].astype(ty)
        stats = want["stats"].reshape(45, 4).astype(F32)
        dout, dn = (rng.standard_normal(shape).astype(ty) for _ in range(2))
        dout, dn = (None if out is None else dout), (None if normed is None else dn)
        grads = {"residual": args[0], "branch": args[1], "gate": q["gate"], "post_weight": q["post_weight"], "pre_weight": q["pre_weight"]}
        grads = {k: np.full(v.shape, np.nan, ty) for k, v in grads.items() if v is not None and not (k == "pre_weight" and dn is None)}
        space = Space(backend)
        put = space.put
        backend.block_norm_backward(put(o), put(args[1]), put(stats), out_grad=put(dout), normed_grad=put(dn), post_norm=post, residual_scale=0.5, branch_scale=2.0,
                                    post_weight=put(q["post_weight"]), gate=put(q["gate"]), pre_weight=put(q["pre_weight"]) if dn is not None else None,
                                    **{k + "_grad": put(v) for k, v in grads.items()})
        want = block_norm_backward(o, args[1], stats, dout, dn, of_rows(q, shape), 0.5, 2.0, False, post, shape)
        for name, buffer in grads.items():
            value, error = want[name] if name in ("residual", "branch") else column_sum(want[name], (0, 1))
            check(space.get(buffer)[0].reshape(value.shape), value, error, ty, (case, name))


def test_results_on_their_inputs(backend):
    """The sum written over the residual, the gradients over the gradients: the bits are those of separate buffers."""
    rng = np.random.default_rng(4)
    for shape in ((6, 40), (3, 5, 1000), (4, 6000)):
        rows = int(np.prod(shape[:-1]))
        h, y, dout, dn = (rng.standard_normal(shape).astype(F16) for _ in range(4))
        w = rng.standard_normal(shape[-1]).astype(F16)
        results = []
        for place in (False, True):
            space = Space(backend)
            put = space.put
            h2, y2, dout2, dn2 = h.copy(), y.copy(), dout.copy(), dn.copy()
            out, normed = (h2, y2) if place else (np.empty_like(h), np.empty_like(y))
            stats = np.empty((rows, 4), F32)
            backend.block_norm(put(h2), put(y2), out=put(out), normed=put(normed), stats=put(stats), pre_weight=put(w), post_weight=put(w), kind="layer")
            o = space.get(out)[0]
            n = space.get(normed)[0]
            s = space.get(stats)[0]
            space = Space(backend)
            put = space.put
            dh, dy = (dout2, dn2) if place else (np.empty_like(h), np.empty_like(y))
            backend.block_norm_backward(put(o), put(y), put(s), out_grad=put(dout2), normed_grad=put(dn2), residual_grad=put(dh), branch_grad=put(dy),
                                        pre_weight=put(w), post_weight=put(w), kind="layer")
            results.append((o, n, s, space.get(dh)[0], space.get(dy)[0]))
        for a, b in zip(*results):
            assert np.array_equal(a, b)


def test_columns_of_one_buffer(backend):
    """Tensors side by side in one buffer share addresses' range but no element."""
    rng = np.random.default_rng(5)
    wide = rng.standard_normal((11, 4 * 64)).astype(F32)
    h, y, out, normed = (wide[:, i * 64:(i + 1) * 64] for i in range(4))
    want = block_norm(h, y, {}, 1.0, 1.0, False, 1e-5, True)
    space = Space(backend)
    put = space.put
    backend.block_norm(put(h), put(y), out=put(out), normed=put(normed))
    storage, root = space.buffers[id(wide)]
    now = np.empty_like(root)
    backend.copy_to_host(now, storage, 0)
    assert np.array_equal(now[:, :128], wide[:, :128])
    check(now[:, 128:192], *want["out"], F32, "out")
    check(now[:, 192:], *want["normed"], F32, "normed")


def test_no_rows(backend):
    """Sums over no rows are zeros; nothing else is written."""
    w = np.ones(24, F32)
    empty, stats, grad = np.empty((0, 24), F32), np.empty((0, 4), F32), np.full(24, np.nan, F32)
    space = Space(backend)
    put = space.put
    backend.block_norm(put(empty), put(empty.copy()), out=put(np.empty((0, 24), F32)), normed=put(np.empty((0, 24), F32)), pre_weight=put(w))
    backend.block_norm_backward(put(empty), put(empty), put(stats), out_grad=put(empty), normed_grad=put(empty), pre_weight=put(w), pre_weight_grad=put(grad))
    assert not space.get(grad)[0].any()


def test_rows_of_zeros_infinities_and_nan(backend):
    """What is in one row stays there; zeros have a finite norm."""
    rng = np.random.default_rng(6)
    h, y = (rng.standard_normal((6, 520)).astype(F32) for _ in range(2))
    h[1], y[1], y[2], h[3, 7], y[4, 5] = 0, 0, 0, np.inf, np.nan
    out, normed, stats = np.empty_like(h), np.empty_like(h), np.empty((6, 4), F32)
    space = Space(backend)
    put = space.put
    backend.block_norm(put(h), put(y), out=put(out), normed=put(normed), stats=put(stats), kind="layer")
    got = space.get(normed)[0]
    want = block_norm(h[[0, 1, 2, 5]], y[[0, 1, 2, 5]], {}, 1.0, 1.0, True, 1e-5, True)
    check(got[[0, 1, 2, 5]], *want["normed"], F32, "normed")
    assert not got[1].any() and np.isnan(got[3]).all() and np.isnan(got[4]).all()


def test_gradients_against_differences(backend):
    """Central differences of sum(out * a + normed * b) in F32: the step 2^-5 leaves a term of the third order, below 2^-10 * 40 here, and roundings of the
    sums over the step, 2^-24 * 600 / 2^-4: a limit of 0.05 holds both with values of order 1."""
    rng = np.random.default_rng(7)
    shape, width = (3, 40), 40
    v = {"residual": rng.standard_normal(shape), "branch": rng.standard_normal(shape), "post_weight": rng.standard_normal(width), "gate": rng.standard_normal(width),
         "pre_weight": rng.standard_normal(width), "post_bias": rng.standard_normal(width), "pre_bias": rng.standard_normal(width)}
    v = {k: x.astype(F32) for k, x in v.items()}
    a, b = (rng.standard_normal(shape).astype(F32) for _ in range(2))

    def forward(v):
        space = Space(backend)
        put = space.put
        out, normed, stats = np.empty(shape, F32), np.empty(shape, F32), np.empty((3, 4), F32)
        backend.block_norm(put(v["residual"]), put(v["branch"]), out=put(out), normed=put(normed), stats=put(stats), kind="layer", eps=0.1,
                           **{k: put(v[k]) for k in WEIGHTS + ("gate",)})
        return [space.get(x)[0] for x in (out, normed, stats)]

    out, normed, stats = forward(v)
    grads = {k: np.empty_like(x) for k, x in v.items()}
    space = Space(backend)
    put = space.put
    backend.block_norm_backward(put(out), put(v["branch"]), put(stats), out_grad=put(a), normed_grad=put(b), kind="layer",
                                **{k: put(v[k]) for k in ("post_weight", "post_bias", "gate", "pre_weight")}, **{k + "_grad": put(x) for k, x in grads.items()})
    for name, buffer in grads.items():
        got = space.get(buffer)[0].reshape(-1)
        for i in (0, len(got) // 2, len(got) - 1):
            value = []
            for step in (2.0 ** -5, -2.0 ** -5):
                moved = {k: x.copy() for k, x in v.items()}
                moved[name].reshape(-1)[i] += F32(step)
                o, n, _ = forward(moved)
                value.append((o.astype(np.float64) * a + n.astype(np.float64) * b).sum())
            assert abs((value[0] - value[1]) / 2.0 ** -4 - got[i]) <= 0.05 * (1 + abs(got[i])), name
