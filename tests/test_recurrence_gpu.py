"""Gated recurrences and their gradients against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import Space, check, placed, rows_view
from language_steps import CHUNK, gates, recurrence, recurrence_backward

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16
TYPES = [(F32, F32), (F16, F16), (F16, F32)]


def problem(rng, shape, types, kind, remember=0.0):
    """Inputs, gates of channels that remember for longer and shorter, a state in front."""
    x = rng.standard_normal(shape).astype(types[0])
    means = rng.standard_normal(shape[-1]) * 1.5 + remember
    g = rng.standard_normal(shape) + means
    gate = (g + 1.0 if kind == "sigmoid" else -np.exp(0.5 * g - 2.0)).astype(types[1])
    return x, gate, rng.standard_normal((shape[0], shape[-1])).astype(F32)


def nan(shape, dtype=F32):
    return np.full(shape, np.nan, dtype)


def forward(backend, x, gate, initial, lengths, kind, layout="dense", out=None, final=None):
    space = Space(backend)
    put = space.put
    out = rows_view(x.shape, x.dtype.type, layout) if out is None else out
    final = nan((x.shape[0], x.shape[2])) if final is None else final
    states = nan((x.shape[0], -(-x.shape[1] // CHUNK), x.shape[2]))
    backend.gated_recurrence(put(x), put(gate), put(out), initial=put(initial), final=put(final), states=put(states), lengths=put(lengths), kind=kind)
    got, rest = space.get(out)
    assert rest
    backend.synchronize()
    return got, space.get(final)[0], space.get(states)[0]


def run(backend, x, gate, initial, lengths, kind, layout, dout, dfinal):
    want = recurrence(x, gate, initial, lengths, kind)
    out, final, states = forward(backend, x, gate, initial, lengths, kind, layout)
    check(out, *want["out"], x.dtype.type, "out")
    check(final, *want["final"], F32, "final")
    check(states, *want["states"], F32, "states")
    grads = recurrence_backward(x, gate, initial, lengths, kind, dout, dfinal)
    space = Space(backend)
    put = space.put
    dx, dgate, dinitial = rows_view(x.shape, x.dtype.type, layout), rows_view(x.shape, gate.dtype.type, layout), nan(initial.shape if initial is not None else (x.shape[0], x.shape[2]))
    backend.gated_recurrence_backward(put(x), put(gate), put(states), out_grad=put(dout), final_grad=put(dfinal), x_grad=put(dx), gate_grad=put(dgate),
                                      initial_grad=put(dinitial), lengths=put(lengths), kind=kind)
    for view, name, dtype in ((dx, "x", x.dtype.type), (dgate, "gate", gate.dtype.type), (dinitial, "initial", F32)):
        got, rest = space.get(view)
        assert rest, name
        check(got, *grads[name], dtype, name)
    backend.synchronize()


SHAPES = [((1, 1, 1), "dense"), ((3, 1, 7), "dense"), ((2, 2, 64), "pitch"), ((1, 15, 8), "dense"), ((2, 16, 33), "odd"), ((2, 17, 64), "dense"), ((3, 128, 66), "dense"),
          ((3, 129, 66), "swapped"), ((2, 300, 1), "dense"), ((2, 1000, 40), "offset"), ((1, 2050, 96), "pitch"), ((5, 255, 130), "backwards"), ((2, 700, 333), "odd"),
          ((1, 4100, 34), "dense")]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("shape,layout", SHAPES)
def test_recurrence_and_gradients(backend, types, kind, shape, layout):
    rng = np.random.default_rng(shape[1] + shape[2])
    x, gate, initial = problem(rng, shape, types, kind)
    dout, dfinal = rng.standard_normal(shape).astype(types[0]), rng.standard_normal(initial.shape).astype(F32)
    run(backend, placed(x, layout), placed(gate, layout), initial, None, kind, layout, placed(dout, layout), dfinal)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("shape", [(6, 1, 5), (6, 40, 33), (7, 300, 64), (6, 2100, 40)])
def test_sequences_of_different_lengths(backend, types, kind, shape):
    """From no step to all; what lies behind an end is no number and is not read."""
    rng = np.random.default_rng(shape[1])
    x, gate, initial = problem(rng, shape, types, kind)
    dout, dfinal = rng.standard_normal(shape).astype(types[0]), rng.standard_normal(initial.shape).astype(F32)
    lengths = np.array([0, shape[1], 1, max(0, shape[1] - 1), shape[1] // 2, min(17, shape[1])] + [shape[1] // 3] * (shape[0] - 6)).astype(np.int32 if kind == "exp" else np.int64)
    for b, n in enumerate(lengths):
        x[b, n:], gate[b, n:], dout[b, n:] = np.nan, np.inf, np.nan
    run(backend, x, gate, initial, lengths, kind, "dense", dout, dfinal)


def test_lengths_outside(backend):
    rng = np.random.default_rng(0)
    x, gate, initial = problem(rng, (4, 50, 8), (F32, F32), "sigmoid")
    lengths = np.array([-1, 51, 1 << 40, 20])
    space = Space(backend)
    put = space.put
    out, final = nan(x.shape), nan(initial.shape)
    backend.gated_recurrence(put(x), put(gate), put(out), initial=put(initial), final=put(final), lengths=put(lengths))
    with pytest.raises(IndexError):
        backend.synchronize()
    want = recurrence(x, gate, initial, np.clip(lengths, 0, 50), "sigmoid")
    check(space.get(out)[0], *want["out"], F32, "out")
    check(space.get(final)[0], *want["final"], F32, "final")


@pytest.mark.parametrize("types", [(F16, F16), (F16, F32)])
@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("shape,layout", [((1, 9300, 64), "dense"), ((2, 5300, 34), "dense"), ((1, 6200, 33), "odd"), ((2, 10500, 72), "pitch")])
def test_few_channels_of_long_sequences(backend, types, kind, shape, layout):
    """Clusters that tell each other of window after window; sequences that end in an early one, for whose later blocks nothing is left."""
    rng = np.random.default_rng(shape[1])
    x, gate, initial = problem(rng, shape, types, kind)
    dout, dfinal = rng.standard_normal(shape).astype(types[0]), rng.standard_normal(initial.shape).astype(F32)
    lengths = np.array([shape[1] - 5, 1100][: shape[0]], np.int64)
    run(backend, placed(x, layout), placed(gate, layout), initial, lengths, kind, layout, placed(dout, layout), dfinal)


@pytest.mark.parametrize("shape", [(2, 1, 64), (2, 70, 64), (1, 1500, 33)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_results_over_inputs(backend, shape, dtype):
    """out on x or gate, a state that is carried on where it lies; gradients on what they are computed from."""
    rng = np.random.default_rng(shape[1])
    x, gate, initial = problem(rng, shape, (dtype, dtype), "sigmoid")
    dout, dfinal = rng.standard_normal(shape).astype(dtype), rng.standard_normal(initial.shape).astype(F32)
    out, final, states = forward(backend, x, gate, initial, None, "sigmoid")
    for on in ("x", "gate"):
        a = {"x": x.copy(), "gate": gate.copy()}
        state = initial.copy()
        got = forward(backend, a["x"], a["gate"], state, None, "sigmoid", out=a[on], final=state)
        for g, w in zip(got, (out, final, states)):
            assert np.array_equal(g, w), on

    def backward(place):
        a = {"x": x.copy(), "gate": gate.copy(), "dout": dout.copy(), "dfinal": dfinal.copy(), "dx": nan(shape, dtype), "dgate": nan(shape, dtype), "dinitial": nan(initial.shape)}
        space = Space(backend)
        put = lambda k: space.put(a[k])  # noqa: E731
        backend.gated_recurrence_backward(put("x"), put("gate"), space.put(states), out_grad=put("dout"), final_grad=put("dfinal"), x_grad=put(place[0]), gate_grad=put(place[1]),
                                          initial_grad=put(place[2]))
        return [space.get(a[k])[0] for k in place]

    apart = backward(("dx", "dgate", "dinitial"))
    for place in (("x", "gate", "dfinal"), ("gate", "x", "dinitial"), ("dout", "dgate", "dfinal"), ("dx", "dout", "dinitial")):
        for g, w in zip(backward(place), apart):
            assert np.array_equal(g, w), place


@pytest.mark.parametrize("shape", [(2, 3, 20), (2, 200, 70)])
def test_parts_that_are_absent(backend, shape):
    """Each result alone has the bits that it has beside the others; an absent state or gradient is zero."""
    rng = np.random.default_rng(1)
    x, gate, _ = problem(rng, shape, (F16, F16), "sigmoid")
    zero = np.zeros((shape[0], shape[2]), F32)
    out, final, states = forward(backend, x, gate, zero, None, "sigmoid")
    space = Space(backend)
    alone = rows_view(shape, F16, "dense")
    backend.gated_recurrence(space.put(x), space.put(gate), space.put(alone))
    assert np.array_equal(space.get(alone)[0], out)
    dout, dfinal = rng.standard_normal(shape).astype(F16), rng.standard_normal(zero.shape).astype(F32)
    names = {"x_grad": (shape, F16), "gate_grad": (shape, F16), "initial_grad": (zero.shape, F32)}

    def backward(want, dout, dfinal):
        space, views = Space(backend), {k: nan(*names[k]) for k in want}
        backend.gated_recurrence_backward(space.put(x), space.put(gate), space.put(states), out_grad=space.put(dout), final_grad=space.put(dfinal),
                                          **{k: space.put(v) for k, v in views.items()})
        return {k: space.get(v)[0] for k, v in views.items()}

    every = backward(names, dout, dfinal)
    for k in names:
        assert np.array_equal(backward([k], dout, dfinal)[k], every[k]), k
    for given, nothing in ((dict(dout=dout, dfinal=None), dict(dout=dout, dfinal=zero)), (dict(dout=None, dfinal=dfinal), dict(dout=np.zeros_like(dout), dfinal=dfinal)),
                           (dict(dout=None, dfinal=None), dict(dout=np.zeros_like(dout), dfinal=zero))):
        a, b = backward(names, **given), backward(names, **nothing)
        for k in names:
            assert np.array_equal(a[k], b[k]), k


def test_one_sequence_without_a_batch(backend):
    rng = np.random.default_rng(2)
    x, gate, initial = problem(rng, (1, 333, 48), (F16, F32), "exp")
    want = forward(backend, x, gate, initial, np.array([300]), "exp")
    space = Space(backend)
    put = space.put
    out, final, states = rows_view((333, 48), F16, "dense"), nan((48,)), nan((21, 48))
    backend.gated_recurrence(put(x[0]), put(gate[0]), put(out), initial=put(initial[0]), final=put(final), states=put(states), lengths=put(np.array(300)), kind="exp")
    for view, w in zip((out, final, states), want):
        assert np.array_equal(space.get(view)[0], w[0])


def test_rows_that_stand_for_many(backend):
    """One gate of every step, one input of every sequence, one state in front of all: views without a stride."""
    rng = np.random.default_rng(3)
    shape = (3, 150, 34)
    x, gate, initial = problem(rng, shape, (F32, F32), "sigmoid")
    x, gate, initial = np.broadcast_to(x[:1], shape), np.broadcast_to(gate[:, :1], shape), np.broadcast_to(initial[:1], (3, 34))
    own = [np.ascontiguousarray(t) for t in (x, gate, initial)]
    want = forward(backend, *own, None, "sigmoid")
    space = Space(backend)
    out, final = nan(shape), nan((3, 34))
    backend.gated_recurrence(space.put(x), space.put(gate), space.put(out), initial=space.put(initial), final=space.put(final))
    assert np.array_equal(space.get(out)[0], want[0]) and np.array_equal(space.get(final)[0], want[1])


@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_gates_that_begin_anew_or_hold(backend, kind, dtype):
    """-inf forgets everything, however large it was; +inf (sigmoid) and 0 (exp, without an input) keep the state to the last bit."""
    rng = np.random.default_rng(4)
    shape = (2, 260, 48)
    x, gate, initial = problem(rng, shape, (dtype, dtype), kind)
    initial = (initial * 1e6).astype(F32)
    x[:, :40] *= dtype(100)
    for t in (0, 7, 130, 200):
        gate[:, t, ::2] = -np.inf
    out, final, states = forward(backend, x, gate, initial, None, kind)
    for t in (0, 7, 130, 200):
        assert np.array_equal(out[:, t, ::2], x[:, t, ::2])
    value, bound = recurrence(x, gate, initial, None, kind)["out"]
    if dtype == F16:  # a state above 65520 is infinite there
        value = np.where(np.abs(value) >= 65520, np.copysign(np.inf, value), value)
    check(out, value, bound, dtype, "out")
    gate[...] = np.inf if kind == "sigmoid" else 0.0
    if kind == "exp":
        x[...] = 0
    _, final, states = forward(backend, x, gate, initial, None, kind)
    assert np.array_equal(final, initial) and np.array_equal(states, np.broadcast_to(initial[:, None], states.shape))
    # the gradient passes a gate that holds, and none that begins anew
    dfinal = rng.standard_normal(initial.shape).astype(F32)
    gate[0, 133] = -np.inf
    space = Space(backend)
    dinitial, dx = nan(initial.shape), nan(shape, dtype)
    backend.gated_recurrence_backward(space.put(x), space.put(gate), space.put(forward(backend, x, gate, initial, None, kind)[2]), final_grad=space.put(dfinal),
                                      initial_grad=space.put(dinitial), x_grad=space.put(dx), kind=kind)
    got = space.get(dinitial)[0]
    assert np.array_equal(got[1], dfinal[1]) and not got[0].any()
    assert np.array_equal(space.get(dx)[0][0, 133], dfinal[0].astype(dtype))


@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
def test_a_memory_of_many_steps(backend, kind):
    """Decays just below 1 that are alike in every step: a product of 20000 of them rounded to F32 would be 20000 * 2^-25 = 6e-4 off where each is rounded the same way.
    Here a pulse is followed until little is left of it, and so is its gradient: the bound grows with each step's own rounding alone."""
    length, rates = 20000, np.array([1e-5, 1e-4, 3e-4, 1e-3, 2e-3, 1e-2, 0.3, 0.6, 0.8, 3.0])
    gate = np.ascontiguousarray(np.broadcast_to(np.log(1 / np.expm1(rates)) if kind == "sigmoid" else -rates, (1, length, len(rates))), F32)
    x, initial = np.zeros(gate.shape, F32), np.ones((1, len(rates)), F32)
    out, final, states = forward(backend, x, gate, initial, None, kind)
    a, d, _ = (t[0, 0] for t in gates(gate, kind))
    want = np.exp(np.arange(1, length + 1)[:, None] * np.log1p(-d))
    steps = np.arange(1, length + 1)[:, None]
    # of what is left: (16 + 4 |gate|) EPS of the smaller of a and 1 - a in each step, and two roundings of the state, which go either way: 6 sqrt(steps) of them hold
    relative = steps * np.minimum(d, 1 - d) * (16 + 4 * np.abs(gate[0, 0])) * 2.0 ** -24 + (12 * np.sqrt(steps) + 8 + 4 * steps * (d > 0.4)) * 2.0 ** -24
    on = want > 1e-30
    assert np.all(np.abs(out[0] - want)[on] <= (relative * want)[on]), (np.abs(out[0] - want)[on] / (relative * want)[on]).max()
    space = Space(backend)
    dinitial = nan(initial.shape)
    backend.gated_recurrence_backward(space.put(x), space.put(gate), space.put(states), final_grad=space.put(initial), initial_grad=space.put(dinitial), kind=kind)
    got = space.get(dinitial)[0][0]
    on = want[-1] > 1e-30
    assert np.all(np.abs(got - want[-1])[on] <= (relative[-1] * want[-1])[on])


@pytest.mark.parametrize("types", TYPES)
def test_a_sequence_in_parts_and_token_by_token(backend, types):
    """What continues from a state that was left is the whole sequence, within what both may be off by."""
    rng = np.random.default_rng(5)
    x, gate, initial = problem(rng, (3, 150, 66), types, "sigmoid")
    want = recurrence(x, gate, initial, None, "sigmoid")
    for cuts in ([0, 100, 150], [0, 1, 2, 3, 19, 150], list(range(0, 40)) + [150]):
        state, parts = initial.copy(), []
        for lo, hi in zip(cuts[:-1], cuts[1:]):
            out, state, _ = forward(backend, np.ascontiguousarray(x[:, lo:hi]), np.ascontiguousarray(gate[:, lo:hi]), state, None, "sigmoid")
            parts.append(out)
        check(np.concatenate(parts, 1), *want["out"], types[0], cuts)
        check(state, *want["final"], F32, cuts)


@pytest.mark.parametrize("length", [5, 100, 3000])
def test_growing_states(backend, length):
    """Gates above 0 of the kind exp: growth within F32's range is followed, and a channel without state and input stays at zero however its gates would have it grow."""
    rng = np.random.default_rng(7)
    shape = (2, length, 40)
    x, gate = rng.standard_normal(shape).astype(F32), (rng.standard_normal(shape) * 0.3).astype(F32)
    gate[:, : min(length, 60), ::4] = 0.4
    x[0, :, 1::4], gate[0, :, 1::4] = 0, 30
    initial, dout, dfinal = np.zeros((2, 40), F32), rng.standard_normal(shape).astype(F32), rng.standard_normal((2, 40)).astype(F32)
    dout[0, :, 1::4], dfinal[0, 1::4] = 0, 0
    run(backend, x, gate, initial, None, "exp", "dense", dout, dfinal)


def test_many_short_sequences(backend):
    rng = np.random.default_rng(8)
    for length in (1, 3, 20):
        x, gate, initial = problem(rng, (70001, length, 6), (F16, F16), "sigmoid")
        out, final, states = forward(backend, x, gate, initial, None, "sigmoid")
        some = np.array([0, 1, 65534, 65535, 65536, 70000])
        want = recurrence(x[some], gate[some], initial[some], None, "sigmoid")
        check(out[some], *want["out"], F16, "out")
        check(final[some], *want["final"], F32, "final")
        space = Space(backend)
        dx, dinitial = nan(x.shape, F16), nan(initial.shape)
        backend.gated_recurrence_backward(space.put(x), space.put(gate), space.put(states), out_grad=space.put(out), x_grad=space.put(dx), initial_grad=space.put(dinitial))
        want = recurrence_backward(x[some], gate[some], initial[some], None, "sigmoid", out[some], None)
        check(space.get(dx)[0][some], *want["x"], F16, "x")
        check(space.get(dinitial)[0][some], *want["initial"], F32, "initial")


@pytest.mark.parametrize("shape", [(2, 0, 8), (0, 5, 8), (2, 5, 0)])
def test_nothing_to_do(backend, shape):
    """No step: the state passes through; no sequence or no channel: nothing."""
    x = np.zeros(shape, F32)
    initial, final = np.arange(shape[0] * shape[2], dtype=F32).reshape(shape[0], shape[2]), nan((shape[0], shape[2]))
    space = Space(backend)
    put = space.put
    backend.gated_recurrence(put(x), put(x.copy()), put(x.copy()), initial=put(initial), final=put(final))
    dinitial = nan(final.shape)
    backend.gated_recurrence_backward(put(x), put(x.copy()), put(np.zeros((shape[0], -(-shape[1] // CHUNK), shape[2]), F32)), final_grad=put(initial), initial_grad=put(dinitial))
    backend.synchronize()
    assert np.array_equal(space.get(final)[0], initial) and np.array_equal(space.get(dinitial)[0], initial)


@pytest.mark.parametrize("shape", [(2, 1, 2048), (4, 513, 130), (1, 9000, 40), (40, 600, 256)])
def test_the_same_bits_again(backend, shape):
    rng = np.random.default_rng(6)
    x, gate, initial = problem(rng, shape, (F16, F16), "sigmoid")
    first = forward(backend, x, gate, initial, None, "sigmoid")
    for _ in range(3):
        for a, b in zip(forward(backend, x, gate, initial, None, "sigmoid"), first):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("batch,length,width", [(16, 700, 2048), (3, 5001, 333), (1, 20000, 256), (300, 90, 64)])
@pytest.mark.parametrize("types", [(F16, F16), (F32, F32)])
def test_larger_ones(backend, batch, length, width, types):
    """Some channels of calls that fill the device, forward and backward."""
    rng = np.random.default_rng(length)
    shape = (batch, length, width)
    x, gate = (rng.standard_normal(shape, dtype=F32) for _ in range(2))
    x, gate, dout = x.astype(types[0]), (gate + 1).astype(types[1]), (x * gate).astype(types[0])
    initial, dfinal = (rng.standard_normal((batch, width)).astype(F32) for _ in range(2))
    out, final, states = forward(backend, x, gate, initial, None, "sigmoid")
    space = Space(backend)
    put = space.put
    dx, dgate, dinitial = nan(shape, types[0]), nan(shape, types[1]), nan(initial.shape)
    backend.gated_recurrence_backward(put(x), put(gate), put(states), out_grad=put(dout), final_grad=put(dfinal), x_grad=put(dx), gate_grad=put(dgate), initial_grad=put(dinitial))
    dx, dgate, dinitial = (space.get(t)[0] for t in (dx, dgate, dinitial))
    some = np.unique(np.concatenate([[0, 1, 31, 32, 63, width // 2, width - 2, width - 1], rng.integers(0, width, 4)]))
    some = some[some < width]
    rows = np.unique([0, batch // 2, batch - 1])
    part = lambda t: np.ascontiguousarray(t[rows][..., some])  # noqa: E731
    want = recurrence(part(x), part(gate), part(initial), None, "sigmoid")
    check(part(out), *want["out"], types[0], "out")
    check(part(final), *want["final"], F32, "final")
    check(part(states), *want["states"], F32, "states")
    want = recurrence_backward(part(x), part(gate), part(initial), None, "sigmoid", part(dout), part(dfinal))
    check(part(dx), *want["x"], types[0], "x")
    check(part(dgate), *want["gate"], types[1], "gate")
    check(part(dinitial), *want["initial"], F32, "initial")
    assert np.isfinite(out).all() and np.isfinite(dx).all() and np.isfinite(dgate).all()
