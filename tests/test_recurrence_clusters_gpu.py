"""Sequences that clusters of two, four and eight blocks walk along, two channels to a lane, window after window: some channels against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import Space, check
from language_steps import recurrence, recurrence_backward
from test_recurrence_gpu import F16, F32, forward, nan, problem

pytestmark = pytest.mark.gpu


def view(shape, dtype, layout):
    """dense, or `words`: rows that begin two elements behind a 16-byte boundary, which come in pieces of four bytes."""
    if layout == "dense":
        return np.full(shape, np.nan, dtype)
    return np.full(shape[:-1] + (shape[-1] + 2,), np.nan, dtype)[..., 2:]


# windows of 1024, 512, 256 and 1024 steps
@pytest.mark.parametrize("shape", [(1, 2100, 2048), (2, 1300, 2048), (4, 600, 2048), (2, 3100, 1024)])
@pytest.mark.parametrize("types", [(F16, F16), (F16, F32)])
@pytest.mark.parametrize("kind,layout,ragged", [("sigmoid", "dense", False), ("exp", "words", True), ("exp", "dense", False), ("sigmoid", "words", True)])
def test_windows_of_two_channels(backend, shape, types, kind, layout, ragged):
    rng = np.random.default_rng(shape[1])
    values = problem(rng, shape, types, kind, remember=2.0)
    x, gate, dout = (view(shape, t, layout) for t in types + (F16,))
    x[...], gate[...], initial = values
    dout[...], dfinal = rng.standard_normal(shape, dtype=F32), rng.standard_normal(initial.shape).astype(F32)
    lengths = np.array([shape[1] - 37, shape[1] // 3, shape[1], 5][: shape[0]], np.int64) if ragged else None
    for b, n in enumerate(lengths if ragged else []):
        x[b, n:], gate[b, n:], dout[b, n:] = np.nan, np.inf, np.nan
    out, final, states = forward(backend, x, gate, initial, lengths, kind, out=view(shape, F16, layout))
    again = forward(backend, x, gate, initial, lengths, kind, out=view(shape, F16, layout))
    assert all(np.array_equal(a, b) for a, b in zip((out, final, states), again))
    space = Space(backend)
    put = space.put
    dx, dgate, dinitial = view(shape, F16, layout), view(shape, types[1], layout), nan(initial.shape)
    backend.gated_recurrence_backward(put(x), put(gate), put(states), out_grad=put(dout), final_grad=put(dfinal), x_grad=put(dx), gate_grad=put(dgate), initial_grad=put(dinitial),
                                      lengths=put(lengths), kind=kind)
    got = {}
    for name, t in (("x", dx), ("gate", dgate), ("initial", dinitial)):
        got[name], rest = space.get(t)
        assert rest, name
    backend.synchronize()
    some = np.unique(np.concatenate([[0, 1, 62, 63, 64, shape[2] // 2, shape[2] - 2, shape[2] - 1], rng.integers(0, shape[2], 8)]))
    part = lambda t: np.ascontiguousarray(t[..., some])  # noqa: E731
    want = recurrence(part(x), part(gate), part(initial), lengths, kind)
    check(part(out), *want["out"], F16, "out")
    check(part(final), *want["final"], F32, "final")
    check(part(states), *want["states"], F32, "states")
    want = recurrence_backward(part(x), part(gate), part(initial), lengths, kind, part(dout), part(dfinal))
    for name, dtype in (("x", F16), ("gate", types[1]), ("initial", F32)):
        check(part(got[name]), *want[name], dtype, name)
