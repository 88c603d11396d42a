"""Recurrences whose decays multiply far beyond F32's range, over states and gradients that stay within it, against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import check
from language_steps import recurrence, recurrence_backward
from test_recurrence_gpu import F16, F32, forward, nan, placed, rows_view, Space

pytestmark = pytest.mark.gpu


def held(value, bound, dtype):
    """What F16 has of a value beyond its range: an infinity."""
    return (np.where(np.abs(value) >= 65520, np.copysign(np.inf, value), value) if dtype == F16 else value), bound


def compare(backend, x, gate, initial, lengths, dout, dfinal, layout="dense"):
    """Kind exp, forward and backward.  Bounds are those of every other recurrence: they are relative to what a step adds to, however large its decay."""
    x, gate, dout = (placed(t, layout) for t in (x, gate, dout))
    want = recurrence(x, gate, initial, lengths, "exp")
    out, final, states = forward(backend, x, gate, initial, lengths, "exp", layout)
    check(out, *held(*want["out"], x.dtype.type), x.dtype.type, "out")
    check(final, *want["final"], F32, "final")
    check(states, *want["states"], F32, "states")
    want = recurrence_backward(x, gate, initial, lengths, "exp", dout, dfinal)
    space = Space(backend)
    put = space.put
    dx, dgate, dinitial = rows_view(x.shape, x.dtype.type, layout), rows_view(x.shape, gate.dtype.type, layout), nan(initial.shape)
    backend.gated_recurrence_backward(put(x), put(gate), put(states), out_grad=put(dout), final_grad=put(dfinal), x_grad=put(dx), gate_grad=put(dgate),
                                      initial_grad=put(dinitial), lengths=put(lengths), kind="exp")
    for view, name, dtype in ((dinitial, "initial", F32), (dx, "x", x.dtype.type), (dgate, "gate", gate.dtype.type)):
        got, rest = space.get(view)
        assert rest, name
        check(got, *held(*want[name], dtype), dtype, name)
    backend.synchronize()


# by clusters of eight blocks, some with windows of 2048 steps; by two; by blocks without a cluster; by threads alone
SHAPES = [(1, 2000, 64), (1, 5000, 33), (5, 1000, 512), (40, 300, 256), (2, 100, 64), (3, 16, 40)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rate", [0.8, 6.0])
def test_a_small_state_that_grows(backend, shape, rate):
    """1e-30 times e^102, within a block's steps or within one thread's, and the gradient of that; then nothing changes."""
    x, gate = np.zeros(shape, F32), np.zeros(shape, F32)
    steps = min(shape[1], int(102.4 / rate))
    gate[:, :steps] = np.linspace(0.98, 1.0, shape[2]).astype(F32) * F32(rate)
    small = np.full((shape[0], shape[2]), 1e-30, F32)
    compare(backend, x, gate, small, None, np.zeros(shape, F32), small)


def waves(shape, period, swing, rng):
    """Gates whose sums rise by `swing` and fall again every `period` steps, each channel at a place of its own, and the sums."""
    t = np.arange(shape[1] + 1)[None, :, None] + rng.integers(0, period, (shape[0], 1, shape[2]))
    level = swing * np.abs(2 * (t % period) / period - 1)
    gate = np.diff(level, axis=1).astype(F32)
    return gate, level[:, :1] + np.concatenate([np.zeros((shape[0], 1, shape[2])), np.cumsum(gate.astype(np.float64), 1)], 1)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("period,swing", [(32, 150.0), (300, 150.0), (512, 120.0), (64, 40.0), (700, 6.0)])
def test_states_that_rise_and_fall(backend, shape, period, swing):
    """States from 1e-33 to 1e32 and back (or less far), gradients the other way round: inputs and gradients of a step are a part of what it has."""
    rng = np.random.default_rng(period + shape[1])
    gate, level = waves(shape, period, swing, rng)
    size = np.exp(level - swing / 2)
    noise = lambda part: (rng.standard_normal(shape) * part)  # noqa: E731
    x, initial = (size[:, 1:] * noise(0.02)).astype(F32), size[:, 0].astype(F32)
    dout, dfinal = (noise(0.02) / size[:, 1:]).astype(F32), (1 / size[:, -1]).astype(F32)
    compare(backend, x, gate, initial, None, dout, dfinal)


@pytest.mark.parametrize("types", [(F16, F16), (F16, F32)])
@pytest.mark.parametrize("shape,layout", [((1, 9300, 64), "dense"), ((1, 2500, 33), "odd"), ((1, 2100, 2048), "dense"), ((40, 300, 256), "dense"), ((3, 150, 66), "pitch")])
def test_halves_that_rise(backend, types, shape, layout):
    """A state below F16's least that rises to some hundreds and falls below it again, and its gradient, given behind the last step."""
    rng = np.random.default_rng(shape[1])
    n = min(shape[1], 600)
    gate = np.zeros(shape, types[1])
    rising = np.full(n // 3, 92.0 / (n // 3))
    gate[:, 3 : 3 + len(rising)] = rising[:, None]
    gate[:, 3 + len(rising) : 3 + 2 * len(rising)] = -rising[:, None]
    initial = (1e-37 * rng.uniform(0.5, 1.0, (shape[0], shape[2]))).astype(F32)
    compare(backend, np.zeros(shape, types[0]), gate, initial, None, np.zeros(shape, types[0]), (1 / initial * 1e-3).astype(F32), layout)


def test_sequences_that_end_while_they_grow(backend):
    rng = np.random.default_rng(3)
    shape = (5, 1500, 70)
    gate, level = waves(shape, 300, 150.0, rng)
    size = np.exp(level - 75)
    lengths = np.array([1500, 0, 130, 777, 1499])
    x, dout = (size[:, 1:] * rng.standard_normal(shape) * 0.02).astype(F32), (rng.standard_normal(shape) * 0.02 / size[:, 1:]).astype(F32)
    end = np.take_along_axis(size, lengths[:, None, None], 1)[:, 0]
    for b, n in enumerate(lengths):
        x[b, n:], gate[b, n:], dout[b, n:] = np.nan, np.inf, np.nan
    compare(backend, x, gate, size[:, 0].astype(F32), lengths, dout, (1 / end).astype(F32))


def test_a_decay_that_is_infinite(backend):
    """e^89 is beyond F32: what it meets is not finite, and nothing behind it is, even where the state was zero."""
    for length in (5, 100, 3000):
        gate, x = np.full((1, length, 8), -0.1, F32), np.zeros((1, length, 8), F32)
        gate[0, 2, ::2] = 89
        out, final, _ = forward(backend, x, gate, np.zeros((1, 8), F32), None, "exp")
        assert not np.isfinite(out[0, 2:, ::2]).any() and not np.isfinite(final[0, ::2]).any()
        assert not out[0, :2].any() and not out[0, :, 1::2].any() and not final[0, 1::2].any()
