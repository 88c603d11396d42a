"""Distillation of rows whose logits lie far from zero.  A softmax does not see what is added to its whole row; the powers of two that it is computed by do:
(z - max) / T * log2 e is one multiply-add where max / T * log2 e is small, and the rounding of max / T * log2 e is given back afterwards;
where it is not small the difference comes first, in the softmax at the temperature and in the one without by turns."""
import numpy as np
import pytest

from test_distill_gpu import problem, run

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab,top", [(9, 61, 5), (9, 3001, 70), (9, 66003, 9), (311, 16501, 7)])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
def test_shifts_that_round(backend, dtype, rows, vocab, top, temperature):
    """Rows around values whose product with log2 e / T has few bits behind the point: the bound is that of rows around zero."""
    rng = np.random.default_rng(vocab)
    z, k, t = problem(rng, (rows, vocab), top, dtype)
    shifts = np.array([0.0, 40.0, -75.0, 301.0, -517.0, 1001.0, -1003.0, 1390.0, -1410.0], F32)
    z = (z.astype(F32) + np.resize(shifts, rows)[:, None]).astype(dtype)
    labels = rng.integers(0, vocab, rows)
    for hard in (0.0, 0.3, 1.0):
        run(backend, z, k, t, labels if hard else None, None, temperature, hard, 4.0, some=np.arange(len(shifts)))


# rows around these; 2839 / log2 e = 4096 is where the form changes
SHIFTS = (0.0, 1000.0, -1000.0, 1500.0, -1500.0, 2900.0, -2900.0, 3000.0, -3000.0, 5000.0, -5000.0, 10000.0, -10000.0, 12000.0, -12000.0)


def shifted(rng, rows, vocab, top, dtype):
    z, k, t = problem(rng, (rows, vocab), top, dtype)
    z = (z.astype(F32) + np.resize(np.asarray(SHIFTS, F32), rows)[:, None]).astype(dtype)
    z[len(SHIFTS)] = -10000.0  # the usual mask's value in every column
    labels = rng.integers(0, vocab, rows)
    labels[::4] = k[::4, 0]
    return z, k, t, labels


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab,top", [(17, 61, 5), (17, 3001, 70), (16, 66003, 9), (311, 16501, 7), (311, 40000, 30)])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0, 4.0])
def test_shifted_rows(backend, dtype, rows, vocab, top, temperature):
    """A block to a row, a cluster to a row, blocks that take row after row: losses with the gradient, losses, the gradient alone."""
    rng = np.random.default_rng(vocab)
    z, k, t, labels = shifted(rng, rows, vocab, top, dtype)
    some = np.arange(min(rows, len(SHIFTS) + 1))
    for hard in (0.0, 0.3, 1.0):
        run(backend, z, k, t, labels if hard else None, None, temperature, hard, 4.0, some=some)
