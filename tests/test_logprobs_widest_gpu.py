"""Rows of as many logits as a call takes: 2^31 - 1."""
import numpy as np
import pytest

from vkml_b200 import DeviceTensor, TensorDesc
from vkml_b200.graph import DType

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16
V = (1 << 31) - 1
PIECE = 1 << 25


def row(backend, dtype, shift):
    """V logits of -3 but for three, 2^31 elements behind ones that are no numbers: where a column counted in 31 bits would be found."""
    size = np.dtype(dtype).itemsize
    front = (1 << 31) + 64 + shift
    storage = backend.allocate((front + V) * size)
    backend.copy_from_host(storage, 0, np.full(PIECE, np.nan, dtype))
    piece = np.full(PIECE, -3, dtype)
    for at in range(0, V, PIECE):
        backend.copy_from_host(storage, (front + at) * size, piece[: min(PIECE, V - at)])
    for column, value in ((0, 0), (V - 1, -1), (V - 5, -2)):
        backend.copy_from_host(storage, (front + column) * size, np.array([value], dtype))
    return storage, storage.data + front * size


@pytest.mark.parametrize("dtype,shift", [(F16, 0), (F16, 3), (F32, 1)])
def test_rows_of_two_billion(backend, dtype, shift):
    """One row by a cluster, with entries, and more rows than SMs, which are the same one; and one row's gradient.

    A thread of a row has V / 4096 elements (a cluster) or V / 256 (many rows): a batch of 16 or 32 of them and one addition each, so that the sum is off by V / 4096 / 16 or V / 256 / 16
    half steps at most, and its logarithm by as much."""
    size = np.dtype(dtype).itemsize
    storage, data = row(backend, dtype, shift)
    z = lambda rows: TensorDesc(data, (rows, V), (0, size), DType.of(np.dtype(dtype)))  # noqa: E731
    total = (V - 3) * np.exp(-3.0) + 1 + np.exp(-1.0) + np.exp(-2.0)
    log = np.log(total)
    entropy = log - ((V - 3) * np.exp(-3.0) * -3 - np.exp(-1.0) - 2 * np.exp(-2.0)) / total
    new = lambda dims, t=DType.F32: DeviceTensor.empty(backend, dims, t)  # noqa: E731

    def tokens(rows):
        return DeviceTensor.from_host(backend, np.resize(np.array([V - 1, V - 5, 7, 0]), rows))

    for rows, top, threads in ((1, 5, 4096), (160, 1, 256)):
        off = V / threads / 16 * 2.0 ** -24 * 4 + 1e-5
        lp, h, stats, ids, tops = new((rows,)), new((rows,)), new((rows, 4)), new((rows, top), DType.I64), new((rows, top))
        backend.token_logprobs(z(rows), tokens(rows), lp, entropies=h, stats=stats, top_ids=ids, top_logprobs=tops)
        backend.synchronize()
        assert np.abs(lp.numpy() - (np.resize([-1.0, -2.0, -3.0, 0.0], rows) - log)).max() <= off
        assert np.abs(h.numpy() - entropy).max() <= off
        assert np.array_equal(ids.numpy(), np.broadcast_to([0, V - 1, V - 5, 1, 2][:top], (rows, top)))
        assert np.abs(tops.numpy() - (np.array([0.0, -1.0, -2.0, -3.0, -3.0][:top]) - log)).max() <= off
        assert np.array_equal(stats.numpy()[:, 0], np.zeros(rows))
    stats = DeviceTensor.from_host(backend, np.array([[0, log, entropy, 0]], F32))
    grad = backend.allocate((V + 8) * size)
    backend.copy_from_host(grad, V * size, np.full(8, 9, dtype))
    backend.token_logprobs_backward(z(1), tokens(1), stats, TensorDesc(grad.data, (1, V), (V * size, size), DType.of(np.dtype(dtype))),
                                    logprobs_grad=DeviceTensor.from_host(backend, np.ones(1, F32)), grad_scale=1024.0)
    got = np.empty(16, dtype)
    backend.copy_to_host(got, grad, (V - 8) * size)
    want = -np.exp(np.array([-3, -3, -3, -2, -3, -3, -3, -1.0]) - log) * 1024
    want[7] += 1024
    assert np.all(got[8:] == 9) and np.abs(got[:8] - want).max() <= 1024 * 2.0 ** (-11 if dtype == F16 else -22)
    assert np.all(np.abs(got[:7] - want[:7]) <= np.abs(want[:7]) * 2.0 ** (-10 if dtype == F16 else -18) + (2.0 ** -25 if dtype == F16 else 0))
