"""As many sequences as a call takes: 2^31 - 1 of one step and one channel."""
import numpy as np
import pytest

from vkml_b200 import TensorDesc
from vkml_b200.graph import DType

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16
N, GUARD = (1 << 31) - 1, 1 << 12


class Guarded:
    """A result of N elements between elements that nothing writes."""

    def __init__(self, backend, dtype):
        self.backend, self.dtype, self.size = backend, dtype, np.dtype(dtype).itemsize
        self.storage = backend.allocate((N + 2 * GUARD) * self.size)
        self.guard = np.full(GUARD, -7, dtype)
        for at in (0, N + GUARD):
            backend.copy_from_host(self.storage, at * self.size, self.guard)

    def view(self, *dims):
        return TensorDesc.contiguous(self.storage.data + GUARD * self.size, dims, DType.of(np.dtype(self.dtype)))

    def check(self, value):
        got = np.empty(GUARD, self.dtype)
        for at in (0, N + GUARD):
            self.backend.copy_to_host(got, self.storage, at * self.size)
            assert np.array_equal(got, self.guard), at
        got = np.empty(1 << 20, self.dtype)
        for at in [0, N - len(got)] + [int(p) for p in np.random.default_rng(0).integers(0, N - len(got), 12)]:
            self.backend.copy_to_host(got, self.storage, (GUARD + at) * self.size)
            assert np.all(got == self.dtype(value)), at


def test_each_is_computed_and_nothing_beside_them(backend):
    """Inputs are one element that stands for all; x = 2, gate = 0, h = 6 in front: h = 4, and of a gradient of 8 half goes on, half to x."""
    one = {}
    for name, value, dtype in (("x", 2, F16), ("gate", 0, F16), ("dout", 8, F16), ("initial", 6, F32)):
        storage = backend.allocate(16)
        backend.copy_from_host(storage, 0, np.full(4, value, dtype))
        dims = (N, 1) if name == "initial" else (N, 1, 1)
        one[name] = (TensorDesc(storage.data, dims, (0,) * len(dims), DType.of(np.dtype(dtype))), storage)
    get = lambda name: one[name][0]  # noqa: E731
    out, states = Guarded(backend, F16), Guarded(backend, F32)
    backend.gated_recurrence(get("x"), get("gate"), out.view(N, 1, 1), initial=get("initial"), states=states.view(N, 1, 1))
    backend.synchronize()
    out.check(4)
    states.check(6)
    dinitial = Guarded(backend, F32)
    backend.gated_recurrence_backward(get("x"), get("gate"), states.view(N, 1, 1), out_grad=get("dout"), x_grad=out.view(N, 1, 1), initial_grad=dinitial.view(N, 1))
    backend.synchronize()
    out.check(4)
    dinitial.check(4)
    backend.gated_recurrence_backward(get("x"), get("gate"), states.view(N, 1, 1), out_grad=get("dout"), gate_grad=out.view(N, 1, 1))
    backend.synchronize()
    out.check(8)  # a (1 - a) (h - x) D = 1/4 4 8
