"""Scratch of the language-model operators under capture: a graph of the caller's never holds the context's."""
import numpy as np
import pytest

import vkml_b200 as B
from test_language_together_gpu import RESULTS, capture, operators, runtime, scratch_problem, tensor
from vkml_b200 import DeviceTensor

pytestmark = pytest.mark.gpu


def close(backend, *problems):
    for s in problems:
        for t in s.values():
            t.storage.__del__()
    backend.close()


def test_a_captured_call_needs_a_workspace_however_large_the_contexts_own_is():
    """The eager calls have grown it before, so nothing would have to grow."""
    rt, backend = runtime(), B.Backend(0)
    s = scratch_problem(backend, 11)
    operators(backend, s, None)
    want = [s[k].numpy() for k in RESULTS]
    refused = []

    def calls():
        for call in (lambda: backend.embedding_backward(s["rows"], s["ids"], s["table"]),
                     lambda: backend.block_norm_backward(s["out"], s["branch"], s["stats"], out_grad=s["rows"], residual_grad=s["dh"], post_weight_grad=s["dw"])):
            with pytest.raises(ValueError, match="workspace"):
                call()
            refused.append(call)

    execution = capture(rt, backend.stream, calls)
    assert len(refused) == 2
    rt("cudaGraphExecDestroy", execution)
    operators(backend, s, None)  # the context works on
    for k, x in zip(RESULTS, want):
        assert np.array_equal(s[k].numpy(), x), k
    close(backend, s)


def test_a_replay_after_the_contexts_scratch_has_moved():
    """Captured in a workspace, replayed after larger calls and a trim: the bits of the eager calls."""
    rt, backend = runtime(), B.Backend(0)
    s = scratch_problem(backend, 12)
    operators(backend, s, None)
    want = [s[k].numpy() for k in RESULTS]
    workspace = backend.allocate(1 << 24)
    backend.synchronize()
    execution = capture(rt, backend.stream, lambda: operators(backend, s, workspace))
    n, d, v = 3000, 1024, 9000  # more scratch than any call before
    rows, ids, table = DeviceTensor.empty(backend, (n, d)), tensor(backend, np.arange(n) % v), DeviceTensor.empty(backend, (v, d))
    backend.embedding_backward(rows, ids, table)
    backend.synchronize()
    backend.trim()
    for k in RESULTS:
        backend.copy_from_host(s[k].storage, 0, np.zeros(s[k].desc.dims, np.float32))
    backend.synchronize()
    rt("cudaGraphLaunch", execution, backend.stream)
    for k, x in zip(RESULTS, want):
        assert np.array_equal(s[k].numpy(), x), k
    rt("cudaGraphExecDestroy", execution)
    for t in (rows, ids, table):
        t.storage.__del__()
    workspace.__del__()
    close(backend, s)


def test_calls_without_scratch_are_captured_without_a_workspace():
    """A lookup, a block norm, a loss, gradients that sum nothing over rows: one graph, the eager calls' bits."""
    rt, backend = runtime(), B.Backend(0)
    rng = np.random.default_rng(13)
    n, d, v = 40, 96, 50
    s = {k: tensor(backend, rng.standard_normal((n, d)).astype(np.float32)) for k in ("h", "y", "dn")}
    s.update(table=tensor(backend, rng.standard_normal((v, d)).astype(np.float32)), ids=tensor(backend, rng.integers(0, v, n)),
             k=tensor(backend, rng.integers(0, d, (n, 3))), t=tensor(backend, rng.standard_normal((n, 3)).astype(np.float32)))
    results = ("x", "out", "normed", "dlogits", "dh", "dy", "dtable")
    s.update({k: DeviceTensor.empty(backend, (n, d)) for k in results[:-1]}, dtable=DeviceTensor.empty(backend, (v, d)), stats=DeviceTensor.empty(backend, (n, 4)),
             losses=DeviceTensor.empty(backend, (n,)))

    def calls():
        backend.embedding(s["table"], s["ids"], s["x"])
        backend.block_norm(s["x"], s["y"], out=s["out"], normed=s["normed"], stats=s["stats"])
        backend.distill_loss(s["normed"], s["k"], s["t"], s["losses"], grad=s["dlogits"])
        backend.block_norm_backward(s["out"], s["y"], s["stats"], normed_grad=s["dlogits"], residual_grad=s["dh"], branch_grad=s["dy"])
        backend.embedding_backward(s["dh"], s["ids"], s["dtable"])  # few tokens: rows owned by blocks

    calls()
    want = {k: s[k].numpy() for k in results}
    backend.synchronize()
    execution = capture(rt, backend.stream, calls)
    for k in results:
        backend.copy_from_host(s[k].storage, 0, np.zeros(s[k].desc.dims, np.float32))
    backend.synchronize()
    rt("cudaGraphLaunch", execution, backend.stream)
    for k in results:
        assert np.array_equal(s[k].numpy(), want[k]), k
    rt("cudaGraphExecDestroy", execution)
    close(backend, s)


def test_workspaces_that_are_too_small_or_not_aligned(backend):
    """Refused before anything is queued: the results keep their bytes."""
    s = scratch_problem(backend, 14)
    before = {k: s[k].numpy() for k in RESULTS}
    need = backend.embedding_backward_workspace(s["rows"], s["ids"], s["table"])
    workspace = backend.allocate(max(need, 1 << 24))

    class At:
        def __init__(self, offset, nbytes):
            self.data, self.nbytes = workspace.data + offset, nbytes

    for bad in (At(0, 255), At(128, workspace.nbytes - 128), At(8, workspace.nbytes - 8), At(256, 0)):
        with pytest.raises(ValueError, match="workspace"):
            backend.embedding_backward(s["rows"], s["ids"], s["table"], workspace=bad)
        with pytest.raises(ValueError, match="workspace"):
            backend.block_norm_backward(s["out"], s["branch"], s["stats"], out_grad=s["rows"], residual_grad=s["dh"], post_weight_grad=s["dw"], workspace=bad)
    backend.synchronize()
    for k, x in before.items():
        assert np.array_equal(s[k].numpy(), x, equal_nan=True), k
    operators(backend, s, At(256, workspace.nbytes - 256))
    backend.embedding_backward(s["rows"], s["ids"], s["table"], workspace=At(256, need))  # exactly enough
    got = s["table"].numpy()
    backend.embedding_backward(s["rows"], s["ids"], s["table"])
    assert np.array_equal(s["table"].numpy(), got)
