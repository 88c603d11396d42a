"""The language-model operators on tensors without elements, as an allocator hands them out: without storage."""
import numpy as np
import pytest

from vkml_b200 import DeviceTensor
from vkml_b200.graph import DType

pytestmark = pytest.mark.gpu


def test_no_rows_without_storage(backend):
    """Nothing to do but the zeros of sums over no rows."""
    new = lambda *dims, dtype=DType.F32: DeviceTensor.empty(backend, dims, dtype)  # noqa: E731
    rows, half, stats, ids = new(0, 24), new(0, 24, dtype=DType.F16), new(0, 4), new(0, dtype=DType.I64)
    assert rows.desc.data == 0 and ids.desc.data == 0
    vector = lambda x: DeviceTensor.from_host(backend, np.full(24, x, np.float32))  # noqa: E731
    w, table = vector(1.0), DeviceTensor.from_host(backend, np.full((5, 24), np.nan, np.float32))
    grads = {k: vector(np.nan) for k in ("post_weight_grad", "post_bias_grad", "gate_grad", "pre_weight_grad", "pre_bias_grad")}
    backend.embedding(table, ids, rows)
    backend.block_norm(rows, half, out=rows, normed=half, stats=stats, post_weight=w, post_bias=w, gate=w, pre_weight=w, pre_bias=w)
    backend.block_norm_backward(rows, half, stats, out_grad=rows, normed_grad=half, residual_grad=rows, branch_grad=half, post_weight=w, post_bias=w, gate=w, pre_weight=w, **grads)
    for k, g in grads.items():
        assert not g.numpy().any(), k
    k, t, logits = new(0, 3, dtype=DType.I32), new(0, 3), new(0, 9)
    backend.distill_loss(logits, k, t, new(0), labels=ids, stats=stats, grad=new(0, 9), losses_grad=new(0), hard_weight=0.5)
    backend.distill_loss_backward(logits, k, t, stats, new(0, 9), labels=ids, losses_grad=new(0), hard_weight=0.5)
    backend.embedding_backward(rows, ids, table, accumulate=True)
    assert np.isnan(table.numpy()).all()
    backend.embedding_backward(rows, ids, table)
    assert not table.numpy().any()
    empty = new(4, 0)
    backend.embedding(new(5, 0), DeviceTensor.from_host(backend, np.zeros(4, np.int64)), empty)
    backend.block_norm(empty, empty, out=empty, normed=empty)
    backend.synchronize()
