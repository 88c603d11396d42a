"""What the language-model operators refuse, told without a device: shapes, types, layouts, overlaps, options."""
import ctypes as C

import pytest

from vkml_b200 import DType, TensorDesc, _abi, graph

F32, F16, I32, I64, BOOL = DType.F32, DType.F16, DType.I32, DType.I64, DType.BOOL
EMBEDDING, EMBEDDING_BACKWARD, NORM, NORM_BACKWARD, DISTILL, DISTILL_BACKWARD = range(6)
OK, SHAPE, DTYPE, INDEX, NOT_IMPLEMENTED, INVALID = 0, 1, 2, 4, 5, 8


def answer(which, args):
    why = C.create_string_buffer(256)
    status = _abi.load().b200_check_operator(which, args, why, 256)
    assert (status == OK) == (why.value == b""), why.value
    return status


class At:
    """Addresses far apart, one for each tensor."""

    def __init__(self):
        self.next = 1 << 30

    def __call__(self, dims, dtype=F32, strides=None, offset=0):
        self.next += 1 << 30
        t = TensorDesc.contiguous(self.next + offset, dims, dtype)
        return t if strides is None else TensorDesc(t.data, t.dims, tuple(strides), dtype)


def test_structs_are_packed_as_the_header_lays_them_out():
    at = At()
    names = ("residual", "branch", "out", "normed", "stats", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate")
    tensors = [at((2, 8)) for _ in names]
    s = _abi.BlockNormArgs.from_buffer_copy(graph.block_norm_args(tensors, 1.5, 2.5, 0.25, 1, 1))
    assert [getattr(s, n).data for n in names] == [t.data for t in tensors]
    assert (s.residual_scale, s.branch_scale, s.eps, s.kind, s.flags) == (1.5, 2.5, 0.25, 1, 1)
    s = _abi.EmbeddingArgs.from_buffer_copy(graph.embedding_args(tensors[0], tensors[1], tensors[2], 3.0, 1, -7, 256, 99))
    assert (s.rows.data, s.scale, s.flags, s.padding_id, s.workspace, s.workspace_bytes) == (tensors[2].data, 3.0, 1, -7, 256, 99)
    s = _abi.DistillArgs.from_buffer_copy(graph.distill_args([None] * 7 + tensors[:1], 2.0, 0.5, 8.0))
    assert (s.logits.data, s.grad.data, s.temperature, s.hard_weight, s.grad_scale) == (None, tensors[0].data, 2.0, 0.5, 8.0)


def test_embedding():
    at = At()
    table, ids, rows = at((10, 8)), at((3, 4), I64), at((3, 4, 8), F16)

    def says(t=table, i=ids, r=rows, which=EMBEDDING, **k):
        return answer(which, graph.embedding_args(t, i, r, 1.0, **k))

    for which in (EMBEDDING, EMBEDDING_BACKWARD):
        assert says(which=which) == OK
        assert says(t=at((10, 7)), which=which) == SHAPE
        assert says(t=at((10,)), which=which) == SHAPE
        assert says(r=at((3, 5, 8)), which=which) == SHAPE
        assert says(r=at((12, 8)), which=which) == SHAPE
        assert says(i=at((1, 3, 4), I64), r=at((1, 3, 4, 8)), which=which) == SHAPE
        assert says(t=at((10, 8), I32), which=which) == DTYPE
        assert says(r=at((3, 4, 8), BOOL), which=which) == DTYPE
        assert says(i=at((3, 4), F32), which=which) == DTYPE
        assert says(t=at((10, 8), F32, (64, 8)), which=which) == NOT_IMPLEMENTED  # a column between its neighbours
        assert says(t=at((10, 8), F32, (33, 4)), which=which) == NOT_IMPLEMENTED  # no whole elements apart
        assert says(t=at((10, 8), F32, offset=2), which=which) == INVALID         # an odd address
        assert says(t=at((0, 8)), which=which) == INDEX
        assert says(t=TensorDesc(0, (10, 8), (32, 4), F32), which=which) == INVALID
        assert says(t=at((1 << 31, 8)), which=which) == SHAPE
        assert says(flags=2, which=which) == INVALID
    assert says(flags=graph.ACCUMULATE) == INVALID  # the lookup writes its rows
    assert says(flags=graph.ACCUMULATE, which=EMBEDDING_BACKWARD) == OK
    assert says(r=at((3, 4, 8), F32, (0, 32, 4))) == INVALID                                # results on one another
    assert says(r=at((3, 4, 8), F32, (0, 32, 4)), which=EMBEDDING_BACKWARD) == OK           # gradients that stand for many
    assert says(r=at((3, 4, 8), F32, (64, 32, 4))) == INVALID
    assert says(r=TensorDesc(table.data + 64, (3, 4, 8), (128, 32, 4), F32)) == INVALID     # on the table
    assert says(i=TensorDesc(table.data + 64, (3, 4), (32, 8), I64), which=EMBEDDING_BACKWARD) == INVALID
    assert says(which=EMBEDDING_BACKWARD, workspace=table.data, workspace_bytes=1 << 20) == INVALID
    assert says(i=TensorDesc(ids.data, (0, 4), (32, 8), I64), r=at((0, 4, 8))) == OK
    assert answer(9, graph.embedding_args(table, ids, rows, 1.0)) == INVALID


def norm_args(at, **replaced):
    t = {"residual": at((2, 3, 8)), "branch": at((2, 3, 8), F16), "out": at((2, 3, 8)), "normed": at((2, 3, 8), F16), "stats": at((6, 4)),
         "post_weight": at((8,)), "post_bias": at((8,)), "pre_weight": at((8,)), "pre_bias": at((8,)), "gate": at((2, 8))}
    options = {"kind": 0, "flags": 1}
    for k, v in replaced.items():
        (options if k in options else t)[k] = v
    return graph.block_norm_args(list(t.values()), 1.0, 1.0, 1e-5, options["kind"], options["flags"])


def test_block_norm():
    at = At()

    def says(**k):
        return answer(NORM, norm_args(at, **k))

    assert says() == OK
    assert says(kind=2) == INVALID and says(flags=3) == INVALID
    assert says(branch=at((2, 3, 9), F16)) == SHAPE
    assert says(out=at((6, 8))) == SHAPE
    assert says(out=at((2, 3, 8), F16)) == DTYPE        # the residual's type
    assert says(normed=at((2, 3, 8))) == DTYPE
    assert says(residual=at((2, 3, 8), F16), out=at((2, 3, 8), F16), branch=at((2, 3, 8)), normed=at((2, 3, 8))) == DTYPE
    assert says(pre_weight=at((8,), F16)) == DTYPE      # weights of two types
    assert says(post_weight=at((7,))) == SHAPE and says(post_weight=at((1, 8))) == SHAPE
    assert says(post_weight=at((8,), F32, (8,))) == NOT_IMPLEMENTED
    assert says(gate=at((4, 8))) == SHAPE and says(gate=at((0, 8))) == SHAPE and says(gate=at((8,))) == OK and says(gate=at((6, 8))) == OK
    assert says(stats=at((6, 3))) == SHAPE and says(stats=at((5, 4))) == SHAPE and says(stats=at((6, 4), F16)) == DTYPE and says(stats=at((6, 4), offset=8)) == SHAPE
    assert says(flags=0) == INVALID                     # weights of a norm that is not applied
    assert says(flags=0, post_weight=None, post_bias=None) == OK
    assert says(normed=None) == INVALID and says(normed=None, pre_weight=None, pre_bias=None) == OK
    assert says(branch=None) == INVALID                 # a gate of nothing
    assert says(branch=None, gate=None, flags=0, post_weight=None, post_bias=None) == OK
    assert says(residual=None) == OK
    assert says(residual=None, branch=None, gate=None, flags=0, post_weight=None, post_bias=None) == INVALID
    assert says(out=None, normed=None, pre_weight=None, pre_bias=None) == INVALID
    wide = {k: at((2, 16392), F16 if k in ("branch", "normed") else F32) for k in ("residual", "branch", "out", "normed")}
    assert says(**wide, stats=None, **dict.fromkeys(("post_weight", "post_bias", "pre_weight", "pre_bias", "gate"))) == NOT_IMPLEMENTED
    assert says(residual=at((2, 3, 8), F32, (0, 0, 4))) == OK                # a row that stands for many
    assert says(out=at((2, 3, 8), F32, (0, 32, 4))) == INVALID
    assert says(out=at((2, 3, 8), F32, (96, 16, 4))) == INVALID
    h = at((2, 3, 8))
    assert says(residual=h, out=h) == OK
    assert says(residual=h, out=TensorDesc(h.data + 32, h.dims, h.strides, F32)) == INVALID
    w = at((2, 3, 32))
    left, right = (TensorDesc(w.data + 32 * i, (2, 3, 8), w.strides, F32) for i in range(2))
    assert says(residual=left, out=right) == OK          # side by side in one buffer
    assert says(residual=left, out=TensorDesc(w.data + 16, (2, 3, 8), w.strides, F32)) == INVALID
    assert says(post_weight=TensorDesc(h.data, (8,), (4,), F32), residual=h, out=h) == INVALID


def grad_args(at, **replaced):
    t = {"out": at((2, 3, 8)), "branch": at((2, 3, 8), F16), "stats": at((6, 4)), "out_grad": at((2, 3, 8)), "normed_grad": at((2, 3, 8), F16),
         "post_weight": at((8,)), "post_bias": at((8,)), "gate": at((2, 8)), "pre_weight": at((8,)), "residual_grad": at((2, 3, 8)),
         "branch_grad": at((2, 3, 8), F16), "post_weight_grad": at((8,)), "post_bias_grad": at((8,)), "pre_weight_grad": at((8,)),
         "pre_bias_grad": at((8,)), "gate_grad": at((2, 8))}
    options = {"kind": 0, "flags": 1, "workspace": 0, "workspace_bytes": 0}
    for k, v in replaced.items():
        (options if k in options else t)[k] = v
    return graph.block_norm_grad_args(list(t.values()), 1.0, 1.0, options["kind"], options["flags"], options["workspace"], options["workspace_bytes"])


def test_block_norm_backward():
    at = At()

    def says(**k):
        return answer(NORM_BACKWARD, grad_args(at, **k))

    none = dict.fromkeys(("pre_weight", "pre_weight_grad", "pre_bias_grad"))
    assert says() == OK
    assert says(out_grad=None) == OK
    assert says(normed_grad=None) == INVALID and says(normed_grad=None, **none) == OK
    assert says(normed_grad=None, out_grad=None, **none) == INVALID
    assert says(out=None) == INVALID and says(stats=None) == INVALID and says(branch=None) == INVALID
    assert says(gate_grad=at((3, 8))) == SHAPE and says(gate_grad=at((1, 8))) == SHAPE
    assert says(gate=None, gate_grad=None) == OK and says(gate=at((8,)), gate_grad=at((1, 8))) == OK
    assert says(gate_grad=at((2, 8), F16)) == DTYPE     # gradients of two types
    assert says(flags=0) == INVALID
    assert says(flags=0, post_weight=None, post_bias=None, post_weight_grad=None, post_bias_grad=None) == OK
    d = at((2, 3, 8))
    assert says(out_grad=d, residual_grad=d) == OK
    assert says(out_grad=TensorDesc(d.data, d.dims, (0, 0, 4), F32), residual_grad=d) == INVALID
    assert says(residual_grad=at((2, 3, 8), F32, (0, 32, 4))) == INVALID
    s = at((6, 4))
    assert says(stats=s, pre_weight_grad=TensorDesc(s.data, (8,), (4,), F32)) == INVALID
    g = at((8,))
    assert says(pre_weight_grad=g, pre_bias_grad=g) == INVALID
    assert says(workspace=d.data, workspace_bytes=4096, residual_grad=d) == INVALID
    n = C.c_size_t(0)
    lib = _abi.load()
    assert lib.b200_block_norm_backward_workspace(grad_args(at), C.byref(n)) == OK and n.value > 0
    assert lib.b200_block_norm_backward_workspace(grad_args(at, kind=7), C.byref(n)) == INVALID


def distill_args(at, **replaced):
    t = {"logits": at((2, 3, 50), F16), "teacher_ids": at((2, 3, 4), I32), "teacher_logits": at((2, 3, 4)), "labels": at((2, 3), I64), "losses": at((2, 3)),
         "stats": at((6, 4)), "losses_grad": at((2, 3)), "grad": at((2, 3, 50), F16)}
    options = {"temperature": 1.0, "hard_weight": 0.5}
    for k, v in replaced.items():
        (options if k in options else t)[k] = v
    return graph.distill_args(list(t.values()), options["temperature"], options["hard_weight"], 1.0)


@pytest.mark.parametrize("which", [DISTILL, DISTILL_BACKWARD])
def test_distill(which):
    at = At()

    def says(**k):
        if which == DISTILL_BACKWARD:
            k.setdefault("losses", None)
        return answer(which, distill_args(at, **k))

    assert says() == OK
    for temperature in (0.0, -1.0, float("nan"), float("inf")):
        assert says(temperature=temperature) == INVALID
    for hard in (-0.1, 1.5, float("nan")):
        assert says(hard_weight=hard) == INVALID
    assert says(labels=None) == INVALID and says(labels=None, hard_weight=0.0) == OK
    assert says(labels=at((6,), I64)) == SHAPE and says(labels=at((2, 3))) == DTYPE
    assert says(teacher_ids=at((2, 3, 5), I32)) == SHAPE and says(teacher_ids=at((6, 4), I32)) == SHAPE and says(teacher_ids=at((2, 3, 4))) == DTYPE
    assert says(teacher_ids=at((2, 3, 1025), I32), teacher_logits=at((2, 3, 1025))) == NOT_IMPLEMENTED
    assert says(teacher_ids=at((2, 3, 0), I32), teacher_logits=at((2, 3, 0))) == OK
    assert says(logits=at((2, 3, 50), I32)) == DTYPE and says(logits=at((2, 3, 0), F16), grad=at((2, 3, 0), F16)) == SHAPE
    assert says(logits=at((2, 3, 50), F16, (300, 100, 4))) == NOT_IMPLEMENTED
    assert says(grad=at((2, 3, 50))) == DTYPE and says(grad=at((2, 3, 49), F16)) == SHAPE and says(grad=at((2, 3, 50), F16, (0, 100, 2))) == INVALID
    assert says(losses_grad=at((2, 3), F16)) == DTYPE and says(losses_grad=at((2, 3), F32, (0, 0))) == OK
    assert says(stats=at((3, 4))) == SHAPE and says(stats=at((6, 4), F16)) == DTYPE and says(stats=at((6, 4), F32, (32, 4))) == SHAPE and says(stats=at((6, 2))) == SHAPE
    z = at((2, 3, 50), F16)
    assert says(logits=z, grad=z) == OK
    assert says(logits=z, grad=TensorDesc(z.data + 100, z.dims, z.strides, F16)) == INVALID
    ids = at((2, 3, 4), I32)
    assert says(teacher_ids=ids, grad=TensorDesc(ids.data, z.dims, z.strides, F16)) == INVALID
    if which == DISTILL:
        assert says(losses=None, stats=None, grad=None) == INVALID
        assert says(losses=None) == OK and says(grad=None) == OK and says(stats=None) == OK
        assert says(losses=at((2, 3), F16)) == DTYPE and says(losses=at((2, 3), F32, (24, 8))) == NOT_IMPLEMENTED and says(losses=at((6,))) == SHAPE
        assert says(logits=z, losses=TensorDesc(z.data, (2, 3), (12, 4), F32)) == INVALID
    else:
        assert says(losses=at((2, 3))) == INVALID and says(stats=None) == INVALID and says(grad=None) == INVALID


def test_null_arguments():
    lib, n = _abi.load(), C.c_size_t(0)
    assert lib.b200_check_operator(0, None, None, 0) == INVALID
    for name in ("embedding", "embedding_backward", "block_norm", "block_norm_backward", "distill_loss", "distill_loss_backward"):
        assert getattr(lib, "b200_" + name)(None, None) == INVALID
    assert lib.b200_embedding_backward_workspace(None, C.byref(n)) == INVALID
    assert lib.b200_block_norm_backward_workspace(None, C.byref(n)) == INVALID
