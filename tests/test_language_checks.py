"""b200_check_operator tells what the call would answer: limits of extents and the workspace too, without a device."""
import ctypes as C

from test_language_refusals import (DISTILL, DISTILL_BACKWARD, EMBEDDING, EMBEDDING_BACKWARD, F16, F32, I32, I64, INVALID, NORM, NORM_BACKWARD, OK, SHAPE, At, answer,
                                    distill_args, grad_args, norm_args)
from vkml_b200 import TensorDesc, _abi, graph


def size(name, args):
    n = C.c_size_t(0)
    status = getattr(_abi.load(), f"b200_{name}_workspace")(args, C.byref(n))
    return n.value if status == OK else -status


def test_rows_of_a_table():
    at = At()

    def args(width, table=F32, **k):
        return graph.embedding_args(at((4, width), table), at((3,), I64), at((3, width), F16), 1.0, **k)

    assert answer(EMBEDDING, args(1 << 24)) == OK
    for which, width, says in ((EMBEDDING_BACKWARD, (1 << 24) - 1, OK), (EMBEDDING_BACKWARD, 1 << 24, SHAPE)):
        assert answer(which, args(width)) == says
        assert (size("embedding_backward", args(width)) >= 0) == (says == OK)


def test_lookups_of_many_pieces():
    """Blocks of 8 rows of one to 256 odd columns each."""
    at = At()
    says = lambda n, width: answer(EMBEDDING, graph.embedding_args(at((4, width), F32), at((n,), I64, (0,)), at((n, width), F16), 1.0))  # noqa: E731
    assert says((1 << 31) - 1, 255) == OK
    assert says((1 << 31) - 1, 256 * 10 - 1) == SHAPE


def test_an_embeddings_workspace():
    at = At()
    tensors = at((5000, 64)), at((3000,), I64), at((3000, 64), F16)
    need = size("embedding_backward", graph.embedding_args(*tensors, 1.0))
    assert need > 0
    base = 1 << 20

    def says(address, nbytes):
        return answer(EMBEDDING_BACKWARD, graph.embedding_args(*tensors, 1.0, workspace=address, workspace_bytes=nbytes))

    assert says(base, need) == OK and says(base, need + 1) == OK
    assert says(base, need - 1) == INVALID and says(base, 0) == INVALID
    assert says(base + 128, need) == INVALID
    assert says(0, 0) == OK and says(0, need) == OK  # the context's own
    few = at((50, 8)), at((3,), I64), at((3, 8), F16)
    assert size("embedding_backward", graph.embedding_args(*few, 1.0)) == 0
    assert answer(EMBEDDING_BACKWARD, graph.embedding_args(*few, 1.0, workspace=base + 8, workspace_bytes=1)) == OK  # nothing is needed


def test_a_norms_workspace():
    at = At()
    tensors = dict(zip(("out", "branch", "stats", "out_grad", "normed_grad", "residual_grad", "branch_grad"),
                       (at((2, 3, 8)), at((2, 3, 8), F16), at((6, 4)), at((2, 3, 8)), at((2, 3, 8), F16), at((2, 3, 8)), at((2, 3, 8), F16))))
    need = size("block_norm_backward", grad_args(at, **tensors))
    assert need > 0
    base = 1 << 20

    def says(address, nbytes, **more):
        return answer(NORM_BACKWARD, grad_args(at, **tensors, workspace=address, workspace_bytes=nbytes, **more))

    assert says(base, need) == OK
    assert says(base, need - 1) == INVALID and says(base, 0) == INVALID and says(base + 64, need) == INVALID
    assert size("block_norm_backward", grad_args(at, **tensors, workspace=base, workspace_bytes=1)) == need  # the question does not ask for the answer
    none = dict.fromkeys(("post_weight_grad", "post_bias_grad", "pre_weight_grad", "pre_bias_grad", "gate_grad"))
    assert size("block_norm_backward", grad_args(at, **tensors, **none)) == 0
    assert says(base + 64, 1, **none) == OK


def test_many_long_rows_of_logits():
    """Rows that take two blocks each, as their entries ask for: 2^30 of them are as many blocks as a launch has no room for."""
    at = At()

    def losses_alone(n, vocab, top):
        rows = lambda width, dtype, nbytes: at((n, width), dtype, (0, nbytes))  # noqa: E731
        return answer(DISTILL, distill_args(at, logits=rows(vocab, F16, 2), teacher_ids=rows(top, I32, 4), teacher_logits=rows(top, F32, 4), labels=None, stats=None,
                                            losses=at((n,)), losses_grad=None, grad=None, hard_weight=0.0))

    assert losses_alone(1 << 20, 20000, 1000) == OK
    assert losses_alone(1 << 30, 20000, 1000) == SHAPE
    assert losses_alone(1 << 30, 20000, 10) == OK  # blocks that stay take these


def without_storage(t):
    return TensorDesc(0, t.dims, t.strides, t.dtype)


def test_rows_of_no_element_need_no_storage():
    """Weights of their norms are as welcome as with rows, and gradients of sums of nothing."""
    at = At()
    h, y = (without_storage(at((0, 8), dtype)) for dtype in (F32, F16))
    assert answer(NORM, norm_args(at, residual=h, branch=y, out=h, normed=y, stats=None, gate=at((8,)))) == OK
    assert answer(NORM, norm_args(at, residual=h, branch=None, out=h, normed=y, stats=None, gate=None, flags=0, post_weight=None, post_bias=None)) == OK
    assert answer(NORM_BACKWARD, grad_args(at, out=h, branch=y, out_grad=h, normed_grad=y, residual_grad=h, branch_grad=y, stats=None, gate=at((8,)), gate_grad=at((8,)))) == OK
    assert answer(NORM, norm_args(at, residual=without_storage(at((0, 9))))) == SHAPE
    no_width = {k: without_storage(at((2, 3, 0), F16 if k in ("branch", "normed") else F32)) for k in ("residual", "branch", "out", "normed")}
    assert answer(NORM, norm_args(at, **no_width, **{k: without_storage(at((0,))) for k in ("post_weight", "post_bias", "pre_weight", "pre_bias", "gate")})) == OK


def test_a_tensor_without_storage_is_absent_whatever_its_extents():
    """Where a call can do without it: its extents are then those of nothing."""
    at = At()
    for name in ("residual", "stats", "out", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate"):
        for dims in ((2, 3, 8), (7,), (3, 5, 9, 2)):
            assert answer(NORM, norm_args(at, **{name: without_storage(at(dims))})) == OK, (name, dims)
    none = without_storage(at((2, 3, 8), F16))
    assert answer(NORM, norm_args(at, branch=none)) == INVALID  # a gate of nothing
    assert answer(NORM, norm_args(at, branch=none, gate=none, flags=0, post_weight=none, post_bias=none)) == OK
    assert answer(NORM, norm_args(at, branch=none, residual=none, gate=none, flags=0, post_weight=none, post_bias=none)) == INVALID
    for name in ("out_grad", "residual_grad", "branch_grad", "gate_grad", "post_bias", "pre_bias_grad"):
        assert answer(NORM_BACKWARD, grad_args(at, **{name: without_storage(at((2, 3, 8)))})) == OK, name
    for which, losses in ((DISTILL, at((2, 3))), (DISTILL_BACKWARD, without_storage(at((2, 3))))):
        for name in ("labels", "losses_grad"):
            absent = {name: without_storage(at((2, 3), I64 if name == "labels" else F32))}
            assert answer(which, distill_args(at, losses=losses, **absent, hard_weight=0.0)) == OK, name
        assert answer(which, distill_args(at, losses=losses, labels=without_storage(at((2, 3), I64)))) == INVALID  # a weight of nothing
    # what a call cannot do without
    assert answer(DISTILL, distill_args(at, logits=without_storage(at((2, 3, 50), F16)))) == INVALID


def test_temperatures_whose_inverse_times_log2_e_is_not_finite():
    """The smallest temperature is log2(e) / the largest float, 4.24e-39: a logit's exponent is taken by that product."""
    at = At()
    for which, losses in ((DISTILL, at((2, 3))), (DISTILL_BACKWARD, None)):
        for temperature, says in ((2.95e-39, INVALID), (4.2e-39, INVALID), (4.3e-39, OK), (1e-30, OK), (3e38, OK)):
            assert answer(which, distill_args(at, losses=losses, temperature=temperature)) == says, temperature
