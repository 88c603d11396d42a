"""Gated recurrences, token log probabilities and AdamW steps without a device: what the calls refuse, how their arguments are packed, and that the formulas which the
kernels are held to are what they say."""
import ctypes as C

import numpy as np
import pytest

from language_steps import byte_values, logprobs, logprobs_backward, recurrence, recurrence_backward
from test_language_refusals import DTYPE, F16, F32, I32, I64, INVALID, NOT_IMPLEMENTED, OK, SHAPE, At, answer
from vkml_b200 import AdamWTensor, TensorDesc, _abi, adamw_table, graph

RECURRENCE, RECURRENCE_BACKWARD, LOGPROBS, LOGPROBS_BACKWARD, ADAMW = range(16, 21)


def test_structs_are_packed_as_the_header_lays_them_out():
    at = At()
    t = [at((2, 4)) for _ in range(10)]
    names = [n for n, _ in _abi.RecurrenceArgs._fields_][:7]
    s = _abi.RecurrenceArgs.from_buffer_copy(graph.recurrence_args(t[:7], 1))
    assert [getattr(s, n).data for n in names] == [x.data for x in t[:7]] and (s.kind, s.flags) == (1, 0)
    names = [n for n, _ in _abi.RecurrenceGradArgs._fields_][:9]
    s = _abi.RecurrenceGradArgs.from_buffer_copy(graph.recurrence_args(t[:9], 1))
    assert [getattr(s, n).data for n in names] == [x.data for x in t[:9]] and s.kind == 1
    names = [n for n, _ in _abi.TokenLogprobsArgs._fields_][:10]
    s = _abi.TokenLogprobsArgs.from_buffer_copy(graph.logprobs_args(t, 2.0, 8.0))
    assert [getattr(s, n).data for n in names] == [x.data for x in t] and (s.temperature, s.grad_scale) == (2.0, 8.0)
    table = adamw_table([AdamWTensor(*t[:6], weight_decay=0.5, lr_scale=0.25)] * 2)
    e = (_abi.AdamWTensor * 2).from_buffer_copy(table.data)[1]
    assert [getattr(e, n).data for n, _ in _abi.AdamWTensor._fields_[:6]] == [x.data for x in t[:6]] and (e.weight_decay, e.lr_scale) == (0.5, 0.25)
    args, _ = graph.adamw_args(table, 0.5, 7, 0.75, 0.875, 0.125, 2.0, -1)
    s = _abi.AdamWArgs.from_buffer_copy(args)
    assert (s.count, s.step, s.beta1, s.beta2, s.lr, s.eps, s.grad_scale, s.seed) == (2, 7, 0.75, 0.875, 0.5, 0.125, 2.0, 0xFFFFFFFF)
    assert C.string_at(s.tensors, len(table.data)) == table.data and s.lr_on_device.data is None
    one = at((1,))
    s = _abi.AdamWArgs.from_buffer_copy(graph.adamw_args(table, one, one, 0.75, 0.875, 0.125, one, 0)[0])
    assert {s.lr_on_device.data, s.step_on_device.data, s.scale_on_device.data} == {one.data} and (s.step, s.grad_scale) == (1, 1.0)


def recurrence_call(at, **replaced):
    t = {"x": at((2, 40, 8), F16), "gate": at((2, 40, 8), F16), "initial": at((2, 8)), "lengths": at((2,), I64), "out": at((2, 40, 8), F16), "final": at((2, 8)),
         "states": at((2, 3, 8))}
    kind, flags = replaced.pop("kind", 0), replaced.pop("flags", 0)
    t.update(replaced)
    return graph.tensors_bytes(list(t.values())) + graph._RECURRENCE_TAIL.pack(kind, flags)


def test_recurrence():
    at = At()

    def says(**k):
        return answer(RECURRENCE, recurrence_call(at, **k))

    assert says() == OK and says(kind=1) == OK and says(kind=2) == INVALID and says(kind=-1) == INVALID and says(flags=1) == INVALID
    assert says(initial=None, lengths=None, final=None, states=None) == OK
    assert says(gate=at((2, 40, 8))) == OK                                               # gates in F32 beside inputs in F16
    assert says(x=at((2, 40, 8)), out=at((2, 40, 8))) == DTYPE                           # not the other way round
    assert says(x=at((2, 40, 8)), gate=at((2, 40, 8)), out=at((2, 40, 8))) == OK
    assert says(out=at((2, 40, 8))) == DTYPE and says(x=at((2, 40, 8), I32)) == DTYPE and says(gate=at((2, 40, 8), I32)) == DTYPE
    assert says(gate=at((2, 41, 8), F16)) == SHAPE and says(gate=at((80, 8), F16)) == SHAPE and says(out=at((2, 40, 9), F16)) == SHAPE
    assert says(x=at((8,), F16), gate=at((8,), F16), out=at((8,), F16)) == SHAPE
    assert says(x=at((1, 2, 40, 8), F16)) == SHAPE
    assert says(initial=at((8,))) == SHAPE and says(initial=at((2, 9))) == SHAPE and says(initial=at((2, 8), F16)) == DTYPE and says(final=at((3, 8))) == SHAPE
    assert says(initial=at((2, 8), F32, (0, 4))) == OK and says(final=at((2, 8), F32, (0, 4))) == INVALID and says(initial=at((2, 8), F32, (64, 8))) == NOT_IMPLEMENTED
    assert says(lengths=at((2,))) == DTYPE and says(lengths=at((3,), I64)) == SHAPE and says(lengths=at((2, 1), I64)) == SHAPE and says(lengths=at((2,), I32, (0,))) == OK
    assert says(states=at((2, 2, 8))) == SHAPE and says(states=at((2, 3, 8), F16)) == DTYPE and says(states=at((2, 3, 8), F32, (128, 32, 4))) == SHAPE and says(states=at((6, 8))) == SHAPE
    assert says(x=at((2, 40, 8), F16, (640, 16, 4))) == NOT_IMPLEMENTED
    assert says(x=at((2, 40, 8), F16, (0, 0, 2)), gate=at((2, 40, 8), F16, (0, 16, 2))) == OK
    assert says(out=at((2, 40, 8), F16, (0, 16, 2))) == INVALID
    x = at((2, 40, 8), F16)
    assert says(x=x, out=x) == OK and says(gate=x, out=x) == OK and says(x=x, gate=x) == OK and says(x=x, gate=x, out=x) == OK
    assert says(x=x, out=TensorDesc(x.data + 16, x.dims, x.strides, F16)) == INVALID
    half = at((2, 40, 8), F16)
    assert says(gate=TensorDesc(half.data, (2, 40, 8), (1280, 32, 4), F32), out=half) == INVALID   # over a gate of another type
    s = at((2, 8))
    assert says(initial=s, final=s) == OK and says(initial=s, final=TensorDesc(s.data + 4, (2, 8), (32, 4), F32)) == INVALID
    assert says(initial=s, states=TensorDesc(s.data, (2, 3, 8), (96, 32, 4), F32)) == INVALID
    assert says(final=TensorDesc(x.data, (2, 8), (32, 4), F32), x=x) == INVALID and says(states=TensorDesc(x.data, (2, 3, 8), (96, 32, 4), F32), x=x) == INVALID
    assert says(lengths=TensorDesc(x.data, (2,), (8,), I64), out=x) == INVALID
    row = {"x": at((40, 8), F16), "gate": at((40, 8), F16), "out": at((40, 8), F16)}
    assert says(**row, initial=at((8,)), final=at((8,)), states=at((3, 8)), lengths=at((), I32)) == OK
    assert says(**row, initial=at((1, 8)), final=None, states=None, lengths=None) == SHAPE
    empty = {k: TensorDesc(0, (2, 0, 8), (0, 16, 2), F16) for k in ("x", "gate", "out")}
    assert says(**empty, states=TensorDesc(0, (2, 0, 8), (0, 32, 4), F32)) == OK


def recurrence_grad_call(at, **replaced):
    t = {"x": at((2, 40, 8), F16), "gate": at((2, 40, 8)), "lengths": at((2,), I32), "states": at((2, 3, 8)), "out_grad": at((2, 40, 8), F16), "final_grad": at((2, 8)),
         "x_grad": at((2, 40, 8), F16), "gate_grad": at((2, 40, 8)), "initial_grad": at((2, 8))}
    kind = replaced.pop("kind", 0)
    t.update(replaced)
    return graph.recurrence_args(list(t.values()), kind)


def test_recurrence_backward():
    at = At()

    def says(**k):
        return answer(RECURRENCE_BACKWARD, recurrence_grad_call(at, **k))

    assert says() == OK and says(kind=1) == OK and says(kind=3) == INVALID
    assert says(lengths=None, out_grad=None, final_grad=None) == OK
    assert says(states=None) == INVALID and says(x_grad=None, gate_grad=None, initial_grad=None) == INVALID
    for name in ("x_grad", "gate_grad", "initial_grad"):
        assert says(**{k: None for k in ("x_grad", "gate_grad", "initial_grad") if k != name}) == OK
    assert says(x_grad=at((2, 40, 8))) == DTYPE and says(gate_grad=at((2, 40, 8), F16)) == DTYPE and says(out_grad=at((2, 40, 8))) == DTYPE
    assert says(x_grad=at((2, 40, 7), F16)) == SHAPE and says(out_grad=at((80, 8), F16)) == SHAPE and says(initial_grad=at((8,))) == SHAPE
    assert says(out_grad=at((2, 40, 8), F16, (0, 0, 2))) == OK and says(x_grad=at((2, 40, 8), F16, (0, 16, 2))) == INVALID
    x, g, d, f, s = at((2, 40, 8), F16), at((2, 40, 8)), at((2, 40, 8), F16), at((2, 8)), at((2, 3, 8))
    assert says(x=x, x_grad=x) == OK and says(out_grad=d, x_grad=d) == OK and says(gate=g, gate_grad=g) == OK and says(final_grad=f, initial_grad=f) == OK
    assert says(x=x, gate_grad=TensorDesc(x.data, (2, 40, 8), (1280, 32, 4), F32)) == INVALID
    assert says(x_grad=x, gate_grad=TensorDesc(x.data, (2, 40, 8), (1280, 32, 4), F32)) == INVALID
    assert says(states=s, initial_grad=TensorDesc(s.data, (2, 8), (32, 4), F32)) == INVALID
    assert says(states=s, x_grad=TensorDesc(s.data, (2, 40, 8), (640, 16, 2), F16)) == INVALID
    assert says(final_grad=f, x_grad=TensorDesc(f.data, (2, 40, 8), (640, 16, 2), F16)) == INVALID


def logprobs_call(at, forward, **replaced):
    t = {"logits": at((2, 3, 50), F16), "tokens": at((2, 3), I64), "logprobs": at((2, 3)), "entropies": at((2, 3)), "stats": at((6, 4)), "top_ids": at((2, 3, 5), I32),
         "top_logprobs": at((2, 3, 5)), "logprobs_grad": at((2, 3)), "entropies_grad": at((2, 3)), "grad": at((2, 3, 50), F16)}
    for k in ("logprobs_grad", "entropies_grad", "grad") if forward else ("logprobs", "entropies", "top_ids", "top_logprobs"):
        t[k] = None
    temperature, scale = replaced.pop("temperature", 1.0), replaced.pop("scale", 1.0)
    t.update(replaced)
    return graph.logprobs_args(list(t.values()), temperature, scale)


def test_logprobs():
    at = At()

    def says(**k):
        return answer(LOGPROBS, logprobs_call(at, True, **k))

    assert says() == OK
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-39):
        assert says(temperature=temperature) == INVALID
    nothing = dict.fromkeys(("logprobs", "entropies", "stats", "top_ids", "top_logprobs"))
    assert says(**nothing) == INVALID
    for k, x in (("entropies", at((2, 3))), ("stats", at((6, 4))), ("top_ids", at((2, 3, 1), I64)), ("top_logprobs", at((2, 3, 50)))):
        assert says(**{**nothing, k: x}, tokens=None) == OK, k
    assert says(tokens=None) == INVALID and says(tokens=None, logprobs=None) == OK
    assert says(tokens=at((6,), I64)) == SHAPE and says(tokens=at((2, 3))) == DTYPE and says(tokens=at((2, 3), I32, (0, 0))) == OK
    assert says(logprobs=at((2, 3), F16)) == DTYPE and says(logprobs=at((6,))) == SHAPE and says(entropies=at((2, 3), F32, (24, 8))) == NOT_IMPLEMENTED
    assert says(stats=at((3, 4))) == SHAPE and says(stats=at((6, 4), F16)) == DTYPE
    assert says(top_ids=at((2, 3, 6), I32)) == SHAPE and says(top_ids=at((2, 3, 5))) == DTYPE and says(top_logprobs=at((2, 3, 5), F16)) == DTYPE and says(top_ids=at((6, 5), I32)) == SHAPE
    assert says(top_ids=at((2, 3, 51), I32), top_logprobs=None) == SHAPE
    wide = at((2, 3, 500), F16)
    assert says(logits=wide, top_ids=at((2, 3, 129), I32), top_logprobs=None) == NOT_IMPLEMENTED and says(logits=wide, top_ids=at((2, 3, 128), I32), top_logprobs=None) == OK
    assert says(top_ids=at((2, 3, 5), I32, (0, 20, 4))) == INVALID
    assert says(logits=at((2, 3, 50), I32)) == DTYPE and says(logits=at((2, 3, 0), F16)) == SHAPE and says(logits=at((2, 3, 50), F16, (300, 100, 4))) == NOT_IMPLEMENTED
    assert says(logits=at((2, 3, 50), F16, (0, 0, 2))) == OK
    z, h = at((2, 3, 50), F16), at((2, 3))
    assert says(logits=z, logprobs=TensorDesc(z.data, (2, 3), (12, 4), F32)) == INVALID and says(logprobs=h, entropies=h) == INVALID
    assert says(logits=z, top_ids=TensorDesc(z.data, (2, 3, 5), (60, 20, 4), I32)) == INVALID
    assert says(grad=at((2, 3, 50), F16)) == INVALID and says(logprobs_grad=h) == INVALID


def test_logprobs_backward():
    at = At()

    def says(**k):
        return answer(LOGPROBS_BACKWARD, logprobs_call(at, False, **k))

    assert says() == OK and says(logprobs_grad=None) == OK and says(entropies_grad=None) == OK and says(temperature=0.0) == INVALID
    assert says(grad=None) == INVALID and says(stats=None) == INVALID and says(tokens=None) == INVALID and says(tokens=None, logprobs_grad=None) == OK
    assert says(logprobs=at((2, 3))) == INVALID and says(top_ids=at((2, 3, 1), I32)) == INVALID
    assert says(grad=at((2, 3, 50))) == DTYPE and says(grad=at((2, 3, 49), F16)) == SHAPE and says(grad=at((2, 3, 50), F16, (0, 100, 2))) == INVALID
    assert says(logprobs_grad=at((2, 3), F16)) == DTYPE and says(logprobs_grad=at((2, 3), F32, (0, 0))) == OK and says(entropies_grad=at((6,))) == SHAPE
    z, s = at((2, 3, 50), F16), at((6, 4))
    assert says(logits=z, grad=z) == OK and says(logits=z, grad=TensorDesc(z.data + 100, z.dims, z.strides, F16)) == INVALID
    assert says(stats=s, grad=TensorDesc(s.data, z.dims, z.strides, F16)) == INVALID
    # more blocks than a launch has room for: 2^31 - 1 rows of two blocks each
    n = (1 << 31) - 1
    rows = {"tokens": at((n,), I32, (0,)), "stats": TensorDesc.contiguous(1 << 58, (n, 4), F32), "logprobs_grad": None, "entropies_grad": None}
    for width, status in ((8192, OK), (8200, SHAPE)):
        assert says(logits=at((n, width), F16, (0, 2)), grad=TensorDesc.contiguous(1 << 60, (n, width), F16), **rows) == status


def adamw_call(tensors, **options):
    o = {"lr": 0.1, "step": 1, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "grad_scale": 1.0, "seed": 0, **options}
    return graph.adamw_args(adamw_table(tensors), *o.values())


def test_adamw():
    at = At()

    def full(**replaced):
        t = {"param": at((30, 20)), "grad": at((30, 20), F16), "first": at((30, 20)), "second": at((30, 20))}
        t.update(replaced)
        return AdamWTensor(**t)

    def eight(**replaced):
        return full(**{"first": at((150,), I32), "second": at((150,), I32), "scales": at((3, 2)), **replaced})

    def says(*tensors, **options):
        args, keep = adamw_call(tensors or (full(), eight()), **options)
        return answer(ADAMW, args)

    assert says() == OK
    assert AdamWTensor.state_dims(600) == ((150,), (3, 2)) and AdamWTensor.state_dims(1) == ((1,), (1, 2))
    assert says(step=0) == INVALID and says(lr=float("nan")) == INVALID and says(lr=float("inf")) == INVALID and says(lr=-1.0) == OK and says(grad_scale=float("inf")) == INVALID
    for beta in ("beta1", "beta2"):
        assert says(**{beta: 1.0}) == INVALID and says(**{beta: -0.1}) == INVALID and says(**{beta: float("nan")}) == INVALID and says(**{beta: 0.0}) == OK
    assert says(eps=0.0) == INVALID and says(eps=float("inf")) == INVALID
    assert says(lr=at((1,)), step=at((), I64), grad_scale=at((1, 1))) == OK
    assert says(lr=at((2,))) == SHAPE and says(lr=at((1,), F16)) == DTYPE and says(step=at((1,), I32)) == DTYPE and says(grad_scale=at((0,))) == SHAPE
    assert says(full(param=at((30, 20), F16))) == DTYPE and says(full(grad=at((30, 20), I32))) == DTYPE and says(full(first=at((30, 20), F16))) == DTYPE
    assert says(full(first=at((150,), I32))) == DTYPE                                    # one in 8 bits, one in 32
    assert says(full(grad=at((600,)))) == SHAPE and says(full(second=at((20, 30)))) == SHAPE and says(full(param=at((30, 20), F32, (4, 120)))) == NOT_IMPLEMENTED
    assert says(full(scales=at((3, 2)))) == INVALID and says(eight(scales=None)) == INVALID
    assert says(eight(first=at((149,), I32))) == SHAPE and says(eight(first=at((1, 150), I32))) == SHAPE and says(eight(scales=at((2, 2)))) == SHAPE
    assert says(eight(scales=at((3, 2), F32, offset=4))) == SHAPE and says(eight(scales=at((3, 2), F16))) == DTYPE
    assert says(full(copy=at((30, 20), F16))) == OK and says(full(copy=at((30, 20)))) == DTYPE and says(full(copy=at((20, 30), F16))) == SHAPE
    assert says(full(param=TensorDesc(0, (30, 20), (80, 4), F32))) == INVALID
    assert says(full(weight_decay=-0.1)) == INVALID and says(full(weight_decay=float("nan"))) == INVALID and says(full(lr_scale=float("inf"))) == INVALID
    # what is written lies on nothing else: within a tensor, between two, on the numbers on the device; gradients may be shared
    a, b = full(), full()
    assert says(a, b) == OK and says(a, a) == INVALID and says(a, full(grad=a.grad)) == OK
    assert says(full(first=a.param, param=a.param)) == INVALID and says(a, full(copy=TensorDesc(a.grad.data, (30, 20), (40, 2), F16))) == INVALID
    assert says(a, full(second=TensorDesc(b.param.data + 80 * 29, (30, 20), (80, 4), F32)), b) == INVALID
    assert says(a, lr=TensorDesc(a.param.data + 40, (1,), (4,), F32)) == INVALID
    assert says(full(grad=TensorDesc(a.param.data, (30, 20), (80, 4), F32)), a) == INVALID
    empty = {k: TensorDesc(0, (0,), (4,), F32) for k in ("param", "grad", "first", "second")}
    assert says(AdamWTensor(**empty)) == OK
    args, keep = adamw_call(())
    assert answer(ADAMW, args) == OK
    s = _abi.AdamWArgs.from_buffer_copy(args)
    s.tensors, s.count = None, 3
    assert answer(ADAMW, bytes(s)) == INVALID
    s.count = -1
    assert answer(ADAMW, bytes(s)) == INVALID


def test_null_arguments():
    lib = _abi.load()
    for which in range(16, 21):
        assert lib.b200_check_operator(which, None, None, 0) == INVALID
    for name in ("gated_recurrence", "gated_recurrence_backward", "token_logprobs", "token_logprobs_backward", "adamw"):
        assert getattr(lib, "b200_" + name)(None, None) == INVALID


# ---- the formulas -----------------------------------------------------------

@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
def test_a_recurrences_gradient_is_that_of_its_formula(kind):
    """Against central differences in 64 bits (third-order terms: 1e-10 here)."""
    rng = np.random.default_rng(0)
    x, gate, initial = rng.standard_normal((2, 5, 3)), rng.standard_normal((2, 5, 3)) - (1 if kind == "exp" else 0), rng.standard_normal((2, 3))
    lengths = np.array([5, 3])
    dout, dfinal = rng.standard_normal(x.shape), rng.standard_normal(initial.shape)
    got = recurrence_backward(x, gate, initial, lengths, kind, dout, dfinal)
    leaves = {"x": x, "gate": gate, "initial": initial}

    def value(**changed):
        r = recurrence(**{**leaves, **changed}, lengths=lengths, kind=kind)
        return (r["out"][0] * dout).sum() + (r["final"][0] * dfinal).sum()

    for name, leaf in leaves.items():
        for i in np.ndindex(leaf.shape):
            step = np.zeros(leaf.shape)
            step[i] = 1e-5
            assert abs((value(**{name: leaf + step}) - value(**{name: leaf - step})) / 2e-5 - got[name][0][i]) < 1e-8, (name, i)


def test_a_log_probabilitys_gradient_is_that_of_its_formula():
    rng = np.random.default_rng(0)
    z, tokens, ulp, uh = rng.standard_normal((3, 6)) * 2, np.array([2, -1, 5]), np.array([1.5, 2.0, -3.0]), np.array([0.5, -1.0, 2.0])
    want = logprobs(z, tokens, 1.7)
    g, _ = logprobs_backward(z, tokens, want["stats"][0], ulp, uh, 1.7, 2.0)
    for j in range(6):
        step = np.zeros((3, 6))
        step[:, j] = 1e-5
        up, down = logprobs(z + step, tokens, 1.7), logprobs(z - step, tokens, 1.7)
        difference = sum(u * (up[k][0] - down[k][0]) for u, k in ((ulp, "logprobs"), (uh, "entropies"))) / 2e-5 * 2.0
        assert np.abs(difference - g[:, j]).max() < 1e-8


def test_what_the_bytes_stand_for():
    v = byte_values()
    assert v[0] == 0 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and v[0x7E] == 448 and np.isnan(v[0x7F]) and np.array_equal(v[128:255], -v[:127])
    assert np.all(np.diff(v[:127]) > 0)
