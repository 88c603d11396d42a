"""Gated recurrences, token log probabilities and AdamW steps as a training step uses them, with the operators beside them: together, captured into a graph, by two
threads, and on tensors that are larger than 32-bit offsets."""
import ctypes as C
import threading

import numpy as np
import pytest

import vkml_b200 as B
from language import EPS, check
from language_steps import logprobs, moments, recurrence, recurrence_backward, update
from test_language_together_gpu import capture, runtime, tensor
from vkml_b200 import AdamWTensor, DeviceTensor, NodeDesc, TensorDesc, adamw_table
from vkml_b200.graph import DType, Op

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


class Step:
    """A model of one recurrent block, trained by a policy's gradient: embedding -> norm -> two products (inputs and gates) -> recurrence -> norm, gate and the sum with the
    residual stream -> projection -> log probabilities of the tokens, their weighted sum and a share of the entropies -> back to every parameter -> AdamW."""

    vocab, width, batch, length = 301, 64, 3, 37
    lr, decay = 1e-2, 0.1

    def __init__(self, backend, seed=0):
        rng = np.random.default_rng(seed)
        self.backend, n, d, v = backend, self.batch * self.length, self.width, self.vocab
        a = {"table": rng.standard_normal((v, d)) * 0.5, "first": rng.standard_normal(d) * 0.1 + 1, "wx": rng.standard_normal((d, d)) / 8, "wg": rng.standard_normal((d, d)) / 8,
             "post": rng.standard_normal(d) * 0.1 + 1, "pre": rng.standard_normal(d) * 0.1 + 1, "out": rng.standard_normal((d, v)) / 8, "start": rng.standard_normal((self.batch, d))}
        self.params = {k: x.astype(F32) for k, x in a.items()}
        self.ids = rng.integers(0, v, (self.batch, self.length))
        self.tokens = rng.integers(0, v, n)
        self.tokens[-3:] = -1
        self.weights, self.bonus = rng.standard_normal(n).astype(F32), np.full(n, 0.1, F32)
        self.t = {k: tensor(backend, x) for k, x in {**self.params, "ids": self.ids, "tokens": self.tokens, "weights": self.weights, "bonus": self.bonus}.items()}
        e = lambda *dims: DeviceTensor.empty(backend, dims)  # noqa: E731
        self.r = {k: e(n, d) for k in ("x", "n", "in", "gate", "y", "h", "m", "dm", "dh", "dy", "dn", "dn2", "dnorm", "din", "dgate", "dx")}
        self.r.update({"states": e(self.batch, -(-self.length // 16), d), "stats0": e(n, 4), "stats1": e(n, 4), "logits": e(n, v), "logprobs": e(n), "entropies": e(n), "stats2": e(n, 4),
                       "dlogits": e(n, v), **{"d_" + k: e(*x.shape) for k, x in self.params.items()}})
        self.scratch = backend.allocate(1 << 22)
        self.table = None

    def matmul(self, out, a, b):
        four = lambda t: TensorDesc(t.desc.data, (1, 1) + t.desc.dims, (0, 0) + t.desc.strides, t.desc.dtype)  # noqa: E731
        self.backend.compute([NodeDesc(int(Op.MATMUL), four(out), [four(a), four(b)])])

    def rows(self, t):
        return TensorDesc.contiguous(t.desc.data, (self.batch, self.length) + t.desc.dims[1:], t.desc.dtype)

    def gradients(self):
        g, t, r, rows = self.backend, self.t, self.r, self.rows
        g.embedding(t["table"], t["ids"], rows(r["x"]), scale=8.0)
        g.block_norm(rows(r["x"]), None, normed=rows(r["n"]), stats=r["stats0"], pre_weight=t["first"])
        self.matmul(r["in"], r["n"], t["wx"])
        self.matmul(r["gate"], r["n"], t["wg"])
        g.gated_recurrence(rows(r["in"]), rows(r["gate"]), rows(r["y"]), initial=t["start"], states=r["states"])
        g.block_norm(rows(r["x"]), rows(r["y"]), out=rows(r["h"]), normed=rows(r["m"]), stats=r["stats1"], post_weight=t["post"], pre_weight=t["pre"], branch_scale=0.7)
        self.matmul(r["logits"], r["m"], t["out"])
        g.token_logprobs(r["logits"], t["tokens"], r["logprobs"], entropies=r["entropies"], stats=r["stats2"], temperature=1.3)
        g.token_logprobs_backward(r["logits"], t["tokens"], r["stats2"], r["dlogits"], logprobs_grad=t["weights"], entropies_grad=t["bonus"], temperature=1.3)
        self.matmul(r["dm"], r["dlogits"], t["out"].transpose(0, 1))
        self.matmul(r["d_out"], r["m"].transpose(0, 1), r["dlogits"])
        g.block_norm_backward(rows(r["h"]), rows(r["y"]), r["stats1"], normed_grad=rows(r["dm"]), residual_grad=rows(r["dh"]), branch_grad=rows(r["dy"]), post_weight=t["post"],
                              pre_weight=t["pre"], post_weight_grad=r["d_post"], pre_weight_grad=r["d_pre"], branch_scale=0.7, workspace=self.scratch)
        g.gated_recurrence_backward(rows(r["in"]), rows(r["gate"]), r["states"], out_grad=rows(r["dy"]), x_grad=rows(r["din"]), gate_grad=rows(r["dgate"]), initial_grad=r["d_start"])
        self.matmul(r["dn"], r["din"], t["wx"].transpose(0, 1))
        self.matmul(r["dn2"], r["dgate"], t["wg"].transpose(0, 1))
        self.matmul(r["d_wx"], r["n"].transpose(0, 1), r["din"])
        self.matmul(r["d_wg"], r["n"].transpose(0, 1), r["dgate"])
        g.compute([NodeDesc(int(Op.ADD), r["dnorm"].desc, [r["dn"].desc, r["dn2"].desc])])
        g.block_norm_backward(rows(r["x"]), None, r["stats0"], out_grad=rows(r["dh"]), normed_grad=rows(r["dnorm"]), residual_grad=rows(r["dx"]), pre_weight=t["first"],
                              pre_weight_grad=r["d_first"], workspace=self.scratch)
        g.embedding_backward(rows(r["dx"]), t["ids"], r["d_table"], scale=8.0, workspace=self.scratch)

    def optimise(self, step, **options):
        if self.table is None:
            zero = lambda shape, dtype=F32: tensor(self.backend, np.zeros(shape, dtype))  # noqa: E731
            self.state = {}
            for i, (k, x) in enumerate(self.params.items()):
                words, scales = AdamWTensor.state_dims(x.size)
                eight = i % 2 == 1  # states of both kinds
                self.state[k] = AdamWTensor(self.t[k], self.r["d_" + k], *(zero(words, np.int32) if eight else zero(x.shape) for _ in range(2)), scales=zero(scales) if eight else None,
                                            copy=DeviceTensor.empty(self.backend, x.shape, DType.F16), weight_decay=self.decay)
            self.table = adamw_table(list(self.state.values()))
        self.backend.adamw(self.table, lr=self.lr, step=step, seed=1, **options)

    def value(self, a):
        """What the gradients are of, in 64 bits: weighted log probabilities and entropies."""
        a = {k: x.astype(np.float64) for k, x in a.items()}
        norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)  # noqa: E731
        x = 8.0 * a["table"][self.ids]
        n = norm(x) * a["first"]
        i, gate = n @ a["wx"], n @ a["wg"]
        s, h, y = 1 / (1 + np.exp(-gate)), a["start"], []
        for t in range(self.length):
            h = s[:, t] * h + (1 - s[:, t]) * i[:, t]
            y.append(h)
        m = norm(x + 0.7 * norm(np.stack(y, 1)) * a["post"]) * a["pre"]
        z = (m @ a["out"]).reshape(-1, self.vocab) / 1.3
        lq = z - z.max(-1, keepdims=True)
        lq = lq - np.log(np.exp(lq).sum(-1, keepdims=True))
        lp = np.where(self.tokens >= 0, lq[np.arange(len(z)), np.maximum(self.tokens, 0)], 0.0)
        return lp, (lp * self.weights).sum() + (-(np.exp(lq) * lq).sum(-1) * self.bonus).sum()


def test_a_training_step(backend):
    """Log probabilities against the model in 64 bits, every parameter's gradient against its differences there (along a random direction the central difference with step
    1e-4 is off by its third-order term, below 1e-6 of the value here, and the kernels by the products' error, 4e-6 relative at these sizes through three layers: 2e-4 of the gradient's
    and the direction's lengths holds both), and the parameters that the step leaves against the formulas with these gradients."""
    step = Step(backend)
    step.gradients()
    lp, _ = step.value(step.params)
    assert np.allclose(step.r["logprobs"].numpy(), lp, rtol=1e-4, atol=1e-4)
    rng = np.random.default_rng(1)
    grads = {k: step.r["d_" + k].numpy() for k in step.params}
    for k, x in step.params.items():
        direction = rng.standard_normal(x.shape)
        up, down = (step.value({**step.params, k: x.astype(np.float64) + s * direction})[1] for s in (1e-4, -1e-4))
        size = np.linalg.norm(grads[k].astype(np.float64)) * np.linalg.norm(direction)
        assert abs((grads[k].astype(np.float64) * direction).sum() - (up - down) / 2e-4) <= 2e-4 * size, k
    step.optimise(1)
    for k, x in step.params.items():
        m, v = moments(grads[k], np.zeros(x.shape), np.zeros(x.shape), 0.9, 0.999)
        p, bound = update(x, (m[0], m[1] + 4 * EPS * np.abs(m[0])), v, step.lr, step.decay, 1, 0.9, 0.999, 1e-8)
        got = step.t[k].numpy()
        check(got, p, bound, F32, k)
        assert np.array_equal(step.state[k].copy.numpy(), got.astype(F16)), k


def test_the_same_bits_again_and_between_other_work(backend):
    step, other = Step(backend), Step(backend, 1)
    step.gradients()
    first = {k: step.r["d_" + k].numpy() for k in step.params}
    for _ in range(2):
        other.gradients()
        step.gradients()
        other.gradients()
    for k, x in first.items():
        assert np.array_equal(step.r["d_" + k].numpy(), x), k


def problem(backend, seed):
    """Calls of every kind: a cluster's recurrence and its gradients, a cluster's row and blocks' rows of logits, states of 8 bits, numbers on the device."""
    rng = np.random.default_rng(seed)
    a = {"x": rng.standard_normal((2, 900, 136)).astype(F16), "gate": rng.standard_normal((2, 900, 136)).astype(F16), "dout": rng.standard_normal((2, 900, 136)).astype(F16),
         "state": rng.standard_normal((2, 136)).astype(F32), "z": rng.standard_normal((3, 40000)).astype(F32), "z2": rng.standard_normal((400, 3000)).astype(F16),
         "tokens": rng.integers(0, 40000, 3), "tokens2": rng.integers(0, 3000, 400), "w": rng.standard_normal(400).astype(F32), "param": rng.standard_normal(5000).astype(F32),
         "grad": rng.standard_normal(5000).astype(F16), "first": np.zeros(1250, np.int32), "second": np.zeros(1250, np.int32), "scales": np.zeros((20, 2), F32), "lr": np.array([0.1], F32),
         "step": np.array([3]), "scale": np.array([0.5], F32)}
    s = {k: tensor(backend, x) for k, x in a.items()}
    for k, dims, dtype in (("out", (2, 900, 136), DType.F16), ("final", (2, 136), DType.F32), ("states", (2, 57, 136), DType.F32), ("dx", (2, 900, 136), DType.F16),
                           ("dgate", (2, 900, 136), DType.F16), ("dstate", (2, 136), DType.F32), ("lp", (3,), DType.F32), ("ids", (3, 30), DType.I32), ("tops", (3, 30), DType.F32),
                           ("lp2", (400,), DType.F32), ("stats2", (400, 4), DType.F32), ("dz2", (400, 3000), DType.F16)):
        s[k] = DeviceTensor.empty(backend, dims, dtype)
    s["table"] = adamw_table([AdamWTensor(s["param"], s["grad"], s["first"], s["second"], scales=s["scales"])])
    return s


RESULTS = ("out", "final", "states", "dx", "dgate", "dstate", "lp", "ids", "tops", "lp2", "dz2", "param", "first", "second", "scales")


def operators(g, s):
    g.gated_recurrence(s["x"], s["gate"], s["out"], initial=s["state"], final=s["final"], states=s["states"])
    g.gated_recurrence_backward(s["x"], s["gate"], s["states"], out_grad=s["dout"], x_grad=s["dx"], gate_grad=s["dgate"], initial_grad=s["dstate"])
    g.token_logprobs(s["z"], s["tokens"], s["lp"], top_ids=s["ids"], top_logprobs=s["tops"])
    g.token_logprobs(s["z2"], s["tokens2"], s["lp2"], stats=s["stats2"])
    g.token_logprobs_backward(s["z2"], s["tokens2"], s["stats2"], s["dz2"], logprobs_grad=s["w"])
    g.adamw(s["table"], lr=s["lr"], step=s["step"], grad_scale=s["scale"], seed=9)


def test_captured_and_replayed(backend):
    """Two graphs replayed beside each other on streams of their own, eager calls between: the eager calls' bits after as many steps, with a rate that a copy changes on the way."""
    rt = runtime()
    problems, same = [problem(backend, seed) for seed in range(3)], [problem(backend, seed) for seed in range(3)]
    rates = [np.array([x], F32) for x in (0.1, 0.05, 0.2)]
    for rate in rates:
        for s in same:
            backend.copy_from_host(s["lr"].storage, 0, rate)
            operators(backend, s)
    want = [[s[k].numpy() for k in RESULTS] for s in same]
    graphs, streams = [], []
    for s in problems[:2]:
        backend.synchronize()
        graphs.append(capture(rt, backend.stream, lambda: operators(backend, s)))  # (nothing runs yet)
        stream = C.c_void_p()
        rt("cudaStreamCreateWithFlags", C.byref(stream), 1)
        streams.append(stream)
    for rate in rates:
        for s in problems:
            backend.copy_from_host(s["lr"].storage, 0, rate)
        backend.synchronize()
        for graph, stream in zip(graphs, streams):
            rt("cudaGraphLaunch", graph, stream)
        operators(backend, problems[2])
        for stream in streams:
            rt("cudaStreamSynchronize", stream)
        backend.synchronize()
    for s, w in zip(problems, want):
        for k, x in zip(RESULTS, w):
            assert np.array_equal(s[k].numpy(), x, equal_nan=x.dtype.kind == "f"), k
    for graph, stream in zip(graphs, streams):
        rt("cudaGraphExecDestroy", graph)
        rt("cudaStreamDestroy", stream)


def test_long_sequences_beside_each_other(backend):
    """Clusters of several graphs on the device at once, many windows each, a state that is carried on from replay to replay: the eager calls' bits."""
    rt = runtime()

    def prepared(seed):
        rng = np.random.default_rng(seed)
        length, width = (9300, 64) if seed % 2 else (7001, 33)
        s = {k: tensor(backend, rng.standard_normal((1, length, width)).astype(F16)) for k in ("x", "gate", "dout")}
        s["state"] = tensor(backend, rng.standard_normal((1, width)).astype(F32))
        for k, dims, dtype in (("out", (1, length, width), DType.F16), ("states", (1, -(-length // 16), width), DType.F32), ("dx", (1, length, width), DType.F16),
                               ("dgate", (1, length, width), DType.F16), ("dstate", (1, width), DType.F32)):
            s[k] = DeviceTensor.empty(backend, dims, dtype)
        return s

    def calls(s):
        backend.gated_recurrence(s["x"], s["gate"], s["out"], initial=s["state"], final=s["state"], states=s["states"])
        backend.gated_recurrence_backward(s["x"], s["gate"], s["states"], out_grad=s["dout"], x_grad=s["dx"], gate_grad=s["dgate"], initial_grad=s["dstate"])

    seeds, rounds = (0, 1, 2, 3), 4
    problems, same = [prepared(i) for i in seeds], [prepared(i) for i in seeds]
    for s in same:
        for _ in range(rounds):
            calls(s)
    backend.synchronize()
    graphs, streams = [], []
    for s in problems:
        graphs.append(capture(rt, backend.stream, lambda: calls(s)))
        stream = C.c_void_p()
        rt("cudaStreamCreateWithFlags", C.byref(stream), 1)
        streams.append(stream)
    for _ in range(rounds):
        for graph, stream in zip(graphs, streams):
            rt("cudaGraphLaunch", graph, stream)
    for stream in streams:
        rt("cudaStreamSynchronize", stream)
    for s, w in zip(problems, same):
        for k in ("out", "state", "states", "dx", "dgate", "dstate"):
            assert np.array_equal(s[k].numpy(), w[k].numpy()), k
    backend.synchronize()
    for graph, stream in zip(graphs, streams):
        rt("cudaGraphExecDestroy", graph)
        rt("cudaStreamDestroy", stream)


def test_two_threads_with_a_context_each():
    """Both begin at the same time; the bits are those of one after the other."""
    contexts = [B.Backend(0) for _ in range(2)]
    problems = [problem(c, 21) for c in contexts]
    start, errors = threading.Barrier(2), []

    def work(i):
        try:
            start.wait()
            for _ in range(20):
                operators(contexts[i], problems[i])
            contexts[i].synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    alone = problem(contexts[0], 21)
    for _ in range(20):
        operators(contexts[0], alone)
    for k in RESULTS:
        a, b, c = (s[k].numpy() for s in (*problems, alone))
        assert np.array_equal(a, b) and np.array_equal(a, c), k
    for c, s in zip(contexts, problems):
        for t in list(s.values()) + (list(alone.values()) if c is contexts[0] else []):
            if isinstance(t, DeviceTensor):
                t.storage.__del__()
        c.close()


def test_far_steps_and_rows(backend):
    """Steps and rows whose offsets pass 2^31 elements and 2^32 bytes."""
    step, n, d = 1 << 22, 1100, 96  # elements from one row to the next: 1100 rows reach over 4.6e9 elements
    storage, more = (backend.allocate((n * step + 2 * d) * 2) for _ in range(2))
    rng = np.random.default_rng(0)
    x, gate = rng.standard_normal((1, n, d)).astype(F16), (rng.standard_normal((1, n, d)) + 1).astype(F16)
    order = tensor(backend, np.arange(n))
    far_x, far_gate = (TensorDesc(storage.data + 2 * d * i, (n, d), (step * 2, 2), DType.F16) for i in range(2))
    far_out = TensorDesc(more.data, (n, d), (step * 2, 2), DType.F16)
    backend.embedding(tensor(backend, x[0]), order, far_x)
    backend.embedding(tensor(backend, gate[0]), order, far_gate)
    states, back = DeviceTensor.empty(backend, (-(-n // 16), d)), DeviceTensor.empty(backend, (n, d), DType.F16)
    backend.gated_recurrence(far_x, far_gate, far_out, states=states)
    backend.embedding(far_out, order, back)
    check(back.numpy()[None], *recurrence(x, gate, None, None, "sigmoid")["out"], F16, "out")
    dinitial = DeviceTensor.empty(backend, (d,))
    backend.gated_recurrence_backward(far_x, far_gate, states, out_grad=far_out, x_grad=far_x, gate_grad=far_gate, initial_grad=dinitial)  # over what they are computed from
    want = recurrence_backward(x, gate, None, None, "sigmoid", back.numpy()[None], None)
    got = DeviceTensor.empty(backend, (n, d), DType.F16)
    for far, name in ((far_x, "x"), (far_gate, "gate")):
        backend.embedding(far, order, got)
        check(got.numpy()[None], *want[name], F16, name)
    check(dinitial.numpy()[None], *want["initial"], F32, "initial")
    # rows of logits
    z, tokens = rng.standard_normal((n, d)).astype(F16), rng.integers(0, d, n)
    backend.embedding(tensor(backend, z), order, far_x)
    lp, stats, ids = DeviceTensor.empty(backend, (n,)), DeviceTensor.empty(backend, (n, 4)), DeviceTensor.empty(backend, (n, 7), DType.I32)
    backend.token_logprobs(far_x, tensor(backend, tokens), lp, stats=stats, top_ids=ids)
    want = logprobs(z, tokens, 1.0, 7)
    check(lp.numpy(), *want["logprobs"], F32, "logprobs")
    assert np.array_equal(ids.numpy(), want["top_ids"])
    ones = tensor(backend, np.ones(n, F32))
    backend.token_logprobs_backward(far_x, tensor(backend, tokens), stats, far_out, logprobs_grad=ones)
    dense = DeviceTensor.empty(backend, (n, d), DType.F16)
    backend.token_logprobs_backward(tensor(backend, z), tensor(backend, tokens), stats, dense, logprobs_grad=ones)
    backend.embedding(far_out, order, back)
    assert np.array_equal(back.numpy(), dense.numpy())


def test_profiles_name_the_calls(backend):
    s = problem(backend, 5)
    backend.set_profiling(True)
    operators(backend, s)
    names = [name for name, _ in backend.last_profile()]
    backend.set_profiling(False)
    assert names == ["gated_recurrence", "gated_recurrence_backward", "token_logprobs", "token_logprobs", "token_logprobs_backward", "adamw"]
