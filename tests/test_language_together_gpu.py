"""The language-model operators as a training step uses them: together, captured into a graph, beside other work, and on tensors that are larger than
32-bit offsets."""
import ctypes as C

import numpy as np
import pytest

import vkml_b200 as B
from language import EPS, Space, block_norm, block_norm_backward, check, column_sum, distill, embedding_backward
from vkml_b200 import DeviceTensor, NodeDesc, TensorDesc
from vkml_b200.graph import DType, Op

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


def tensor(backend, array):
    return DeviceTensor.from_host(backend, np.ascontiguousarray(array))


class Step:
    """A model of two blocks, trained by distillation: embedding -> (product, block norm) twice -> projection -> loss, and back to every parameter.
    The first block's input is the norm of the embedding; what a block adds passes its norm and gate."""

    vocab, width, batch, length, top = 301, 64, 3, 11, 5

    def __init__(self, backend, seed=0):
        rng = np.random.default_rng(seed)
        self.backend, n, d, v = backend, self.batch * self.length, self.width, self.vocab
        self.a = {"table": rng.standard_normal((v, d)) * 0.5, "ids": rng.integers(0, v, (self.batch, self.length)), "first": rng.standard_normal(d) * 0.1 + 1}
        for i in range(2):
            self.a.update({f"w{i}": rng.standard_normal((d, d)) / 8, f"post{i}": rng.standard_normal(d) * 0.1 + 1, f"gate{i}": rng.standard_normal((self.batch, d)) * 0.3 + 0.5,
                           f"pre{i}": rng.standard_normal(d) * 0.1 + 1})
        self.a.update({"teacher_ids": rng.integers(0, v, (n, self.top)).astype(np.int32), "teacher": rng.standard_normal((n, self.top)), "labels": rng.integers(0, v, n),
                       "weights": rng.random(n) + 0.5})
        self.a = {k: x.astype(F32) if x.dtype == np.float64 else x for k, x in self.a.items()}
        self.t = {k: tensor(backend, x) for k, x in self.a.items()}
        e = lambda *dims: DeviceTensor.empty(backend, dims)  # noqa: E731
        self.r = {"x": e(n, d), "n": [e(n, d) for _ in range(3)], "h": [e(n, d) for _ in range(2)], "y": [e(n, d) for _ in range(2)], "stats": [e(n, 4) for _ in range(3)],
                  "logits": e(n, v), "losses": e(n), "dlogits": e(n, v), "dn": [e(n, d) for _ in range(3)], "dh": [e(n, d) for _ in range(2)],
                  "dy": [e(n, d) for _ in range(2)], "dx": e(n, d), "dtable": e(v, d), "dtied": e(v, d), "dfirst": e(d),
                  **{f"d{k}{i}": e(*self.a[f"{k}{i}"].shape) for k in ("w", "post", "gate", "pre") for i in range(2)}}
        self.scratch = backend.allocate(1 << 22)

    def matmul(self, out, a, b):
        four = lambda t: TensorDesc(t.desc.data, (1, 1) + t.desc.dims, (0, 0) + t.desc.strides, t.desc.dtype)  # noqa: E731
        self.backend.compute([NodeDesc(int(Op.MATMUL), four(out), [four(a), four(b)])])

    def rows(self, t):
        d = t.desc
        return TensorDesc.contiguous(d.data, (self.batch, self.length) + d.dims[1:], d.dtype)

    def run(self):
        g, t, r, rows = self.backend, self.t, self.r, self.rows
        g.embedding(t["table"], t["ids"], rows(r["x"]), scale=8.0)
        g.block_norm(rows(r["x"]), None, normed=rows(r["n"][0]), stats=r["stats"][0], pre_weight=t["first"])
        h = r["x"]
        for i in range(2):
            self.matmul(r["y"][i], r["n"][i], t[f"w{i}"])
            g.block_norm(rows(h), rows(r["y"][i]), out=rows(r["h"][i]), normed=rows(r["n"][i + 1]), stats=r["stats"][i + 1], post_weight=t[f"post{i}"], gate=t[f"gate{i}"],
                         pre_weight=t[f"pre{i}"], branch_scale=0.7)
            h = r["h"][i]
        self.matmul(r["logits"], r["n"][2], t["table"].transpose(0, 1))  # the projection is tied to the embedding
        g.distill_loss(r["logits"], t["teacher_ids"], t["teacher"], r["losses"], labels=t["labels"], grad=r["dlogits"], losses_grad=t["weights"], temperature=2.0,
                       hard_weight=0.3)
        self.matmul(r["dn"][2], r["dlogits"], t["table"])
        self.matmul(r["dtied"], r["dlogits"].transpose(0, 1), r["n"][2])
        above = None
        for i in (1, 0):
            g.block_norm_backward(rows(r["h"][i]), rows(r["y"][i]), r["stats"][i + 1], out_grad=None if above is None else rows(above), normed_grad=rows(r["dn"][i + 1]),
                                  residual_grad=rows(r["dh"][i]), branch_grad=rows(r["dy"][i]), post_weight=t[f"post{i}"], gate=t[f"gate{i}"], pre_weight=t[f"pre{i}"],
                                  post_weight_grad=r[f"dpost{i}"], gate_grad=r[f"dgate{i}"], pre_weight_grad=r[f"dpre{i}"], branch_scale=0.7, workspace=self.scratch)
            above = r["dh"][i]
            self.matmul(r["dn"][i], r["dy"][i], t[f"w{i}"].transpose(0, 1))
            self.matmul(r[f"dw{i}"], r["n"][i].transpose(0, 1), r["dy"][i])
        g.block_norm_backward(rows(r["x"]), None, r["stats"][0], out_grad=rows(above), normed_grad=rows(r["dn"][0]), residual_grad=rows(r["dx"]), pre_weight=t["first"],
                              pre_weight_grad=r["dfirst"], workspace=self.scratch)
        # the table's gradient: the projection's, and the tokens' added to it
        g.copy_device_to_device([(r["dtable"].storage, 0, r["dtied"].storage, 0, r["dtied"].desc.nbytes)])
        g.embedding_backward(rows(r["dx"]), t["ids"], r["dtable"], scale=8.0, accumulate=True, workspace=self.scratch)

    NAMES = ["losses", "dtable", "dfirst"] + [f"d{k}{i}" for k in ("w", "post", "gate", "pre") for i in range(2)]

    def results(self):
        return {k: self.r[k].numpy() for k in self.NAMES}

    def loss(self, a):
        """The weighted sum of the losses in 64 bits, of parameters `a`."""
        a = {k: x.astype(np.float64) if x.dtype == F32 else x for k, x in a.items()}
        norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)  # noqa: E731
        h = 8.0 * a["table"][a["ids"]]
        n = norm(h) * a["first"]
        for i in range(2):
            h = h + 0.7 * a[f"gate{i}"][:, None, :] * norm(n @ a[f"w{i}"]) * a[f"post{i}"]
            n = norm(h) * a[f"pre{i}"]
        z = (n @ a["table"].T).reshape(-1, self.vocab)
        soft = lambda x: x - x.max(-1, keepdims=True) - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))  # noqa: E731
        log_p, log_q = soft(a["teacher"] / 2.0), soft(z / 2.0)
        kd = 4.0 * (np.exp(log_p) * (log_p - np.take_along_axis(log_q, a["teacher_ids"].astype(np.int64), 1))).sum(-1)
        ce = -soft(z)[np.arange(len(z)), a["labels"]]
        losses = 0.7 * kd + 0.3 * ce
        return losses, (losses * a["weights"]).sum()


def test_a_training_step(backend):
    """Losses against the model in 64 bits, every parameter's gradient against its differences there: along a random direction of a whole parameter the central
    difference with step 1e-4 is off by its third-order term, below 1e-6 of the value here, and the kernels by the products' error (4e-6 relative at these sizes, through
    two layers and their norms): 2e-4 of the gradient's and the direction's lengths holds both."""
    step = Step(backend)
    step.run()
    got = step.results()
    losses, _ = step.loss(step.a)
    assert np.allclose(got["losses"], losses, rtol=1e-4, atol=1e-4)
    rng = np.random.default_rng(1)
    for name in step.NAMES[1:]:
        of = name[1:]
        direction = rng.standard_normal(step.a[of].shape)
        value = []
        for sign in (1e-4, -1e-4):
            a = {k: x.astype(np.float64) if x.dtype == F32 else x for k, x in step.a.items()}
            a[of] = a[of] + sign * direction
            value.append(step.loss(a)[1])
        want = (value[0] - value[1]) / 2e-4
        size = np.linalg.norm(got[name].astype(np.float64)) * np.linalg.norm(direction)
        assert abs((got[name].astype(np.float64) * direction).sum() - want) <= 2e-4 * size, name


def test_the_same_bits_again_and_between_other_work(backend):
    step, other = Step(backend), Step(backend, 1)
    step.run()
    first = step.results()
    for _ in range(2):
        other.run()
        step.run()
        other.run()
    for k, x in step.results().items():
        assert np.array_equal(x, first[k]), k


@pytest.mark.parametrize("large,small", [(1000, 320), (4096, 264), (8192, 4104), (16384, 8200)])
def test_a_size_again_after_a_smaller_one(backend, large, small):
    """The widths, and the numbers of a teacher's entries, in turn: what a kernel was allowed for a size holds when the size comes back."""
    rng = np.random.default_rng(large)

    def norms(width, kind):
        a = {k: rng0.standard_normal((5, width)).astype(F32) for k in ("h", "y", "dout", "dn")}
        t = {k: tensor(backend, x) for k, x in a.items()}
        t.update({k: DeviceTensor.empty(backend, (5, width)) for k in ("out", "normed", "dh", "dy")}, stats=DeviceTensor.empty(backend, (5, 4)), dw=DeviceTensor.empty(backend, (width,)))
        backend.block_norm(t["h"], t["y"], out=t["out"], normed=t["normed"], stats=t["stats"], kind=kind)
        backend.block_norm_backward(t["out"], t["y"], t["stats"], out_grad=t["dout"], normed_grad=t["dn"], residual_grad=t["dh"], branch_grad=t["dy"], pre_weight_grad=t["dw"],
                                    kind=kind)
        return [t[k].numpy() for k in ("out", "normed", "dh", "dy", "dw")]

    logits = tensor(backend, rng.standard_normal((300, 16384)).astype(F16))

    def distilled(top):
        ids, teacher = tensor(backend, rng0.integers(0, 16384, (300, top))), tensor(backend, rng0.standard_normal((300, top)).astype(F32))
        losses, stats, grad, again = (DeviceTensor.empty(backend, s, d) for s, d in (((300,), DType.F32), ((300, 4), DType.F32), ((300, 16384), DType.F16), ((300, 16384), DType.F16)))
        backend.distill_loss(logits, ids, teacher, losses, stats=stats, temperature=2.0)
        backend.distill_loss(logits, ids, teacher, losses, stats=stats, grad=grad, temperature=2.0)
        backend.distill_loss_backward(logits, ids, teacher, stats, again, temperature=2.0)
        return [x.numpy() for x in (losses, stats, grad, again)]

    results = []
    for width in (large, small, large):
        rng0 = np.random.default_rng(width)
        results.append(norms(width, "rms") + norms(width, "layer") + distilled(min(1024, width // 16)))
    for x, y in zip(results[0], results[2]):
        assert np.array_equal(x, y)


class Runtime:
    """The few calls of the CUDA runtime that capture and launch a graph."""

    def __init__(self):
        self.lib = C.CDLL("libcudart.so.12")

    def __call__(self, name, *args):
        assert getattr(self.lib, name)(*args) == 0, name


def runtime():
    try:
        return Runtime()
    except OSError:
        pytest.skip("no shared CUDA runtime to capture with")


def capture(rt, stream, calls):
    rt("cudaStreamBeginCapture", C.c_void_p(stream), 2)
    calls()
    graph, execution = C.c_void_p(), C.c_void_p()
    rt("cudaStreamEndCapture", C.c_void_p(stream), C.byref(graph))
    rt("cudaGraphInstantiate", C.byref(execution), graph, 0)
    return execution


def operators(g, s, workspace):
    """Calls whose scratch matters: sorted tokens, sums over rows."""
    g.embedding_backward(s["rows"], s["ids"], s["table"], workspace=workspace)
    g.block_norm_backward(s["out"], s["branch"], s["stats"], out_grad=s["rows"], normed_grad=s["normed_grad"], residual_grad=s["dh"], branch_grad=s["dy"], pre_weight=s["w"],
                          pre_weight_grad=s["dw"], post_weight=s["w"], post_weight_grad=s["dw2"], gate=s["w"], gate_grad=s["dgate"], workspace=workspace)


def scratch_problem(backend, seed):
    rng = np.random.default_rng(seed)
    n, d, v = 3000, 320, 5000
    a = {k: rng.standard_normal((n, d)).astype(F32) for k in ("rows", "out", "branch", "normed_grad")}
    a.update({"stats": np.abs(rng.standard_normal((n, 4))).astype(F32) + 1, "w": rng.standard_normal(d).astype(F32), "ids": rng.integers(0, v, n)})
    s = {k: tensor(backend, x) for k, x in a.items()}
    s.update({"table": DeviceTensor.empty(backend, (v, d)), "dh": DeviceTensor.empty(backend, (n, d)), "dy": DeviceTensor.empty(backend, (n, d)),
              **{k: DeviceTensor.empty(backend, (d,)) for k in ("dw", "dw2", "dgate")}})
    return s


RESULTS = ("table", "dh", "dy", "dw", "dw2", "dgate")


def test_captured_and_replayed(backend):
    """Two graphs with a workspace each, replayed beside each other on streams of their own, and an eager call between: the eager calls' bits."""
    rt = runtime()
    problems = [scratch_problem(backend, seed) for seed in range(3)]
    want = []
    for s in problems:
        operators(backend, s, None)
        want.append([s[k].numpy() for k in RESULTS])
    graphs, streams = [], []
    for s in problems[:2]:
        workspace = backend.allocate(1 << 24)
        backend.synchronize()
        graphs.append((capture(rt, backend.stream, lambda: operators(backend, s, workspace)), workspace))
        stream = C.c_void_p()
        rt("cudaStreamCreateWithFlags", C.byref(stream), 1)
        streams.append(stream)
    zeros = {k: np.zeros(problems[0][k].desc.dims, F32) for k in RESULTS}
    for s in problems:
        for k in RESULTS:
            backend.copy_from_host(s[k].storage, 0, zeros[k])
    backend.synchronize()
    for _ in range(5):
        for (graph, _), stream in zip(graphs, streams):
            rt("cudaGraphLaunch", graph, stream)
        operators(backend, problems[2], None)
    for stream in streams:
        rt("cudaStreamSynchronize", stream)
    for s, w in zip(problems, want):
        for k, x in zip(RESULTS, w):
            assert np.array_equal(s[k].numpy(), x), k
    for (graph, _), stream in zip(graphs, streams):
        rt("cudaGraphExecDestroy", graph)
        rt("cudaStreamDestroy", stream)


def test_scratch_does_not_grow_under_capture():
    """A call that would have to grow the context's scratch is refused, and the context works on."""
    rt = runtime()
    backend = B.Backend(0)
    n, d, v = 3000, 1024, 9000  # 50 MB of scratch: more than a context begins with
    rows, ids, table = DeviceTensor.empty(backend, (n, d)), tensor(backend, np.arange(n) % v), DeviceTensor.empty(backend, (v, d))
    need = backend.embedding_backward_workspace(rows, ids, table)
    refused = []

    def call():
        try:
            backend.embedding_backward(rows, ids, table)
        except ValueError as e:
            refused.append(str(e))

    assert need > 0
    backend.synchronize()
    execution = capture(rt, backend.stream, call)
    assert refused and "workspace" in refused[0]
    rt("cudaGraphExecDestroy", execution)
    backend.embedding_backward(rows, ids, table)
    backend.synchronize()
    with pytest.raises(ValueError):  # too small, and not aligned
        backend.embedding_backward(rows, ids, table, workspace=backend.allocate(need - 256))
    backend.synchronize()
    backend.close()


def test_two_contexts(backend):
    """Contexts have streams and scratch of their own."""
    second = B.Backend(0)
    a, b = scratch_problem(backend, 7), scratch_problem(second, 7)
    for _ in range(3):
        operators(backend, a, None)
        operators(second, b, None)
    for k in RESULTS:
        assert np.array_equal(a[k].numpy(), b[k].numpy()), k
    for t in b.values():
        t.storage.__del__()
    second.close()


def test_far_rows(backend):
    """Rows, tables and logits whose offsets pass 2^31 elements and 2^32 bytes."""
    step = 1 << 22  # elements from one row to the next: 1100 rows reach over 4.6e9 elements
    n, d = 1100, 96
    storage = backend.allocate((n * step + d) * 2)
    far = TensorDesc(storage.data, (n, d), (step * 2, 2), DType.F16)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((n, d)).astype(F16)
    ids = rng.permutation(n).astype(np.int64)
    dense, index = tensor(backend, x), tensor(backend, ids)
    back = DeviceTensor.empty(backend, (n, d), DType.F16)
    backend.embedding(dense, index, far)                      # far rows written
    backend.embedding(far, index, back)                       # a far table read
    assert np.array_equal(back.numpy(), x[ids][ids])
    table = DeviceTensor.empty(backend, (n, d), DType.F32)
    backend.embedding_backward(far, index, table)             # far rows summed: one to each id
    assert np.array_equal(table.numpy()[ids], x[ids].astype(F32))
    backend.embedding_backward(dense, index, far)             # a far table written: more tokens than blocks that own rows
    backend.embedding(far, index, back)
    assert np.array_equal(back.numpy(), x)
    normed = DeviceTensor.empty(backend, (n, d), DType.F16)
    h = x[np.argsort(ids)]
    backend.block_norm(far, None, normed=normed.desc, kind="layer")
    check(normed.numpy(), *block_norm(h, None, {}, 1.0, 1.0, True, 1e-5, False)["normed"], F16, "normed")
    backend.block_norm(normed.desc, None, out=far, kind="layer")
    backend.embedding(far, tensor(backend, np.arange(n)), back)
    assert np.array_equal(back.numpy(), normed.numpy())
    k, t = np.zeros((n, 1), np.int32), np.zeros((n, 1), F32)
    losses, stats, grad = DeviceTensor.empty(backend, (n,)), DeviceTensor.empty(backend, (n, 4)), DeviceTensor.empty(backend, (n, d), DType.F16)
    want = distill(normed.numpy()[-3:], k[-3:], t[-3:], None, None, 1.0, 0.0, 1.0)
    backend.distill_loss(far, tensor(backend, k), tensor(backend, t), losses, stats=stats, grad=grad)
    check(losses.numpy()[-3:], *want["losses"], F32, "losses")
    check(grad.numpy()[-3:], *want["grad"], F16, "gradient")
    backend.distill_loss_backward(far, tensor(backend, k), tensor(backend, t), stats, far)  # over the logits
    backend.embedding(far, tensor(backend, np.arange(n)), back)
    check(back.numpy()[-3:], *want["grad"], F16, "gradient")


def test_many_far_rows_of_logits(backend):
    """The kernel of many rows with offsets past 2^31 elements."""
    rows, vocab, step = 520, 17000, 1 << 23
    storage = backend.allocate((rows * step + vocab) * 2)
    far = TensorDesc(storage.data, (rows, vocab), (step * 2, 2), DType.F16)
    rng = np.random.default_rng(1)
    z = rng.standard_normal((rows, vocab), dtype=F32).astype(F16)
    backend.embedding(tensor(backend, z), tensor(backend, np.arange(rows)), far)
    k, t = rng.integers(0, vocab, (rows, 7)), rng.standard_normal((rows, 7)).astype(F32)
    losses, grad = DeviceTensor.empty(backend, (rows,)), DeviceTensor.empty(backend, (rows, vocab), DType.F16)
    backend.distill_loss(far, tensor(backend, k), tensor(backend, t), losses, grad=grad, grad_scale=64.0)
    some = np.array([0, 300, rows - 1])
    want = distill(z[some], k[some], t[some], None, None, 1.0, 0.0, 64.0)
    check(losses.numpy()[some], *want["losses"], F32, "losses")
    check(grad.numpy()[some], *want["grad"], F16, "gradient")
