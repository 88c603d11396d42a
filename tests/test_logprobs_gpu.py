"""Token log probabilities, entropies, the likeliest tokens and the gradient against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import Space, check, placed, rows_view
from language_steps import logprobs, logprobs_backward

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


def nan(shape, dtype=F32):
    return np.full(shape, np.nan, dtype)


def forward(backend, z, tokens, temperature=1.0, top=0, ids=np.int32, layout="dense"):
    """(logprobs, entropies, stats, top ids, top logprobs) as flat rows."""
    rows, lead = int(np.prod(z.shape[:-1])), z.shape[:-1]
    space = Space(backend)
    put = space.put
    lp, h, stats = nan(lead) if tokens is not None else None, nan(lead), nan((rows, 4))
    top_ids, tops = (rows_view(lead + (top,), ids, layout), rows_view(lead + (top,), F32, layout)) if top else (None, None)
    backend.token_logprobs(put(z), put(tokens), put(lp), entropies=put(h), stats=put(stats), top_ids=put(top_ids), top_logprobs=put(tops), temperature=temperature)
    got = []
    for view, shape in ((lp, (rows,)), (h, (rows,)), (stats, (rows, 4)), (top_ids, (rows, top)), (tops, (rows, top))):
        if view is None:
            got.append(None)
            continue
        x, rest = space.get(view)
        assert rest
        got.append(x.reshape(shape))
    return got


def compare(got, z, tokens, temperature, top, some=None):
    flat, rows = np.ascontiguousarray(z).reshape(-1, z.shape[-1]), int(np.prod(z.shape[:-1]))
    some = np.arange(rows) if some is None else some
    want = logprobs(flat[some], None if tokens is None else np.ascontiguousarray(tokens).reshape(-1)[some], temperature, top)
    lp, h, stats, ids, tops = got
    if tokens is not None:
        check(lp[some], *want["logprobs"], F32, "logprobs")
    check(h[some], *want["entropies"], F32, "entropies")
    check(stats[some], *want["stats"], F32, "stats")
    if top:
        assert np.array_equal(ids[some], want["top_ids"])
        check(tops[some], *want["top_logprobs"], F32, "top_logprobs")


SHAPES = [((1, 1), 1, "dense", 1.0), ((3, 7), 7, "dense", 1.0), ((16, 1000), 5, "dense", 1.0), ((2, 3, 33), 20, "odd", 2.0), ((2, 5, 4097), 64, "offset", 0.7), ((4, 2, 1024), 128, "swapped", 0.5),
          ((3, 8000), 100, "pitch", 1.5), ((5, 32000), 50, "dense", 2.0), ((2, 50001), 17, "dense", 1.0), ((2, 2, 100000), 33, "odd", 3.0), ((2, 300007), 5, "dense", 1.0),
          ((300, 517), 3, "dense", 1.0), ((2, 128000), 128, "pitch", 2.0), ((700, 128), 128, "dense", 1.0), ((3, 1030), 128, "offset", 1.0), ((64, 16384), 1, "dense", 1.0),
          ((600, 9000), 30, "backwards", 1.0)]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shape,top,layout,temperature", SHAPES)
def test_log_probabilities_and_gradient(backend, dtype, shape, top, layout, temperature):
    rng = np.random.default_rng(shape[-1] + top)
    z = (rng.standard_normal(shape, dtype=F32) * 2.5).astype(dtype)
    lead, rows = shape[:-1], int(np.prod(shape[:-1]))
    tokens = rng.integers(0, shape[-1], lead).astype(np.int32 if layout == "odd" else np.int64)
    tokens.reshape(-1)[rows // 2] = -1 if rows > 2 else tokens.reshape(-1)[rows // 2]
    some = np.unique(np.concatenate([[0, rows // 2, rows - 1], rng.integers(0, rows, 8)])) if rows * shape[-1] > 1 << 18 else np.arange(rows)
    z = placed(z, layout)
    got = forward(backend, z, tokens, temperature, top, np.int64 if layout == "pitch" else np.int32, layout)
    compare(got, z, tokens, temperature, top, some)
    backend.synchronize()
    ulp, uh = (rng.standard_normal(lead) * 8).astype(F32), rng.standard_normal(lead).astype(F32)
    ulp.reshape(-1)[0], uh.reshape(-1)[0] = (0, 0) if rows > 1 else (1, 1)
    space = Space(backend)
    put = space.put
    grad = rows_view(shape, dtype, layout)
    backend.token_logprobs_backward(put(z), put(tokens), put(got[2]), put(grad), logprobs_grad=put(ulp), entropies_grad=put(uh), temperature=temperature, grad_scale=4.0)
    g, rest = space.get(grad)
    assert rest
    flat = lambda x: np.ascontiguousarray(x).reshape(rows, -1)[some]  # noqa: E731
    want = logprobs_backward(flat(z), flat(tokens)[:, 0], got[2][some], flat(ulp)[:, 0], flat(uh)[:, 0], temperature, 4.0)
    check(flat(g), *want, dtype, "gradient")
    assert np.isfinite(g).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab,top", [(40, 10), (1000, 20), (9000, 128), (40001, 33)])
def test_forbidden_and_equal_logits(backend, dtype, vocab, top):
    """Rows of few values and of forbidden columns: fewer left than are wanted, one left, none left, all alike, two values, the lowest finite value, rising and falling."""
    rng = np.random.default_rng(vocab)
    z = rng.standard_normal((16, vocab)).astype(dtype)
    few = rng.permutation(vocab)[:max(1, top // 3)]
    mask = np.ones(vocab, bool)
    mask[few] = False
    z[0, mask] = -np.inf
    z[1] = -np.inf
    z[1, vocab // 2] = 3
    z[2] = -np.inf
    z[3] = 1.5
    z[4] = np.where(rng.random(vocab) < 0.5, 2.0, -2.0)
    z[5, mask] = np.finfo(dtype).min
    z[6] = np.finfo(dtype).min
    z[7] = np.linspace(-4, 4, vocab).astype(dtype)
    z[8] = np.linspace(4, -4, vocab).astype(dtype)
    z[9] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    z[10, : vocab // 2] = -np.inf
    z[11] = np.round(z[11])
    z[12] = 0
    z[12, vocab - top:] = 1
    z[13] = 100 * z[13]
    z[14, 5:9] = 7
    z[15] = np.finfo(dtype).max
    tokens = rng.integers(0, vocab, 16)
    tokens[0], tokens[1] = few[0], vocab // 2
    got = forward(backend, z, tokens, 1.0, top)
    compare(got, z, tokens, 1.0, top)
    ulp, uh = (rng.standard_normal(16) + 3).astype(F32), (rng.standard_normal(16) + 3).astype(F32)
    space = Space(backend)
    grad = nan(z.shape, dtype)
    backend.token_logprobs_backward(space.put(z), space.put(tokens), space.put(got[2]), space.put(grad), logprobs_grad=space.put(ulp), entropies_grad=space.put(uh))
    check(space.get(grad)[0], *logprobs_backward(z, tokens, got[2], ulp, uh, 1.0, 1.0), dtype, "gradient")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("size,temperature", [(30, 1.0), (30, 0.02), (30000, 0.2), (30000, 400.0), (0.01, 1e-3), (5, 1e30)])
def test_rows_that_rise(backend, dtype, size, temperature):
    """Each stretch's largest logit above the last one's, from far below or far above zero; and the other way round."""
    vocab = 40003
    rng = np.random.default_rng(3)
    z = np.linspace(-size, size, vocab) + rng.standard_normal((6, vocab)) * size / 50
    z[1::2] = z[1::2, ::-1]
    z[2:4] += size
    z[4:] -= size
    z = z.astype(dtype)
    tokens = z.astype(F32).argmax(1)
    tokens[0] = 17
    got = forward(backend, z, tokens, temperature, 5)
    compare(got, z, tokens, temperature, 5)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab,top,layout", [(160, 9001, 0, "offset"), (160, 9001, 20, "dense"), (400, 5000, 128, "dense"), (700, 2600, 7, "odd"), (149, 70000, 3, "dense")])
def test_rows_that_leave_room(backend, dtype, rows, vocab, top, layout):
    """More rows than SMs and fewer than the device holds blocks of a few warps."""
    rng = np.random.default_rng(rows + top)
    z = placed((rng.standard_normal((rows, vocab), dtype=F32) * 2.5).astype(dtype), layout)
    tokens = rng.integers(0, vocab, rows)
    some = np.unique(np.concatenate([[0, 147, 148, rows - 1], rng.integers(0, rows, 8)]))
    compare(forward(backend, z, tokens, 1.0, top, layout=layout), z, tokens, 1.0, top, some)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab", [9, 3000, 70001])
def test_rows_that_hold_no_numbers(backend, dtype, vocab):
    """+inf and not-a-number: no numbers where the formulas have none, the neighbours untouched, the top in order."""
    rng = np.random.default_rng(vocab)
    z = rng.standard_normal((5, vocab)).astype(dtype)
    z[1, 4], z[2, vocab - 1], z[3, 0], z[3, 5] = np.inf, np.nan, np.nan, np.inf
    got = forward(backend, z, np.arange(5), 1.0, 6)
    want = logprobs(z, np.arange(5), 1.0, 6)
    assert np.array_equal(got[3], want["top_ids"])
    good = np.array([0, 4])
    compare([g[good] for g in got], z[good], np.arange(5)[good], 1.0, 6)
    for r in (1, 2, 3):
        assert np.isnan(got[0][r]) and np.isnan(got[1][r]) and np.isnan(got[4][r]).all()
    # rows whose gradients are zero have zeros, whatever they hold
    weight = np.array([1, 0, 0, 0, 1], F32)
    space = Space(backend)
    grad = nan(z.shape, dtype)
    backend.token_logprobs_backward(space.put(z), space.put(np.arange(5)), space.put(got[2]), space.put(grad), logprobs_grad=space.put(weight))
    g = space.get(grad)[0]
    assert not g[1:4].any() and np.isfinite(g).all() and g[0].any()


def test_tokens_that_are_none_or_outside(backend):
    rng = np.random.default_rng(1)
    z = rng.standard_normal((6, 50)).astype(F32)
    tokens = np.array([-1, -(1 << 62), 50, 1 << 40, 49, 0])
    space = Space(backend)
    lp, stats, grad = nan((6,)), nan((6, 4)), nan((6, 50))
    backend.token_logprobs(space.put(z), space.put(tokens), space.put(lp), stats=space.put(stats))
    with pytest.raises(IndexError):
        backend.synchronize()
    got, got_stats = space.get(lp)[0], space.get(stats)[0]
    assert not got[:4].any() and got[4:].all()
    weight = np.ones(6, F32)
    backend.token_logprobs_backward(space.put(z), space.put(tokens), space.put(got_stats), space.put(grad), logprobs_grad=space.put(weight))
    with pytest.raises(IndexError):
        backend.synchronize()
    g = space.get(grad)[0]
    assert not g[:4].any()
    check(g, *logprobs_backward(z, tokens, got_stats, weight, None, 1.0, 1.0), F32, "gradient")
    backend.synchronize()


@pytest.mark.parametrize("shape", [(4, 100), (2, 40000), (3, 130001), (300, 5001)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_gradient_over_the_logits(backend, shape, dtype):
    rng = np.random.default_rng(2)
    z, tokens = rng.standard_normal(shape).astype(dtype), rng.integers(0, shape[-1], shape[0])
    stats = forward(backend, z, tokens)[2]
    ulp, uh = np.full(shape[0], 5, F32), np.full(shape[0], 0.5, F32)
    results = []
    for grad in (nan(shape, dtype), z):
        space = Space(backend)
        backend.token_logprobs_backward(space.put(z), space.put(tokens), space.put(stats), space.put(grad), logprobs_grad=space.put(ulp), entropies_grad=space.put(uh))
        results.append(space.get(grad)[0])
    assert np.array_equal(*results)


def test_gradients_by_one_of_the_two(backend):
    """Of log probabilities alone, of entropies alone, of a number for all rows."""
    rng = np.random.default_rng(3)
    z, tokens = rng.standard_normal((7, 777)).astype(F32), rng.integers(0, 777, 7)
    stats = forward(backend, z, tokens)[2]
    one, every = np.array([2.0], F32), np.broadcast_to(np.array([2.0], F32), (7,))
    for ulp, uh in ((every, None), (None, every), (every, every)):
        space = Space(backend)
        grad = nan(z.shape)
        put = lambda t: None if t is None else space.put(t)  # noqa: E731
        backend.token_logprobs_backward(space.put(z), space.put(tokens), space.put(stats), space.put(grad), logprobs_grad=put(ulp), entropies_grad=put(uh))
        check(space.get(grad)[0], *logprobs_backward(z, tokens, stats, ulp, uh, 1.0, 1.0), F32, "gradient")
    space = Space(backend)
    grad = nan(z.shape)
    backend.token_logprobs_backward(space.put(z), None, space.put(stats), space.put(grad), entropies_grad=space.put(np.repeat(one, 7)))
    check(space.get(grad)[0], *logprobs_backward(z, None, stats, None, np.repeat(one, 7), 1.0, 1.0), F32, "gradient without tokens")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shift", [1e4, -3e4])
def test_logits_far_from_zero(backend, dtype, shift):
    rng = np.random.default_rng(4)
    z = (rng.standard_normal((20, 3001)) * 30 + shift).astype(dtype)
    tokens = z.argmax(1)
    got = forward(backend, z, tokens, 0.9, 9)
    compare(got, z, tokens, 0.9, 9)


def test_each_result_alone(backend):
    """Within the bounds that hold it beside the others.  (Not the same bits: how many threads share a row goes by the entries that are wanted, and sums by the threads.)"""
    rng = np.random.default_rng(5)
    z, tokens = rng.standard_normal((9, 2222)).astype(F16), rng.integers(0, 2222, 9)
    want = logprobs(z, tokens, 1.3, 40)
    for name, view in {"logprobs": nan((9,)), "entropies": nan((9,)), "stats": nan((9, 4)), "top_ids": np.zeros((9, 40), np.int32), "top_logprobs": nan((9, 40))}.items():
        space = Space(backend)
        backend.token_logprobs(space.put(z), space.put(tokens), **{name: space.put(view)}, temperature=1.3)
        got = space.get(view)[0]
        if name == "top_ids":
            assert np.array_equal(got, want[name])
        else:
            check(got, *want[name], F32, name)


def test_a_teachers_entries(backend):
    """What token_logprobs finds is what distill_loss reads: distilling a model from its own whole distribution has no loss and no gradient."""
    rng = np.random.default_rng(6)
    z = rng.standard_normal((33, 100)).astype(F32)
    space = Space(backend)
    put = space.put
    ids, tops, losses, grad = np.zeros((33, 100), np.int64), nan((33, 100)), nan((33,)), nan((33, 100))
    backend.token_logprobs(put(z), top_ids=put(ids), top_logprobs=put(tops))
    backend.distill_loss(put(z), put(ids), put(tops), put(losses), grad=put(grad))
    # both distributions' logarithms are off by 2^-20 at most
    assert np.abs(space.get(losses)[0]).max() < 2.0 ** -18 and np.abs(space.get(grad)[0]).max() < 2.0 ** -18


@pytest.mark.parametrize("rows,vocab", [(1, 128000), (40, 50000), (2000, 3000), (5000, 64)])
def test_the_same_bits_again(backend, rows, vocab):
    rng = np.random.default_rng(7)
    z, tokens = (rng.standard_normal((rows, vocab), dtype=F32) * 2).astype(F16), rng.integers(0, vocab, rows)
    first = forward(backend, z, tokens, 1.0, 25)
    for _ in range(3):
        for a, b in zip(forward(backend, z, tokens, 1.0, 25), first):
            assert np.array_equal(a, b)


def test_no_rows(backend):
    z = np.zeros((0, 10), F32)
    space = Space(backend)
    put = space.put
    backend.token_logprobs(put(z), put(np.zeros((0,), np.int64)), put(nan((0,))), top_ids=put(np.zeros((0, 3), np.int32)))
    backend.token_logprobs_backward(put(z), put(np.zeros((0,), np.int64)), put(nan((0, 4))), put(z.copy()))
    z = np.ones((4, 10), F32)  # no top
    h = nan((4,))
    backend.token_logprobs(put(z), entropies=put(h), top_ids=put(np.zeros((4, 0), np.int32)))
    assert np.abs(space.get(h)[0] - np.log(10)).max() < 1e-6
