"""Distillation losses and gradients against plain formulas in 64 bits."""
import numpy as np
import pytest

from language import EPS, Space, check, distill, placed, rows_view

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


def problem(rng, shape, top, dtype, ids=np.int32):
    rows, vocab = int(np.prod(shape[:-1])), shape[-1]
    teacher = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
    k = (np.argpartition(-teacher, top - 1, 1) if top < vocab else np.argsort(-teacher, 1))[:, :top].astype(ids)
    t = np.take_along_axis(teacher, k.astype(np.int64), 1).astype(dtype)
    z = (teacher * 0.6 + rng.standard_normal((rows, vocab), dtype=np.float32)).astype(dtype)
    return z.reshape(shape), k.reshape(shape[:-1] + (top,)), t.reshape(shape[:-1] + (top,))


def run(backend, z, k, t, labels, weights, temperature, hard, scale, layout="dense", in_place=False, some=None):
    """Losses, stats and gradient at once; the losses alone; the gradient alone: each against the formulas in the rows `some` (all)."""
    rows, vocab = int(np.prod(z.shape[:-1])), z.shape[-1]
    lead = z.shape[:-1]
    some = np.arange(rows) if some is None else some
    flat = lambda x, *shape: None if x is None else np.ascontiguousarray(x).reshape(rows, *shape)[some]  # noqa: E731
    given = flat(z, vocab), flat(k, -1), flat(t, -1), flat(labels), flat(weights), temperature, hard, scale
    want = distill(*given)
    options = dict(temperature=temperature, hard_weight=hard, grad_scale=scale)
    space = Space(backend)
    put = space.put
    losses, stats = np.full(lead, np.nan, F32), np.full((rows, 4), np.nan, F32)
    grad = z if in_place else rows_view(z.shape, z.dtype.type, layout)
    backend.distill_loss(put(z), put(k), put(t), put(losses), labels=put(labels), stats=put(stats), grad=put(grad), losses_grad=put(weights), **options)
    got, rest = space.get(grad)
    assert rest
    check(got.reshape(rows, vocab)[some], *want["grad"], z.dtype.type, "gradient with the losses")
    check(space.get(losses)[0].reshape(-1)[some], *want["losses"], F32, "losses")
    got_stats = space.get(stats)[0]
    check(got_stats[some], *want["stats"], F32, "stats")
    space = Space(backend)
    put = space.put
    losses2, stats2 = np.full(lead, np.nan, F32), np.full((rows, 4), np.nan, F32)
    backend.distill_loss(put(z), put(k), put(t), put(losses2), labels=put(labels), stats=put(stats2), **options)
    check(space.get(losses2)[0].reshape(-1)[some], *want["losses"], F32, "losses alone")
    check(space.get(stats2)[0][some], *want["stats"], F32, "stats alone")
    space = Space(backend)
    put = space.put
    grad = z if in_place else rows_view(z.shape, z.dtype.type, layout)
    backend.distill_loss_backward(put(z), put(k), put(t), put(got_stats), put(grad), labels=put(labels), losses_grad=put(weights), **options)
    want = distill(*given, got_stats[some])
    got, rest = space.get(grad)
    assert rest
    check(got.reshape(rows, vocab)[some], *want["grad"], z.dtype.type, "gradient alone")
    return got


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shape,top,layout,temperature,hard", [
    ((1, 1), 1, "dense", 1.0, 0.0), ((3, 7), 7, "dense", 1.0, 0.5), ((16, 1000), 8, "dense", 1.0, 0.5), ((2, 3, 33), 5, "odd", 2.0, 0.0),
    ((2, 5, 4097), 64, "offset", 4.0, 0.1), ((4, 2, 1024), 100, "swapped", 0.5, 1.0), ((3, 8000), 1024, "pitch", 1.5, 0.25), ((5, 32000), 50, "dense", 2.0, 0.0),
    ((2, 50001), 17, "dense", 1.0, 0.9), ((2, 2, 100000), 33, "odd", 3.0, 0.3), ((2, 300007), 5, "dense", 1.0, 0.0), ((300, 517), 3, "dense", 1.0, 0.5),
    ((2, 128000), 200, "pitch", 2.0, 0.5)])
def test_losses_and_gradient(backend, dtype, shape, top, layout, temperature, hard):
    rng = np.random.default_rng(shape[-1] + top)
    z, k, t = problem(rng, shape, top, dtype, np.int64 if layout == "pitch" else np.int32)
    lead = shape[:-1]
    labels = rng.integers(0, shape[-1], lead).astype(np.int32 if layout == "odd" else np.int64) if hard else None
    weights = (rng.random(lead) * 8 + 1).astype(F32)
    weights.reshape(-1)[0] = 0 if weights.size > 1 else 1
    run(backend, placed(z, layout), placed(k, layout), placed(t, layout), labels, weights, temperature, hard, 4.0, layout)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shape,top,layout,temperature,hard", [
    ((300, 16384), 8, "dense", 1.0, 0.5), ((150, 2, 17001), 33, "odd", 2.0, 0.0), ((297, 32768), 64, "dense", 1.0, 0.0), ((301, 40003), 5, "offset", 2.0, 0.3),
    ((2, 150, 52000), 100, "swapped", 1.5, 1.0), ((320, 98304), 3, "dense", 1.0, 0.1), ((299, 99001), 40, "pitch", 2.0, 0.5)])
def test_many_rows(backend, dtype, shape, top, layout, temperature, hard):
    """More rows than blocks: every row's sums, loss and columns are its own."""
    rng = np.random.default_rng(shape[-1])
    rows, vocab = int(np.prod(shape[:-1])), shape[-1]
    z = rng.standard_normal(shape, dtype=np.float32).astype(dtype) * dtype(2)
    k = rng.integers(-1, vocab, shape[:-1] + (top,)).astype(np.int32)
    t = rng.standard_normal(shape[:-1] + (top,)).astype(dtype)
    labels = rng.integers(-1, vocab, shape[:-1]) if hard else None
    weights = (rng.random(shape[:-1]) * 8).astype(F32)
    weights.reshape(-1)[::7] = 0
    some = np.unique(np.concatenate([[0, 1, 2, 147, 148, 149, rows // 2, rows - 2, rows - 1], rng.integers(0, rows, 4)]))
    run(backend, placed(z, layout), placed(k, "dense"), placed(t, layout), labels, weights, temperature, hard, 4.0, layout, some=some)


@pytest.mark.parametrize("shape", [(4, 100), (2, 40000), (2, 130001), (300, 17000), (300, 100003)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_gradient_over_the_logits(backend, shape, dtype):
    rng = np.random.default_rng(2)
    z, k, t = problem(rng, shape, 9, dtype)
    labels = rng.integers(0, shape[-1], shape[:-1])
    some = np.array([0, shape[0] // 2, shape[0] - 1])
    apart = run(backend, z, k, t, labels, None, 2.0, 0.5, 8.0, some=some)
    assert np.array_equal(run(backend, z.copy(), k, t, labels, None, 2.0, 0.5, 8.0, in_place=True, some=some), apart)


def test_a_view_of_longer_sequences(backend):
    """Logits without the last position of each sequence, labels without the first: views, nothing copied."""
    rng = np.random.default_rng(3)
    z, k, t = problem(rng, (3, 6, 777), 4, F16)
    labels = rng.integers(0, 777, (3, 6))
    whole = np.zeros((3, 6, 777), F16)
    space = Space(backend)
    put = space.put
    losses = np.full((3, 5), np.nan, F32)
    backend.distill_loss(put(z[:, :-1]), put(k[:, :-1]), put(t[:, :-1]), put(losses), labels=put(labels[:, 1:]), grad=put(whole[:, :-1]), hard_weight=0.5)
    want = distill(z[:, :-1].reshape(15, 777), k[:, :-1].reshape(15, 4), t[:, :-1].reshape(15, 4), labels[:, 1:].reshape(-1), None, 1.0, 0.5, 1.0)
    check(space.get(losses)[0].reshape(-1), *want["losses"], F32, "losses")
    got, rest = space.get(whole[:, :-1])
    assert rest  # the last positions keep their zeros
    check(got.reshape(15, 777), *want["grad"], F16, "gradient")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab,top", [(3, 40, 64), (5, 200, 65), (300, 333, 100), (2, 90001, 1024), (298, 9001, 70), (297, 33001, 120), (299, 18000, 300)])
def test_many_entries_that_repeat(backend, dtype, rows, vocab, top):
    """More entries than there are different columns: each column is written once, with all that its entries take off."""
    rng = np.random.default_rng(top)
    z = rng.standard_normal((rows, vocab), dtype=np.float32).astype(dtype)
    columns = rng.choice(vocab, max(2, min(vocab, top * 2 // 3)), replace=False)
    columns[:2] = 0, vocab - 1
    k = rng.choice(columns, (rows, top)).astype(np.int32)
    k[rng.random(k.shape) < 0.1] = -1
    t = rng.standard_normal((rows, top)).astype(dtype)
    labels = rng.choice(columns, rows)
    labels[::5] = -1
    some = np.unique([0, 1, rows // 2, rows - 1])
    run(backend, z, k, t, labels, None, 2.0, 0.25, 4.0, some=some)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab", [50, 70000])
def test_entries_that_are_none_and_entries_that_repeat(backend, dtype, vocab):
    """Ids below 0, rows without any, a column named several times, -inf of the teacher; labels below 0; a label on a teacher's column."""
    rng = np.random.default_rng(4)
    z, k, t = problem(rng, (8, vocab), 6, dtype)
    k[0, 2:] = -1
    k[1] = -1
    k[2] = k[2, 0]
    k[3, 1], k[3, 4] = k[3, 0], k[3, 5]
    t[4, :3] = -np.inf
    t[5] = -np.inf
    t[6] = np.finfo(dtype).min
    labels = rng.integers(0, vocab, 8)
    labels[0], labels[1], labels[2], labels[3] = -1, -100, k[2, 0], k[3, 4]
    for hard in (0.0, 0.5, 1.0):
        run(backend, z, k, t, labels, None, 2.0, hard, 16.0)
    run(backend, z, k, t, None, None, 1.0, 0.0, 16.0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab", [40, 66000])
def test_masked_logits(backend, dtype, vocab):
    """Columns at -inf or at the type's lowest value; whole rows of either; a row of one finite logit; a teacher that wants a masked column."""
    rng = np.random.default_rng(5)
    z, k, t = problem(rng, (7, vocab), 4, dtype)
    low = np.finfo(dtype).min
    masked = np.setdiff1d(np.arange(vocab), k[0])[: vocab // 2]
    z[0, masked] = -np.inf
    z[1, np.setdiff1d(np.arange(vocab), k[1])] = low
    z[2] = -np.inf
    z[3] = low
    z[4] = -np.inf
    z[4, k[4, 0]] = 1.0
    k[4] = k[4, 0]
    z[5, k[5, 1]] = -np.inf
    labels = k[:, 0].astype(np.int64)
    run(backend, z, k, t, labels, None, 1.0, 0.5, 1.0)
    run(backend, z, k, t, labels, None, 2.0, 0.0, 1.0)


def test_rows_of_padding_hold_anything(backend):
    """A losses' gradient of 0 is a row of zeros, whatever lies in the row, in the teacher's, and in the other rows."""
    rng = np.random.default_rng(6)
    for vocab in (300, 90000):
        z, k, t = problem(rng, (4, vocab), 5, F32)
        z[1], t[1], z[2, 3], t[3, 0] = np.nan, np.nan, np.inf, np.inf
        weights = np.array([1, 0, 0, 0], F32)
        labels = np.zeros(4, np.int64)
        space = Space(backend)
        put = space.put
        losses, grad, stats = np.empty(4, F32), np.empty((4, vocab), F32), np.empty((4, 4), F32)
        options = dict(labels=put(labels), losses_grad=put(weights), hard_weight=0.3)
        backend.distill_loss(put(z), put(k), put(t), put(losses), grad=put(grad), stats=put(stats), **options)
        want = distill(z[:1], k[:1], t[:1], labels[:1], weights[:1], 1.0, 0.3, 1.0)
        got = space.get(grad)[0]
        check(got[:1], *want["grad"], F32, "gradient")
        assert not got[1:].any()
        check(space.get(losses)[0][:1], *want["losses"], F32, "losses")
        backend.distill_loss_backward(put(z), put(k), put(t), put(stats), put(grad), **options)
        assert not space.get(grad)[0][1:].any()


def test_indices_out_of_range(backend):
    """An id or a label at or above V is an index error and no entry."""
    rng = np.random.default_rng(7)
    z, k, t = problem(rng, (3, 60), 4, F32, np.int64)
    bad, labels = k.copy(), np.array([3, 2 ** 35, 5])
    bad[0, 1], bad[2, 3] = 60, 2 ** 33
    space = Space(backend)
    put = space.put
    losses, grad = np.empty(3, F32), np.empty((3, 60), F32)
    backend.distill_loss(put(z), put(bad), put(t), put(losses), labels=put(labels), grad=put(grad), hard_weight=0.5)
    with pytest.raises(IndexError):
        backend.synchronize()
    want = distill(z, bad, t, labels, None, 1.0, 0.5, 1.0)
    check(space.get(losses)[0], *want["losses"], F32, "losses")
    check(space.get(grad)[0], *want["grad"], F32, "gradient")
    backend.synchronize()


def test_no_rows(backend):
    space = Space(backend)
    put = space.put
    backend.distill_loss(put(np.empty((0, 9), F32)), put(np.empty((0, 2), np.int32)), put(np.empty((0, 2), F32)), put(np.empty(0, F32)), grad=put(np.empty((0, 9), F32)))
    z, k, t = np.ones((2, 9), F32), np.empty((2, 0), np.int32), np.empty((2, 0), F32)
    losses, grad = np.full(2, np.nan, F32), np.full((2, 9), np.nan, F32)
    backend.distill_loss(put(z), put(k), put(t), put(losses), grad=put(grad))  # a teacher without entries
    assert not space.get(losses)[0].any() and not space.get(grad)[0].any()


def test_gradient_against_differences(backend):
    """Central differences of the losses, computed in F32: with a step of 2^-6 the third derivative leaves under 2^-12 and the losses' own roundings
    (2^-21 and a few of their size) over the step 2^-13: 2^-9 holds both with the gradients' sizes here."""
    rng = np.random.default_rng(9)
    z, k, t = problem(rng, (2, 40), 5, F32)
    labels = np.array([1, 7])

    def losses_of(z):
        space = Space(backend)
        put = space.put
        losses = np.empty(2, F32)
        backend.distill_loss(put(z), put(k), put(t), put(losses), labels=put(labels), temperature=2.0, hard_weight=0.25)
        return space.get(losses)[0].astype(np.float64)

    space = Space(backend)
    put = space.put
    losses, grad = np.empty(2, F32), np.empty((2, 40), F32)
    backend.distill_loss(put(z), put(k), put(t), put(losses), labels=put(labels), grad=put(grad), temperature=2.0, hard_weight=0.25)
    got = space.get(grad)[0]
    for r, c in ((0, 0), (0, 1), (0, int(k[0, 2])), (1, 7), (1, 39), (1, int(k[1, 0]))):
        up, down = z.copy(), z.copy()
        up[r, c] += F32(2.0 ** -6)
        down[r, c] -= F32(2.0 ** -6)
        assert abs((losses_of(up)[r] - losses_of(down)[r]) / 2.0 ** -5 - got[r, c]) <= 2.0 ** -9
