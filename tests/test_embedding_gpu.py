"""Embedding lookup with scaling and its gradient against plain sums in 64 bits."""
import numpy as np
import pytest

from language import EPS, Space, check, embedding_backward, placed, rows_view

pytestmark = pytest.mark.gpu

TYPES = [(np.float32, np.float32), (np.float32, np.float16), (np.float16, np.float32), (np.float16, np.float16)]


def ids_of(rng, shape, vocab, dtype=np.int64, skew=True):
    u = rng.random(shape)
    ids = np.minimum(vocab - 1, ((vocab + 1.0) ** u - 1 if skew else u * vocab)).astype(dtype)
    return ids


@pytest.mark.parametrize("table_type,row_type", TYPES)
@pytest.mark.parametrize("shape,vocab,width,layout", [
    ((1,), 1, 1, "dense"), ((7,), 5, 8, "dense"), ((4, 8), 1000, 64, "dense"), ((3, 5), 11, 33, "offset"), ((3, 67), 300, 1000, "pitch"),
    ((5, 9), 40, 24, "odd"), ((6, 4), 40, 136, "swapped"), ((2, 130), 64, 2048, "backwards")])
def test_lookup(backend, table_type, row_type, shape, vocab, width, layout):
    rng = np.random.default_rng(vocab * 7 + width)
    table = placed(rng.standard_normal((vocab, width)).astype(table_type), "pitch" if layout in ("pitch", "swapped") else "offset" if layout == "offset" else "dense")
    ids = ids_of(rng, shape, vocab, np.int32 if layout == "pitch" else np.int64)
    if layout == "swapped":
        ids = np.ascontiguousarray(ids.T).T
    rows = rows_view(shape + (width,), row_type, layout if len(shape) > 1 or layout != "swapped" else "dense")
    space = Space(backend)
    backend.embedding(space.put(table), space.put(ids), space.put(rows), scale=1.7)
    got, rest = space.get(rows)
    backend.synchronize()
    # one product, rounded, and rounded again to the rows' type: the same bits
    assert np.array_equal(got, (table[ids].astype(np.float32) * np.float32(1.7)).astype(row_type)) and rest


def test_lookup_out_of_range(backend):
    table, ids = np.ones((5, 16), np.float32), np.array([4, -1, 5, 0, 2 ** 40], np.int64)
    rows = np.full((5, 16), 7, np.float32)
    space = Space(backend)
    t, i, r = space.put(table), space.put(ids), space.put(rows)
    backend.embedding(t, i, r)
    with pytest.raises(IndexError):
        backend.synchronize()
    got, _ = space.get(rows)
    assert np.array_equal(got[:, 0], [1, 0, 0, 1, 0])
    backend.synchronize()  # the error was told once


@pytest.mark.parametrize("row_type,table_type", TYPES)
@pytest.mark.parametrize("shape,vocab,width,layout,accumulate", [
    ((1,), 1, 1, "dense", False), ((5,), 3, 8, "dense", True), ((4, 8), 1000, 64, "dense", False), ((3, 700), 90, 33, "odd", False),
    ((2, 1500), 1200, 130, "pitch", True), ((4, 1024), 700, 256, "swapped", False), ((9, 401), 2000, 72, "backwards", True),
    ((1, 9000), 17, 40, "dense", False), ((3, 5000), 40000, 16, "dense", False), ((0,), 6, 8, "dense", False), ((2, 0), 6, 8, "dense", True),
    ((40, 1000), 64, 1032, "dense", False), ((17, 1023), 3000, 1025, "offset", True)])
def test_gradient(backend, row_type, table_type, shape, vocab, width, layout, accumulate):
    rng = np.random.default_rng(vocab * 3 + width)
    ids = ids_of(rng, shape, vocab, np.int32 if layout == "odd" else np.int64)
    padding = None if layout == "dense" else vocab - 1
    if padding is not None and len(shape) == 2:
        ids[:, shape[1] * 3 // 4:] = padding
    grad = placed(rng.standard_normal(shape + (width,)).astype(row_type), layout)
    before = rng.standard_normal((vocab, width)).astype(table_type)
    table = placed(before, "pitch" if layout in ("pitch", "odd") else "offset" if layout == "offset" else "dense")
    if not accumulate:
        table[...] = np.nan
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t, scale=0.75, padding_id=padding, accumulate=accumulate)
    got, rest = space.get(table)
    want, bound, touched = embedding_backward(ids, grad, vocab, 0.75, padding, before if accumulate else None)
    check(got, want, bound, table_type, "table gradient")
    assert rest
    if accumulate:  # rows without a token keep their bytes
        assert np.array_equal(got[~touched], before[~touched])
    else:
        assert not got[~touched].any()
    # the same bits again, in another workspace
    again = Space(backend)
    g, i, t = again.put(grad), again.put(ids), again.put(table)
    ws = backend.allocate(max(1, backend.embedding_backward_workspace(g, i, t)))
    backend.embedding_backward(g, i, t, scale=0.75, padding_id=padding, accumulate=accumulate, workspace=ws)
    assert np.array_equal(again.get(table)[0], got, equal_nan=True)
    backend.synchronize()


@pytest.mark.parametrize("count,vocab,width", [(1024, 255, 8), (1025, 256, 8), (16384, 65535, 4), (16385, 65536, 4), (70001, 300, 3), (131072, 70000, 8), (131073, 900, 8),
                                               (600000, 66000, 5), (1200000, 130, 8)])
@pytest.mark.parametrize("skew", [False, True])
def test_gradient_of_many_tokens(backend, count, vocab, width, skew):
    """Counts at which the sort changes over, and ids of one, two and three digits."""
    rng = np.random.default_rng(count)
    ids = ids_of(rng, (count,), vocab, np.int32 if skew else np.int64, skew)
    grad = rng.standard_normal((count, width)).astype(np.float32)
    table = np.full((vocab, width), np.nan, np.float32)
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t)
    got = space.get(table)[0]
    want, bound, touched = embedding_backward(ids, grad, vocab, 1.0, None, None)
    check(got, want, bound, np.float32, "table gradient")
    assert not got[~touched].any()
    backend.synchronize()


@pytest.mark.parametrize("count,vocab,width", [(0, 70000, 64), (1, 70000, 64), (3, 1100000, 4), (128, 5000, 838), (128, 5000, 840), (128, 60, 1000), (129, 60, 1000), (129, 1, 1), (512, 1024, 128), (513, 1024, 128), (512, 1025, 128)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_few_tokens(backend, count, vocab, width, accumulate):
    """The counts and tables at which the rows are no longer owned by blocks."""
    rng = np.random.default_rng(count + width)
    ids, grad = ids_of(rng, (count,), vocab, np.int64, True), rng.standard_normal((count, width)).astype(np.float16)
    table = rng.standard_normal((vocab, width)).astype(np.float32) if accumulate else np.full((vocab, width), np.nan, np.float32)
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t, accumulate=accumulate)
    got = space.get(table)[0]
    want, bound, touched = embedding_backward(ids, grad, vocab, 1.0, None, table if accumulate else None)
    check(got, want, bound, np.float32, "table gradient")
    assert np.array_equal(got[~touched], table[~touched]) if accumulate else not got[~touched].any()


@pytest.mark.parametrize("count,vocab", [(3000, 4), (30000, 50000), (200000, 9)])
def test_gradient_of_one_token(backend, count, vocab):
    """Every token the same: one list, as long as there are tokens."""
    rng = np.random.default_rng(5)
    ids, grad = np.full(count, vocab - 2, np.int64), rng.standard_normal((count, 48)).astype(np.float16)
    table = np.full((vocab, 48), np.nan, np.float32)
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t)
    want, bound, _ = embedding_backward(ids, grad, vocab, 1.0, None, None)
    check(space.get(table)[0], want, bound, np.float32, "table gradient")


@pytest.mark.parametrize("count", [40, 5000])
def test_gradient_leaves_bad_ids_out(backend, count):
    """Ids out of range are an index error and add to no row; padding is neither, in the table or outside of it."""
    rng = np.random.default_rng(6)
    ids, grad = rng.integers(0, 30, count), rng.standard_normal((count, 24)).astype(np.float32)
    ids[::7], ids[3::11] = 30, 40
    for padding, raises in ((40, True), (30, True), (None, True)):
        table = np.full((30, 24), np.nan, np.float32)
        space = Space(backend)
        g, i, t = space.put(grad), space.put(ids), space.put(table)
        backend.embedding_backward(g, i, t, padding_id=padding)
        if raises:
            with pytest.raises(IndexError):
                backend.synchronize()
        want, bound, _ = embedding_backward(ids, grad, 30, 1.0, padding, None)
        check(space.get(table)[0], want, bound, np.float32, "table gradient")
    ids[3::11] = 30
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t, padding_id=30)
    backend.synchronize()  # nothing but padding was left out


@pytest.mark.parametrize("count", [0, 3, 600, 40000])
def test_rows_without_a_token_are_zeros_whatever_the_scale(backend, count):
    ids, grad = np.full(count, 3, np.int64), np.ones((count, 16), np.float32)
    table = np.full((9, 16), np.nan, np.float32)
    space = Space(backend)
    backend.embedding_backward(space.put(grad), space.put(ids), space.put(table), scale=float("inf"))
    got = space.get(table)[0]
    assert not np.delete(got, 3, 0).any() and (count == 0 or np.isinf(got[3]).all())


def test_one_token(backend):
    """An id without extents: one row."""
    table, ids, row = np.arange(12, dtype=np.float32).reshape(3, 4), np.array(2, np.int32), np.empty(4, np.float32)
    space = Space(backend)
    backend.embedding(space.put(table), space.put(ids), space.put(row))
    assert np.array_equal(space.get(row)[0], table[2])
    grad = np.full((3, 4), np.nan, np.float32)
    backend.embedding_backward(space.put(row + 1), space.put(ids), space.put(grad))
    assert not space.get(grad)[0][:2].any()


def test_repeated_row_of_gradients(backend):
    """A gradient that is one row for all tokens (stride 0), as that of a sum is."""
    ids = np.arange(5000, dtype=np.int64).reshape(50, 100) % 7
    grad = np.broadcast_to(np.arange(40, dtype=np.float32), (50, 100, 40))
    table = np.full((9, 40), np.nan, np.float32)
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t)
    want, bound, _ = embedding_backward(ids, grad, 9, 1.0, None, None)
    check(space.get(table)[0], want, bound, np.float32, "table gradient")


def test_gradient_against_differences(backend):
    """d/dtable of sum(rows * g): the function is linear, so a difference over any step is the derivative."""
    rng = np.random.default_rng(8)
    ids, g = rng.integers(0, 6, 20), rng.standard_normal((20, 8)).astype(np.float32)
    table = rng.standard_normal((6, 8)).astype(np.float32)
    space = Space(backend)
    rows, grad = np.empty((20, 8), np.float32), np.empty((6, 8), np.float32)
    backend.embedding_backward(space.put(g), space.put(ids), space.put(grad), scale=2.0)
    got = space.get(grad)[0]
    for v, c in ((0, 0), (3, 5), (5, 7)):
        value = []
        for step in (0.5, -0.5):
            moved = table.copy()
            moved[v, c] += np.float32(step)
            s = Space(backend)
            backend.embedding(s.put(moved), s.put(ids), s.put(rows), scale=2.0)
            value.append((s.get(rows)[0].astype(np.float64) * g).sum())
        # 20 * 8 products of two factors each rounded once: 2^-24 of their sizes
        assert abs((value[0] - value[1]) - got[v, c]) <= 200 * EPS * (np.abs(g).sum() * np.abs(table).max() * 2)
