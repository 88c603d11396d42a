"""Token ids at the ends of their type."""
import numpy as np
import pytest

from language import Space, check, embedding_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [40, 5000])
@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("end", ["min", "max"])
@pytest.mark.parametrize("padding", [None, 3, -7])
def test_the_types_ends_are_out_of_range(backend, count, dtype, end, padding):
    """One such id is an index error, with a padding id, without one, and with one below 0, which is none."""
    rng = np.random.default_rng(count)
    ids, grad = rng.integers(0, 30, count).astype(dtype), rng.standard_normal((count, 24)).astype(np.float32)
    ids[count // 2] = getattr(np.iinfo(dtype), end)
    table = np.full((30, 24), np.nan, np.float32)
    space = Space(backend)
    g, i, t = space.put(grad), space.put(ids), space.put(table)
    backend.embedding_backward(g, i, t, padding_id=padding)
    with pytest.raises(IndexError):
        backend.synchronize()
    want, bound, _ = embedding_backward(ids, grad, 30, 1.0, padding if padding == 3 else None, None)
    check(space.get(table)[0], want, bound, np.float32, "table gradient")
    backend.embedding_backward(g, i, t, padding_id=-int(2 ** 63))  # the type's lowest value as a padding id: none
    with pytest.raises(IndexError):
        backend.synchronize()


def test_one_token_of_its_own(backend):
    """An id without extents: its row of the gradient is the token's, the others are zeros; added to what is there, theirs stay."""
    row, ids = np.array([1.5, -2.0, 0.25, 3.0], np.float32), np.array(2, np.int32)
    for before in (None, np.arange(12, dtype=np.float32).reshape(3, 4)):
        table = np.full((3, 4), np.nan, np.float32) if before is None else before.copy()
        space = Space(backend)
        backend.embedding_backward(space.put(row), space.put(ids), space.put(table), scale=2.0, accumulate=before is not None)
        want = np.zeros((3, 4), np.float32) if before is None else before.copy()
        want[2] += 2 * row
        assert np.array_equal(space.get(table)[0], want)
