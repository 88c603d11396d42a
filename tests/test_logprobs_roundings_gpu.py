"""Log probabilities of long rows within as many roundings as a row's sum has."""
import numpy as np
import pytest

import language_steps
from test_logprobs_gpu import F16, F32, compare, forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab", [(2, 300007), (300, 128000), (2100, 50000), (2100, 9000)])
def test_long_rows(backend, monkeypatch, dtype, rows, vocab):
    """A thread takes batches of four vectors, 16 elements at least, half of them to either of two sums: 16 terms of a sum at most, one addition of the two and one to what the
    thread has.  Rows of so many columns have 64 threads or more, so vocab / 1024 batches at most; a tree over at most 4096 threads follows, 12 additions.  Each move of the number that a thread's sums
    are beside of is five roundings (a function's four and a product's): a few moves of a thread that meets a larger element are counted by the rest of vocab / 512 + 32."""
    monkeypatch.setattr(language_steps, "_rounds", lambda n: n / 512 + 32)
    rng = np.random.default_rng(vocab)
    z = (rng.standard_normal((rows, vocab), dtype=F32) * 2.5).astype(dtype)
    tokens = rng.integers(0, vocab, rows)
    some = np.unique(np.concatenate([[0, rows - 1], rng.integers(0, rows, 10)]))
    compare(forward(backend, z, tokens, 0.9), z, tokens, 0.9, 0, some)
