"""The language-model operators called at once: a context and a thread each, first calls included."""
import threading

import numpy as np
import pytest

import vkml_b200 as B
from test_language_together_gpu import RESULTS, operators, scratch_problem

pytestmark = pytest.mark.gpu


def test_two_threads_with_a_context_each():
    """Both begin at the same time, in sizes that no call had before where this file runs alone; the bits are those of one after the other."""
    contexts = [B.Backend(0) for _ in range(2)]
    problems = [scratch_problem(c, 21) for c in contexts]
    start, got, errors = threading.Barrier(2), [None, None], []

    def work(i):
        try:
            start.wait()
            for _ in range(20):
                operators(contexts[i], problems[i], None)
            got[i] = [problems[i][k].numpy() for k in RESULTS]
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    operators(contexts[0], problems[0], None)
    for k, a, b in zip(RESULTS, *got):
        assert np.array_equal(a, b), k
        assert np.array_equal(a, problems[0][k].numpy()), k
    for c, s in zip(contexts, problems):
        for t in s.values():
            t.storage.__del__()
        c.close()
