"""b200_check_operator leaves the device alone: a process may ask it first and fork afterwards."""
import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
    import os, sys
    sys.path[:0] = ["tests", "."]
    from test_language_refusals import (DISTILL, DISTILL_BACKWARD, EMBEDDING, EMBEDDING_BACKWARD, F16, F32, I64, NORM, NORM_BACKWARD, OK, At, answer, distill_args, grad_args,
                                        norm_args)
    from vkml_b200 import graph
    at = At()
    embedding = graph.embedding_args(at((50000, 64)), at((9000,), I64), at((9000, 64), F16), 1.0)
    for which, args in ((EMBEDDING, embedding), (EMBEDDING_BACKWARD, embedding), (NORM, norm_args(at)), (NORM_BACKWARD, grad_args(at)), (DISTILL, distill_args(at)),
                        (DISTILL_BACKWARD, distill_args(at, losses=None))):
        assert answer(which, args) == OK
    child = os.fork()
    if child == 0:
        status = 1
        try:
            import numpy as np
            from vkml_b200 import Backend, DeviceTensor
            backend = Backend(0)
            table, ids, rows = DeviceTensor.from_host(backend, np.arange(12, dtype=np.float32).reshape(3, 4)), DeviceTensor.from_host(backend, np.array([2, 0])), DeviceTensor.empty(backend, (2, 4))
            backend.embedding(table, ids, rows)
            status = 0 if np.array_equal(rows.numpy(), [[8, 9, 10, 11], [0, 1, 2, 3]]) else 2
        finally:
            os._exit(status)
    sys.exit(os.waitstatus_to_exitcode(os.waitpid(child, 0)[1]))
"""


def test_a_fork_after_the_checks():
    """The child has the device to itself and computes on it."""
    alone = dict(os.environ, OPENBLAS_NUM_THREADS="1", OMP_NUM_THREADS="1")  # (a process of several threads had better not fork)
    done = subprocess.run([sys.executable, "-c", textwrap.dedent(SCRIPT)], capture_output=True, text=True, timeout=120, env=alone)
    assert done.returncode == 0, done.stderr[-2000:]
