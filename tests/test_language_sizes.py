"""What the size of a workspace is told without a device: enough for every way in which a device divides the call."""
import ctypes as C

import pytest

from vkml_b200 import DType, TensorDesc, _abi, graph


@pytest.mark.parametrize("count", [513, 8192, 8193, 16384, 16385, 32768, 32769, 70000])
def test_sorted_tokens(count):
    """Tokens and their places twice, a bit for each row, and 256 counts for each tile of 1024 tokens (2048 where there are more than 65536) and one
    tile more: 8193 to 16384 tokens are such tiles in a cluster of 16 blocks, and half as many where a device takes 8 at most."""
    whole = lambda n: -(-n // 256) * 256  # noqa: E731
    vocab = 5000
    args = graph.embedding_args(TensorDesc.contiguous(1 << 30, (vocab, 1), DType.F32), TensorDesc.contiguous(2 << 30, (count,), DType.I64),
                                TensorDesc.contiguous(3 << 30, (count, 1), DType.F32), 1.0)
    n = C.c_size_t(0)
    assert _abi.load().b200_embedding_backward_workspace(args, C.byref(n)) == 0
    tiles = -(-count // (1024 if count <= 65536 else 2048))
    least = 2 * whole(count * 8) + whole(-(-vocab // 32) * 4) + 1024 * (tiles + 1)
    assert n.value >= least, (n.value, least)
