"""The backward workspace of the vocabulary cross entropy: logits are never kept, however narrow the model is."""
import ctypes as C

import pytest

from wfe_amd import _lib

MB = 1 << 20
F32, F16, BF16 = 0, 1, 2


def workspace(rows, dim, vocab, dtype, grads, reduction=2):
    d = _lib.WfeLinearCe(0, dtype, rows, rows, 0, dim, dim, dim, vocab, 64, reduction, -100, dtype, dtype)
    got = _lib.lib().wfe_linear_ce_workspace_bytes(C.byref(d), None, 1, grads)
    assert got > 0
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256, 384, 768, 1280, 4096, 16384])
@pytest.mark.parametrize("rows,vocab", [(1, 51866), (255, 1 << 24), (7168, 51866), (28672, 51866), (80000, 51866),
                                        (1 << 20, 1 << 17), (1 << 24, 8192), (1 << 24, 300), (2_200_000, 257)])
def test_probabilities_take_a_fixed_room(rows, vocab, dim, dtype):
    size = 4 if dtype == F32 else 2
    up = lambda n, to: (n + to - 1) // to * to  # noqa: E731
    one = up(rows, 256) * dim * 4
    for reduction in (0, 2):
        rows_again = up(rows, 256) * dim * size + 512 if reduction == 0 else 0
        assert workspace(rows, dim, vocab, dtype, 2, reduction) <= (512 + 96) * MB + rows_again + 1024
        hidden = max(64 * MB, one, min(4 * one, 512 * MB))
        assert workspace(rows, dim, vocab, dtype, 1, reduction) <= 512 * MB + hidden + 1024
        assert workspace(rows, dim, vocab, dtype, 3, reduction) <= (512 + 96) * MB + hidden + rows_again + 2048
    if rows * vocab * size > 8 << 30:
        assert workspace(rows, dim, vocab, dtype, 2) < rows * vocab * size // 10
