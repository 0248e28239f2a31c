"""Descriptions at the limits of the C entry points: what does not fit a launch is refused before any device call."""
import ctypes as C

import pytest

from wfe_amd import _lib

F32, F16, BF16 = 0, 1, 2
ANY = 64                                       # an address that nothing reads


def backward(rows, vocab, dim, dtype):
    lib = _lib.lib()
    d = _lib.WfeEmbedding(0, dtype, rows, dim, 0, dim, vocab, 64, dtype, -1, 1.0)
    need = lib.wfe_embedding_workspace_bytes(C.byref(d))
    assert need > 0
    # (a workspace a byte short: what fits is refused for that, still before any device call)
    rc = lib.wfe_embedding_backward(C.byref(d), ANY, ANY, ANY, ANY, need - 1, None)
    assert rc == _lib.ERR_ARG
    return lib.wfe_last_error(None).decode()


@pytest.mark.parametrize("rows,vocab,dim,dtype,fits", [
    (1 << 24, 1000, 16384, F32, False), (1 << 24, 1 << 24, 16384, BF16, False), (16, 1 << 24, 16384, F32, False),
    (1 << 24, 1000, 16384, F16, True), (1 << 23, 1000, 16384, F32, True), (1 << 24, 1 << 24, 64, F32, True),
    (1 << 24, 51866, 8192, F32, True), (16, 1 << 22, 16384, F32, True), (16, 1 << 24, 16384, BF16, False)])
def test_embedding_gradients_beyond_a_launch(rows, vocab, dim, dtype, fits):
    text = backward(rows, vocab, dim, dtype)
    assert ("workspace" in text) == fits and ("more than one launch" in text) != fits, text
    slab = 256 if dtype == F32 else 512
    slabs = (dim + slab - 1) // slab
    threads = (-(-rows // 16) * slabs if rows > 16 else 0) * 64 + -(-vocab // 8) * slabs * 64
    assert (threads < 1 << 32) == fits
