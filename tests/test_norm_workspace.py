"""The norm backward's workspace follows the rows (CPU; what it computes is tested on the GPU)."""
import ctypes

import pytest

from easyllm_amd import _lib

A = 1 << 20  # an aligned address nobody reads


@pytest.mark.parametrize("rows,h,blocks", [
    (0, 64, 1), (1, 64, 1), (5, 64, 2), (1, 2048, 1), (2, 4096, 1), (3, 4096, 2), (1, 8192, 1), (7, 8192, 7),  # blocks of 4, 2 and 1 rows
    (1024, 2048, 256), (8192, 2048, 256), (8193, 2048, 512), (4096, 4096, 256), (4097, 4096, 512), (4096, 5120, 512), (100000, 8192, 256)])
def test_three_sets_of_the_launched_blocks_partial_rows(rows, h, blocks):
    assert _lib.norm_bwd_workspace_bytes(rows, h) == 3 * blocks * h * 4


def test_nothing_less_is_taken():
    _lib.load()
    grad = ctypes.byref(_lib.LayerGrad(A, None, 0))
    for rows, h in ((1, 8192), (300, 264), (9000, 2048)):
        size = _lib.norm_bwd_workspace_bytes(rows, h)
        with pytest.raises(RuntimeError, match="workspace"):
            _lib.call("ezl_norm_bwd", 0, A, None, A, A, A, A, None, A, None, grad, None, None, A, size - 1, rows, h, None)
