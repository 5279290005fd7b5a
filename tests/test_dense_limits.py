"""The dense operators at the edges of what they accept: the longest rows, empty batches, the largest and smallest factors."""
import ctypes as C

import pytest

from xstar_moe import capi


def _w4(rows, cols, group=128):
    w = capi.XsMoeW4()
    w.codes_dev = w.scales_dev = 4096
    w.rows, w.cols, w.group = rows, cols, group
    return w


# ---- no GPU needed ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 12, 16])
@pytest.mark.parametrize("cols", [2**24, 2**27, 2**28 - 2048, 2**28, 400_000_000, 480_000_000, 2**29, 2**30 - 2**16, 2**30 - 128, 2**30])
def test_rows_that_no_shared_memory_holds_ask_for_the_scratch_of_larger_batches(tokens, cols):
    """a token of 2^24 columns is 32 MB: such a batch is made ready in the workspace (two bytes a column), whatever 32 bits make of its size"""
    L, n = capi.lib(), C.c_size_t(0)
    w = _w4(8, cols // 128 * 128)
    assert L.xs_moe_linear_w4_workspace_bytes(C.byref(w), tokens, C.byref(n)) == 0
    assert n.value > 2 * tokens * w.cols
    if 2 * w.cols <= 2**30:  # rows of the gate and up matrix
        gate_up, down = _w4(2 * w.cols, 128), _w4(128, w.cols)
        assert L.xs_moe_mlp_w4_workspace_bytes(C.byref(gate_up), C.byref(down), tokens, C.byref(n)) == 0
        assert n.value > 2 * tokens * w.cols + 2 * gate_up.rows
