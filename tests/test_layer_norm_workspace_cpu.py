"""The workspace of layer_norm's backward: as much as its partial sums take, and
no call with less.  No GPU is needed: the calls are refused before a launch."""
import ctypes

import pytest

from cign_b200 import _lib

P = ctypes.c_void_p(4096)  # never followed


def partial_sums(n, d):
    """Rows of at most 8192 columns: a partial sum per block of rows, at most 1776; wider ones: one per chunk of 16
    rows or more, and a float per row."""
    if d <= 8192:
        return 2 * min(n, 1776) * d * 4
    chunk = max(16, -(-n // 1776))
    return 2 * -(-n // chunk) * d * 4 + -(-n // 4) * 16


@pytest.mark.parametrize("n,d", [(1, 1), (5, 8192), (1776, 2560), (100000, 1024), (1, 8193), (16, 9000), (17, 9000), (2000, 40000),
                                 (28416, 8193), (28417, 8193), (1 << 30, 10000), (3, 16776960)])
def test_size_and_refusal(n, d):
    lib = _lib.load_library()
    need = lib.cign_layer_norm_bwd_workspace_bytes(n, d)
    assert need == partial_sums(n, d)
    for ws, size in ((P, need - 1), (None, need)):
        assert lib.cign_layer_norm_bwd(n, d, 0, 0, P, d, P, d, None, P, P, P, P, P, ws, size, None) == 1


def test_wide_rows_take_a_fraction_of_their_input():
    need = _lib.load_library().cign_layer_norm_bwd_workspace_bytes
    assert need(2000, 40000) == 40_008_000 and need(2000, 40000) < 2000 * 40000 * 4 / 7
    assert need(0, 10) == 0 and need(10, 0) == 0
