"""Sizes of the linear products that no launch takes (2^32 work-items and more) are refused before it, without a GPU."""
import ctypes

import pytest

from deep_optimization_amd import _lib

BUF = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUF) + 255) // 256 * 256  # an address that no refused call reads
ODD = AT + 2                                     # rows at any element: 32 x 64 and 64 x 64 tiles only
BF, FP = _lib.BF16, _lib.F32


@pytest.mark.parametrize("M,N", [(1 << 29, 128), (1 << 24, 1 << 13), ((1 << 30) - 200, 128), (1 << 18, 1 << 19)])
def test_results_of_more_tiles_than_a_launch_takes(M, N):
    L, K = _lib.lib(), 64
    assert ((M + 63) // 64) * ((N + 63) // 64) * 256 >= 1 << 32
    forward = L.dopt_linear_forward(ODD, K, AT, K, BF, M, N, K, None, FP, None, 0, AT, BF, None, None)
    # dx [M, N'] of N' = N in features, K out features; dw [M', N] of M' = M out features
    input_grad = L.dopt_linear_input_grad(ODD, K, AT, N, BF, M, K, N, None, 0, AT, None)
    assert forward == _lib.EUNSUPPORTED and input_grad == _lib.EUNSUPPORTED and b"tiles" in L.dopt_last_error()
    assert [L.dopt_linear_tile(p, M, *nk, 1) for p, nk in ((0, (N, K)), (1, (K, N)))] == [-2, -2]
    # aligned rows have tiles that fit
    assert L.dopt_linear_tile(0, M, N, K, 0) >= 0 and L.dopt_linear_copy_preferred(0, M, N, K, N * K, 1) == 1


def test_weight_gradients_of_more_tiles_than_a_launch_takes():
    L, M, N, K = _lib.lib(), 64, 1 << 20, 1 << 17
    assert L.dopt_linear_weight_grad(ODD, N, AT, K, BF, M, N, K, None, AT, None, None, None, None) == _lib.EUNSUPPORTED
    assert b"tiles" in L.dopt_last_error()


def test_sums_of_more_columns_than_a_launch_takes():
    cols = (1 << 26) - 8
    rows = (_lib.LinearRows * 4)(*[_lib.LinearRows(AT, cols, None, 2, cols, AT, cols, 0, BF, AT, AT) for _ in range(4)])
    assert _lib.lib().dopt_linear_layout(rows, 4, BF, None) == _lib.EUNSUPPORTED
