"""Scratch and size limits of the fused operators, without a GPU."""
import pytest


@pytest.fixture(scope="module")
def K(built):
    from orion_b200 import kernels
    return kernels


@pytest.mark.parametrize("rows", [1, 127, 129, 1143, 8192, 49152, 49153, 65536, 10**6])
@pytest.mark.parametrize("V,H", [(8, 8), (2048, 64), (2049, 64), (30522, 768), (32000, 1024), (262144, 128)])
def test_scratch_of_the_loss_gradient_is_what_its_documentation_says(K, rows, V, H):
    """Without either gradient the query names what both need: 20 bytes a row (and two numbers), a copy of x, and a piece's dl."""
    total = K.lib().ob200_linear_cross_entropy_backward_workspace(rows, V, H, 0, 0)
    dl = total - 20 * rows - 2 * rows * H
    assert 2 * rows * min(V, 64) <= dl <= max(192 << 20, 4096 * rows) + 5 * 256 + 8


A = 1 << 20   # an aligned address that is never touched: every call below is refused before a launch


def test_a_reduction_that_is_no_multiple_of_8_is_refused(K):
    """Rows that lie far enough apart do not make it one: few rows are read eight elements at a time, past the row's end into what lies
    behind it."""
    L = K.lib()
    for k in (1, 4, 12, 60, 1028):
        ld = (k + 15) // 8 * 8
        assert L.ob200_linear_act_bf16(A, A, A, None, None, 0, None, 0, 0.0, None, 0, 4, 8, k, ld, ld, 0, None, 0, 1, None) == -2
        assert L.ob200_linear_act_backward_bf16(A, None, A, A, A, A, None, 0, 0, 0.0, None, 0, 4, 8, k, ld, ld, 0, A, 1 << 30, 1, None) == -2


@pytest.mark.parametrize("size", [2**31 - 1, 2**31 - 8, 2**31 - 65528])
def test_sizes_that_positions_of_32_bits_do_not_hold_are_refused(K, size):
    """A walk over blocks of rows, pieces of a vocabulary or tiles would step past 2^31 behind the last one."""
    L = K.lib()
    wide = size // 8 * 8
    for M, N, k in ((size, 8, 8), (4, size, 8), (4, 8, wide)):
        assert L.ob200_linear_act_workspace(M, N, k) == 0 and L.ob200_linear_act_backward_workspace(M, N, k, 2, 0.0, 1, 1, 1) == 0
        assert L.ob200_linear_act_bf16(A, A, A, None, None, 0, None, 0, 0.0, None, 0, M, N, k, k, k, 0, A, 1 << 60, 1, None) == -1
        assert L.ob200_linear_act_backward_bf16(A, None, A, A, A, A, None, 0, 0, 0.0, None, 0, M, N, k, k, k, 0, A, 1 << 60, 1, None) == -1
        assert L.ob200_linear_cross_entropy_workspace(M, N, k) == 0 and L.ob200_linear_cross_entropy_backward_workspace(M, N, k, 1, 1) == 0
        assert L.ob200_linear_cross_entropy_forward(A, A, A, A, A, A, A, M, N, k, k, k, -100, 1, A, 1 << 60, 1, None) == -1
        assert L.ob200_linear_cross_entropy_backward(A, A, A, A, A, 0, None, A, A, M, N, k, k, k, -100, A, 1 << 60, 1, None) == -1


def test_the_largest_sizes_have_a_plan(K):
    L, most = K.lib(), 2**31 - 65536
    assert L.ob200_linear_act_backward_workspace(most, 8, 8, 2, 0.1, 1, 1, 1) >= 2 * 8 * most
    assert L.ob200_linear_cross_entropy_backward_workspace(128, most, 8, 1, 1) >= 128 * 16
    assert L.ob200_linear_cross_entropy_backward_workspace(most, 8, 8, 1, 1) >= 20 * most + 2 * 8 * most
