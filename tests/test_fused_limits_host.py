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
