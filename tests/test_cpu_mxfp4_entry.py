"""Refusals of the microscaled 4-bit entry points that need no GPU: the host
checks its arguments before anything is launched."""
import pytest

from qtpytorch_amd import _lib as L

SOME = 1 << 12  # an address that is never read


def _grad(entry, m, n, k, out):
    """dy and the codes given wherever they have elements."""
    dy, q = (SOME if m and n else 0), (SOME if k else 0)
    return getattr(L.lib(), entry)(dy, L.MXK_IN_BF16, m, n, q, q, k, L.MXK_IN_BF16, out, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("m,n,k", [(0, 8, 64), (8, 8, 64), (1 << 30, 1 << 21, 1 << 25)])
def test_gradient_of_the_weight_without_a_result_is_refused(m, n, k):
    """Also where the sum is empty (zeros are written) and where m * n * k passes 64 bits."""
    assert _grad("mxk_mxfp4_grad_b", m, n, k, 0) == L.MXK_EINVAL
    assert b"null pointer" in L.lib().mxk_last_error()


@pytest.mark.parametrize("m,n,k", [(8, 0, 64), (8, 8, 64), (1 << 30, 1 << 21, 1 << 25)])
def test_gradient_of_the_input_without_a_result_is_refused(m, n, k):
    assert _grad("mxk_mxfp4_grad_a", m, n, k, 0) == L.MXK_EINVAL
    assert b"null pointer" in L.lib().mxk_last_error()


@pytest.mark.parametrize("entry,sizes", [("mxk_mxfp4_grad_a", [(0, 8, 64), (8, 8, 0)]),
                                         ("mxk_mxfp4_grad_b", [(8, 0, 64), (8, 8, 0)])])
def test_gradients_without_elements_need_no_result(entry, sizes):
    for m, n, k in sizes:
        assert _grad(entry, m, n, k, 0) == L.MXK_OK
