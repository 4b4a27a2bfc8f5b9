"""More arguments that the type vectors' entry points refuse before they launch anything."""
import pytest


@pytest.mark.parametrize("eps", [float("inf"), 1e39])
def test_an_eps_that_is_no_finite_float(eps):
    """1e39 is finite as the host layer's number and infinite as the kernels' float, where a result would be the bias."""
    from libmolgrid_amd import _capi
    a = 0x10000                                   # an address that nothing reads
    assert _capi.lib.mg_layer_norm(3, 5, 0, 0, a, a, a, eps, a, a, a, None) == _capi.MG_ERR_INVALID_ARGUMENT
    assert _capi.lib.mg_encode_types(3, 4, 5, 0, 0, 0, a, a, 1.0, a, a, eps, 0.1, 1, 2, None, a, None) == \
        _capi.MG_ERR_INVALID_ARGUMENT
    size = _capi.lib.mg_encode_types_backward_workspace_size(3, 4, 5)
    assert _capi.lib.mg_encode_types_backward(3, 4, 5, 0, 0, 0, a, a, a, 1.0, a, eps, 0.1, 1, 2, None, a, a, a, a, size,
                                              None) == _capi.MG_ERR_INVALID_ARGUMENT
