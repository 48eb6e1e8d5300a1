"""The largest sizes that the output layer's entry points take are refused by
their own checks, not by the launch: HIP takes fewer than 2^32 threads."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)


@pytest.fixture(scope='module')
def lib():
    import os
    from zhusuan_amd import _capi
    import __graft_entry__ as g
    if not os.path.exists(g.LIB):
        g.build()
    return _capi.load()


def test_rows_of_class_logits(lib):
    n = ctypes.c_int64(0)

    def rc(N):
        return lib.zshmc_class_log_prob_workspace(
            P, P, N, 4, 5, 4, 4, 1, 0, 0, ctypes.addressof(n))
    assert rc(2 ** 27) == 0 and rc(2 ** 27 + 1) == 1


@pytest.mark.parametrize('gradient', [0, 1])
def test_tiles_of_class_logits(lib, gradient):
    """2^27 rows over 2^20 classes: refused with the reason, before a launch
    (nothing here is a device pointer)."""
    from zhusuan_amd import _capi
    n = ctypes.c_int64(0)
    N, D, V = 2 ** 27, 64, 2 ** 20
    assert lib.zshmc_class_log_prob_workspace(
        P, P, N, D, V, D, D, 1, gradient, 0, ctypes.addressof(n)) == 0
    if gradient:
        rc = lib.zshmc_class_log_prob_grad(
            P, P, None, P, N, D, V, D, D, 1, 0, 0, P, P, P, P, None, P,
            n.value, None)
    else:
        rc = lib.zshmc_class_log_prob(
            P, P, None, P, N, D, V, D, D, 1, 0, 0, P, None, P, n.value, None)
    assert rc == 1 and 'tiles' in _capi.last_error()


def test_tiles_of_the_8_bit_product(lib):
    from zhusuan_amd import _capi
    assert lib.zshmc_int8_linear(P, 64, P, P, 64, P, None, 2 ** 30, 64,
                                 2 ** 20, P, 2 ** 20, 0, None) == 1
    assert 'tiles' in _capi.last_error()
