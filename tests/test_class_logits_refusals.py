"""What the linear Categorical and the 8-bit rows refuse, before any launch:
the Python checks and the C entry points' own."""
import ctypes

import pytest
import torch

import zhusuan_amd as zs

W = torch.zeros(5, 4)
X = torch.zeros(3, 4)
Y = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize('args,kw,error', [
    ((W.half(), X.half(), Y), {}, TypeError),
    ((W.double(), X.double(), Y), {}, TypeError),
    ((W, X.bfloat16(), Y), {}, TypeError),
    ((W, X, Y.float()), {}, TypeError),
    ((W, X, [0, 1, 2]), {}, TypeError),
    ((W, X[:, :3], Y), {}, ValueError),
    ((W[None], X, Y), {}, ValueError),
    ((W[:0], X, Y), {}, ValueError),
    ((W, X, Y[:2]), {}, ValueError),
    ((W, X, Y[:, None]), {}, ValueError),
    ((W, X, Y), dict(bias=torch.zeros(4)), ValueError),
    ((W, X, Y), dict(bias=torch.zeros(5).double()), TypeError),
    ((W, X, Y), dict(bias=1.0), TypeError),
    ((W, X, Y), dict(ignore_label=2 ** 63), (ValueError, RuntimeError)),
    ((W, X, Y), {}, RuntimeError),                 # CPU tensors
])
def test_linear_categorical_log_prob(args, kw, error):
    with pytest.raises(error):
        zs.linear_categorical_log_prob(*args, **kw)


def test_rows():
    with pytest.raises(TypeError):
        zs.quantize_rows(W.double())
    with pytest.raises(TypeError):
        zs.quantize_rows([1.0])
    with pytest.raises(ValueError):
        zs.quantize_rows(W[:, :0])
    with pytest.raises(RuntimeError, match='MI355X'):
        zs.quantize_rows(W)
    with pytest.raises(TypeError):
        zs.QuantizedRows(W, torch.ones(5))
    with pytest.raises(ValueError):
        zs.QuantizedRows(W.to(torch.int8), torch.ones(4))
    with pytest.raises(RuntimeError, match='MI355X'):
        zs.QuantizedRows(W.to(torch.int8), torch.ones(5))
    with pytest.raises(TypeError):
        zs.quantized_linear(W, X)


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__ as g
    g.build()
    from zhusuan_amd import _capi
    return _capi.load()


P = ctypes.c_void_p(4096)


def test_class_log_prob_entry(lib):
    from zhusuan_amd import _capi
    n = ctypes.c_int64(0)

    def ws(N=3, D=64, V=5, ldx=64, ldw=64, dtype=1, grad=0):
        return lib.zshmc_class_log_prob_workspace(
            P, P, N, D, V, ldx, ldw, dtype, grad, 0, ctypes.addressof(n))
    assert ws() == 0 and n.value > 0
    small = n.value
    assert ws(grad=1) == 0 and n.value > 0
    assert ws(N=0) == 0
    for bad in (dict(N=-1), dict(D=0), dict(V=0), dict(ldx=63), dict(ldw=1),
                dict(dtype=2), dict(N=2 ** 31), dict(D=2 ** 21, ldx=2 ** 21,
                                                     ldw=2 ** 21)):
        assert ws(**bad) == 1, bad
    # too little workspace, misaligned workspace, null pointers
    assert lib.zshmc_class_log_prob(
        P, P, None, P, 3, 64, 5, 64, 64, 1, 0, 0, P, None, P, small - 1,
        None) == 1
    assert 'workspace' in _capi.last_error()
    assert lib.zshmc_class_log_prob(
        P, P, None, P, 3, 64, 5, 64, 64, 1, 0, 0, P, None,
        ctypes.c_void_p(4100), small, None) == 1
    assert lib.zshmc_class_log_prob(
        P, P, None, None, 3, 64, 5, 64, 64, 1, 0, 0, P, None, P, small,
        None) == 1
    assert lib.zshmc_class_log_prob(
        P, P, None, P, 3, 64, 5, 64, 64, 1, 0, 0, P, ctypes.c_void_p(4100), P,
        small, None) == 1
    assert lib.zshmc_class_log_prob_grad(
        P, P, None, P, 3, 64, 5, 64, 64, 1, 0, 0, None, P, P, P, P, P,
        1 << 30, None) == 1
    assert lib.zshmc_class_log_prob_grad(
        P, P, None, P, 3, 64, 5, 64, 64, 1, 0, 0, P, P, P, P, P, P, 16,
        None) == 1
    assert 'workspace' in _capi.last_error()


def test_int8_entries(lib):
    def q(n=3, k=20, ld=20, dtype=0, pitch=32, v=P):
        return lib.zshmc_quantize_rows(P, n, k, ld, dtype, v, pitch, P, None)
    assert q(n=0) == 0
    for bad in (dict(n=-1), dict(k=0), dict(ld=19), dict(dtype=3),
                dict(pitch=16), dict(pitch=40), dict(v=ctypes.c_void_p(4097)),
                dict(v=None)):
        assert q(**bad) == 1, bad
    assert lib.zshmc_dequantize_rows(P, 16, P, 3, 20, P, 20, 0, None) == 1
    assert lib.zshmc_dequantize_rows(P, 32, P, 3, 20, P, 19, 0, None) == 1
    assert lib.zshmc_dequantize_rows(P, 32, P, 0, 20, P, 20, 0, None) == 0

    def lin(xp=32, wp=32, n=3, k=20, v=7, ldo=7, dtype=0, x=P, out=P):
        return lib.zshmc_int8_linear(x, xp, P, P, wp, P, None, n, k, v, out,
                                     ldo, dtype, None)
    assert lin(n=0) == 0
    for bad in (dict(xp=16), dict(wp=40), dict(n=-1), dict(k=0), dict(v=0),
                dict(ldo=6), dict(dtype=-1), dict(x=ctypes.c_void_p(4104)),
                dict(out=None), dict(k=131073, xp=131088, wp=131088)):
        assert lin(**bad) == 1, bad
