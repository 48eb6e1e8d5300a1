"""The gradient call of zs.linear_categorical_log_prob describes to the C entry
the tensors that it holds THEN: saved-tensor hooks (torch.autograd.graph) give
back copies with other strides, or anything at all.  On the CPU, with the
entry points recorded instead of called."""
import ctypes

import pytest
import torch

from zhusuan_amd import _ops

N, D, V = 6, 16, 9


class _Stream(object):
    def __init__(self, device):
        pass

    def __enter__(self):
        return 0

    def __exit__(self, *exc):
        pass


@pytest.fixture
def calls(monkeypatch):
    made = []

    def call(name, *args):
        made.append((name, args))
        if name == 'zshmc_class_log_prob_workspace':
            ctypes.c_int64.from_address(args[-1]).value = 64
    monkeypatch.setattr(_ops._capi, 'call', call)
    monkeypatch.setattr(_ops._capi, 'on_device', _Stream)
    monkeypatch.setattr(_ops, 'require_device', lambda *t: None)
    monkeypatch.setattr(_ops, '_class_workspace', {})
    return made


def sliced(rows):
    return torch.randn(rows, 100)[:, 20:20 + D].requires_grad_()


@pytest.mark.parametrize('which', ['X', 'w', 'both'])
def test_strides_are_those_of_the_tensors_that_came_back(calls, which):
    X = sliced(N) if which != 'w' else torch.randn(N, D, requires_grad=True)
    w = sliced(V) if which != 'X' else torch.randn(V, D, requires_grad=True)
    y = torch.zeros(N, dtype=torch.int64)
    back = []

    def unpack(t):
        t = t.clone(memory_format=torch.contiguous_format)
        back.append(t)
        return t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(),
                                                  unpack):
        lp = _ops.linear_categorical_log_prob(w, X, y)
    forward = dict(calls)['zshmc_class_log_prob']
    assert forward[4:9] == (N, D, V, X.stride(0), w.stride(0))
    del calls[:]
    torch.autograd.grad(lp.sum(), (w, X))
    made = dict(calls)
    gradient = made['zshmc_class_log_prob_grad']
    # a compact copy of either, and its own pitch
    assert gradient[4:9] == (N, D, V, D, D)
    assert {gradient[0], gradient[1]} <= {t.data_ptr() for t in back}
    # ... and the workspace of exactly that layout
    space = made['zshmc_class_log_prob_workspace']
    assert space[0:2] == gradient[0:2] and space[2:7] == gradient[4:9]


@pytest.mark.parametrize('change', [
    lambda t: t.half() if t.dtype == torch.float32 else t,
    lambda t: t[..., :1] if t.dim() == 2 else t,
    lambda t: t[:1],
    lambda t: t.int() if t.dtype == torch.int64 else t,
])
def test_tensors_of_another_kind_are_refused(calls, change):
    X, w = sliced(N), sliced(V)
    b = torch.zeros(V)
    y = torch.zeros(N, dtype=torch.int64)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(),
                                                  change):
        lp = _ops.linear_categorical_log_prob(w, X, y, bias=b)
    with pytest.raises(RuntimeError, match='saved'):
        torch.autograd.grad(lp.sum(), (w, X))
    assert 'zshmc_class_log_prob_grad' not in dict(calls)


def test_other_strides_of_labels_bias_and_statistics(calls):
    """Read as dense arrays, whatever strides they come back with."""
    X, w = sliced(N), sliced(V)
    b = torch.arange(V, dtype=torch.float32)
    y = torch.arange(N)

    def spread(t):
        wide = torch.zeros(t.shape + (2,), dtype=t.dtype)
        wide[..., 0] = t
        return wide[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(),
                                                  spread):
        lp = _ops.linear_categorical_log_prob(w, X, y, bias=b)
    seen = {}

    def call(name, *args):
        if name == 'zshmc_class_log_prob_workspace':
            ctypes.c_int64.from_address(args[-1]).value = 64
        else:
            seen['bias'] = list((ctypes.c_float * V).from_address(args[2]))
            seen['labels'] = list((ctypes.c_int64 * N).from_address(args[3]))
            seen['x'] = list((ctypes.c_float * D).from_address(
                args[0] + 4 * args[7]))
    _ops._capi.call = call
    torch.autograd.grad(lp.sum(), (w, X))
    assert seen['bias'] == b.tolist() and seen['labels'] == y.tolist()
    assert seen['x'] == X[1].tolist()
