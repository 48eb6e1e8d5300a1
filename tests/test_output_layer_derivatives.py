"""Derivatives that the output layer's operators do not have are refused, not
dropped: forward-mode tangents, and any derivative through 8-bit rows.  On the
CPU, up to the first call of an entry point."""
import pytest
import torch
from torch.autograd import forward_ad

import zhusuan_amd as zs
from zhusuan_amd import _ops

N, D, V = 5, 16, 7


class Reached(Exception):
    pass


@pytest.fixture
def stub(monkeypatch):
    def on_device(device):
        raise Reached()
    monkeypatch.setattr(_ops._capi, 'on_device', on_device)
    monkeypatch.setattr(_ops, 'require_device', lambda *t: None)


def tensors():
    return dict(w=torch.randn(V, D), X=torch.randn(N, D),
                bias=torch.randn(V))


def score(t):
    return zs.linear_categorical_log_prob(t['w'], t['X'],
                                          torch.zeros(N, dtype=torch.int64),
                                          bias=t['bias'])


def answer(t):
    rows = zs.QuantizedRows(torch.zeros(V, D, dtype=torch.int8),
                            t.get('scale', torch.ones(V)))
    return zs.quantized_linear(rows, t['X'], bias=t['bias'])


def answer_rows(t):
    rows = zs.QuantizedRows(torch.zeros(V, D, dtype=torch.int8),
                            torch.ones(V))
    X = zs.QuantizedRows(torch.zeros(N, D, dtype=torch.int8),
                         t.get('scale', torch.ones(N)))
    return zs.quantized_linear(rows, X)


def back(t):
    return zs.QuantizedRows(torch.zeros(V, D, dtype=torch.int8),
                            t.get('scale', torch.ones(V))).dequantize()


CASES = [(score, 'w'), (score, 'X'), (score, 'bias'),
         (lambda t: zs.quantize_rows(t['X']), 'X'),
         (answer, 'X'), (answer, 'bias'), (answer, 'scale'),
         (answer_rows, 'scale'), (back, 'scale')]


@pytest.mark.parametrize('call,which', CASES)
def test_forward_mode_tangents(stub, call, which):
    t = tensors()
    t['scale'] = torch.ones(N if call is answer_rows else V)
    with pytest.raises(Reached):
        call(t)
    with forward_ad.dual_level():
        with pytest.raises(Reached):          # (a level alone is no tangent)
            call(t)
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        for grad_mode in (torch.enable_grad(), torch.no_grad()):
            with grad_mode, pytest.raises(RuntimeError, match='forward-mode'):
                call(t)
    t = tensors()
    if which != 'scale':
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda v: call(dict(t, **{which: v})),
                           (t[which],), (torch.ones_like(t[which]),))


@pytest.mark.parametrize('call,which', CASES[3:])
def test_gradients_through_8_bit_rows(stub, call, which):
    t = tensors()
    t['scale'] = torch.ones(N if call is answer_rows else V)
    t[which].requires_grad_()
    with pytest.raises(RuntimeError, match='gradient'):
        call(t)
    with torch.no_grad(), pytest.raises(Reached):
        call(t)
    t[which] = t[which].detach()
    with pytest.raises(Reached):
        call(t)
