"""Categorical over the class logits of no chains at all."""
import pytest
import torch

import zhusuan_amd as zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('N', [10, 3000])
def test_no_chains(N):
    w = torch.zeros(0, 1500, 40, device='cuda', requires_grad=True)
    X = torch.zeros(N, 40, device='cuda')
    y = torch.zeros(N, dtype=torch.int32, device='cuda')
    lp = zs.distributions.Categorical(zs.linear_class_logits(w, X)).log_prob(y)
    assert lp.shape == (0, N)
    gw, = torch.autograd.grad(lp.sum(), w)
    assert gw.shape == w.shape
