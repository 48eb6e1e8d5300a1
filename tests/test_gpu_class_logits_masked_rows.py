"""Rows that a loss leaves out by an upstream gradient of zero -- a mask, a
sample's weight, torch.where -- rather than by ignore_label."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]
IGNORE = -100


def gradients(w, X, y, b, g, ignore=None):
    leaves = [t.detach().clone().requires_grad_() for t in (w, X, b)
              if t is not None]
    lp = zs.linear_categorical_log_prob(
        leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None,
        ignore_label=ignore)
    return lp, torch.autograd.grad(lp, leaves, g)


@pytest.mark.parametrize('ignore', [None, IGNORE])
@pytest.mark.parametrize('N', [1, 70, 300, 1100])
@pytest.mark.parametrize('dtype', BOTH)
def test_zeros_in_the_upstream_gradient(dtype, N, ignore):
    """One row of zero, a mask over n, and nothing but zeros."""
    w, X, y, b, g = problem(N, 96, 700, dtype, 70 + N, True, ignore)
    one = g.clone()
    one[N // 2] = 0
    mask = (torch.arange(N, device='cuda') % 3 == 0).float() / N
    for up in (one, mask, -1e-6 * mask, 1e6 * mask, torch.zeros_like(g)):
        lp, grads = gradients(w, X, y, b, up, ignore)
        (ref, refs), (tol, tols) = class_log_prob(w, X, y, b, ignore, up)
        within(lp, ref, tol, 'log_prob')
        for name, got, r, t in zip(('w', 'X', 'bias'), grads, refs, tols):
            within(got, r, t, name)
        assert bool((grads[1][up == 0] == 0).all())


def test_zeros_through_a_categorical():
    """A masked loss of a model whose classes are taken in pieces."""
    N, D, V = 3000, 40, 1500
    w, X, y, _, g = problem(N, D, V, torch.float32, 71)
    g[::2] = 0
    leaf = w.clone().requires_grad_()
    dist = zs.distributions.Categorical(zs.linear_class_logits(leaf, X))
    lp = dist.log_prob(y.int())
    assert dist._logits_dense is None
    got, = torch.autograd.grad((lp * g).sum(), leaf)
    (_, (dw, _, _)), (_, (tol, _, _)) = class_log_prob(w, X, y, g=g)
    within(got, dw, tol)
