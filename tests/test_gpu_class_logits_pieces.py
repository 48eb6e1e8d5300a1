"""More than one piece of classes at both ends: as many classes as a row of r
holds for few rows, and the smallest pieces that many rows are taken in."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
IGNORE = -100


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N,D,V', [
    (2, 8, 2200003),                 # 4 MB a row of r
    (40001, 16, 5003)])              # 4096 classes
def test_pieces(N, D, V, dtype):
    w, X, y, b, g = problem(N, D, V, dtype, 1, True, IGNORE)
    leaves = [t.detach().requires_grad_() for t in (w, X, b)]
    lp = zs.linear_categorical_log_prob(leaves[0], leaves[1], y,
                                        bias=leaves[2], ignore_label=IGNORE)
    grads = torch.autograd.grad(lp, leaves, g)
    (ref, refs), (tol, tols) = class_log_prob(w, X, y, b, IGNORE, g)
    # (2 200 003 classes: 134 parts a lane one after the other, 32 terms in each,
    # the rest in trees: within the helper's 300)
    within(lp, ref, tol, 'log_prob')
    for name, got, r, t in zip(('w', 'X', 'bias'), grads, refs, tols):
        within(got, r, t, name)
