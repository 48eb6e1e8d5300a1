"""zs.linear_categorical_log_prob under torch.autograd.graph's hooks."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_saved_tensors_that_come_back_compact(dtype):
    """save_on_cpu gives the gradient call compact copies of rows that the
    forward call read inside a wider buffer."""
    w, X, y, b, g = problem(90, 64, 410, dtype, 63, True, -100)
    wide = torch.zeros(90, 400, device='cuda', dtype=dtype)
    wide[:, 8:72] = X
    tall = torch.zeros(410, 136, device='cuda', dtype=dtype)
    tall[:, 72:] = w

    def run(w, X):
        leaves = [t.detach().requires_grad_() for t in (w, X, b)]
        lp = zs.linear_categorical_log_prob(leaves[0], leaves[1], y,
                                            bias=leaves[2], ignore_label=-100)
        return (lp,) + torch.autograd.grad(lp, leaves, g)
    ref = run(w, X)
    with torch.autograd.graph.save_on_cpu():
        got = run(tall[:, 72:], wide[:, 8:72])
    for a, c in zip(got, ref):
        assert torch.equal(a, c)
