"""A class that a constant feature's infinite weight takes out of
zs.linear_categorical_log_prob: its r is 0 in every row, and in the rows behind
the last one and the ignored ones too, where 0 times the weight is no number."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
IGNORE = -100


def ours(w, X, y, b, g, ignore):
    leaves = [t.detach().clone().requires_grad_() for t in (w, X, b)]
    lp = zs.linear_categorical_log_prob(leaves[0], leaves[1], y,
                                        bias=leaves[2], ignore_label=ignore)
    return [lp.detach()] + list(torch.autograd.grad(lp, leaves, g))


@pytest.mark.parametrize('ignore', [None, IGNORE])
@pytest.mark.parametrize('dtype,N', [
    (torch.bfloat16, 61), (torch.bfloat16, 301), (torch.bfloat16, 901),
    (torch.float32, 61), (torch.float32, 301), (torch.float32, 901)])
def test_infinite_weights_mask_a_class(dtype, N, ignore):
    """A constant feature whose weight is -inf (or the type's lowest) takes a
    class out, like a bias: the others' results are those without it."""
    w, X, y, b, g = problem(N, 96, 700, dtype, 62, True, ignore)
    X[:, 40] = 1.
    gone = torch.arange(700, device='cuda') % 9 == 4
    y = torch.where((y % 9 == 4) & (y != IGNORE), torch.zeros_like(y), y)
    w0 = w.clone()
    w0[gone, 40] = 0
    b0 = torch.where(gone, torch.full_like(b, -float('inf')), b)
    ref = ours(w0, X, y, b0, g, ignore)
    for low in (-float('inf'), torch.finfo(dtype).min):
        w[gone, 40] = low
        got = ours(w, X, y, b, g, ignore)
        (lp64, _), (tol, _) = class_log_prob(w0, X, y, b0, ignore, g)
        within(got[0], lp64, tol, low)
        for a, c in ((got[1], ref[1]), (got[3], ref[3])):
            assert bool((a[gone] == 0).all())
            assert bool(a.isfinite().all())
        if low == -float('inf'):     # (finite ones may round otherwise)
            assert torch.equal(got[0], ref[0])
            assert torch.equal(got[1], ref[1])
            assert torch.equal(got[3], ref[3])


@pytest.mark.parametrize('N', [61, 301, 901])
def test_an_infinite_feature_stays_in_its_row(N):
    w, X, y, b, g = problem(N, 96, 700, torch.float32, 63, True)
    ref = ours(w, X, y, b, g, None)
    X2 = X.clone()
    X2[2, 5], X2[40, 90] = float('inf'), -float('inf')
    got = ours(w, X2, y, b, g, None)
    bad = torch.zeros(N, dtype=torch.bool, device='cuda')
    bad[2] = bad[40] = True
    assert torch.equal(got[0].isnan(), bad)
    assert torch.equal(got[0][~bad], ref[0][~bad])
    assert torch.equal(got[2][~bad], ref[2][~bad])
    assert bool(got[2][bad].isnan().all()) and bool(got[1].isnan().all())
