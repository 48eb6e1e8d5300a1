"""Labels outside the classes: NaN where the row counts, nothing where the
caller has taken the row out (torch.where over a padding label)."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize('N', [40, 300])
@pytest.mark.parametrize('dtype', BOTH)
def test_masked_labels_have_no_part(dtype, N):
    w, X, y, b, g = problem(N, 64, 300, dtype, 80, True)
    pad = torch.arange(N, device='cuda') % 7 == 3
    y2 = torch.where(pad, torch.full_like(y, -1), y)
    y2[3] = 300
    leaves = [t.clone().requires_grad_() for t in (w, X, b)]
    lp = zs.linear_categorical_log_prob(leaves[0], leaves[1], y2,
                                        bias=leaves[2])
    assert torch.equal(lp.isnan(), pad)
    loss = (torch.where(pad, torch.zeros_like(lp), lp) * g).sum()
    grads = torch.autograd.grad(loss, leaves)
    kept = torch.where(pad, torch.zeros_like(g), g)
    (_, refs), (_, tols) = class_log_prob(w, X, y, b, None, kept)
    for name, got, r, t in zip(('w', 'X', 'bias'), grads, refs, tols):
        within(got, r, t, name)
    assert bool((grads[1][pad] == 0).all())
    # ... and NaN as soon as one of them counts
    g2 = kept.clone()
    g2[3] = 1.
    lp = zs.linear_categorical_log_prob(leaves[0], leaves[1], y2,
                                        bias=leaves[2])
    gw, gx, gb = torch.autograd.grad(lp, leaves, g2)
    assert bool(gw.isnan().all()) and bool(gb.isnan().all())
    assert torch.equal(gx.isnan().all(1), torch.arange(N, device='cuda') == 3)


def test_padding_labels_through_a_categorical():
    """The same program below and above the size from which the classes are
    taken in pieces."""
    for N in (500, 3000):
        w, X, y, _, g = problem(N, 40, 1500, torch.float32, 81)
        pad = torch.arange(N, device='cuda') % 5 == 0
        y2 = torch.where(pad, torch.full_like(y, -1), y)
        leaf = w.clone().requires_grad_()
        lp = zs.distributions.Categorical(
            zs.linear_class_logits(leaf, X)).log_prob(y2.int())
        assert torch.equal(lp.isnan(), pad)
        got, = torch.autograd.grad(
            (torch.where(pad, torch.zeros_like(lp), lp) * g).sum(), leaf)
        kept = torch.where(pad, torch.zeros_like(g), g)
        (_, (dw, _, _)), (_, (tol, _, _)) = class_log_prob(w, X, y, g=kept)
        within(got, dw, tol)
