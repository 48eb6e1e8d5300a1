"""Plain 64-bit forms of the linear Categorical and of the 8-bit rows, with
element-wise bounds on what the kernels may be off by."""
import math

import torch

U32 = 2.0 ** -24                 # half a step of float32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def class_log_prob(w, X, labels, bias=None, ignore=None, g=None):
    """(log_prob, [dw, dX, db]) in float64 and their tolerances, all on the
    inputs' device.

    The bounds.  A logit is a sum of D products in float32, in any order: off by
    at most D u sum|x w| (u = 2^-24).  float32 factors in two float16 parts make
    it 3 D products, hold a factor to 2^-23 (2 u) and drop the product of the
    lower parts, 2^-22 (4 u): (3 D + 8) u in all, less than (6 D + 1) u from D = 3
    on; the same for the products with r.  (What lies below 2^-38 of an operand's
    largest value is lost as well.)  log-sum-exp moves by no
    more than its arguments; its exponentials are 2^-23 (1 + |l - M|) off -- at
    the 2^-22 |l - M| <= 2^-22 * 64 where they still count -- and summed over
    at most 300 terms one after the other.  r is rounded to the operands' type
    and g p moves by its logit, M and S.  A
    product over k terms adds k u times the sum of magnitudes; the result is
    rounded once to its type."""
    wd, xd = w.detach().double(), X.detach().double()
    N, D = xd.shape
    V = wd.shape[0]
    b = 0 if bias is None else bias.detach().double()
    kept = torch.ones(N, dtype=torch.bool, device=w.device) if ignore is None \
        else labels != ignore
    xd = torch.where(kept[:, None], xd, torch.zeros_like(xd))
    logits = xd @ wd.t() + b
    idx = torch.where(kept, labels, torch.zeros_like(labels)).long()[:, None]
    lse = torch.logsumexp(logits, 1)
    zero = torch.zeros_like(lse)
    lp = torch.where(kept, logits.gather(1, idx)[:, 0] - lse, zero)
    terms = 6 * D + 1 if w.dtype == torch.float32 else D
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        # (a class that the bias takes out moves nothing)
        mag = torch.where(b > -1e30, mag + b.abs(), torch.zeros_like(mag))
    e_logit = (terms + 1) * U32 * mag.amax(1)
    e_sum = (300 + 4 * 64) * U32
    tol_lp = 2 * e_logit + e_sum + 4 * U32 * lp.abs() + 4 * U32 * \
        logits.gather(1, idx)[:, 0].abs()
    if g is None:
        return lp, tol_lp
    gd = torch.where(kept, g.double(), zero)
    p = torch.exp(logits - lse[:, None]) * gd[:, None]
    hot = torch.zeros_like(p).scatter_(1, idx, gd[:, None])
    r = hot - p
    half = HALF[w.dtype]
    e_r = half * r.abs() + p.abs() * (2 * e_logit + e_sum)[:, None] + \
        2 * U32 * (p.abs() + hot.abs())
    k = 6 if w.dtype == torch.float32 else 1
    dw, dx = r.t() @ xd, r @ wd
    tol_w = e_r.t() @ xd.abs() + (k * N + 1) * U32 * (r.abs().t() @ xd.abs()) \
        + half * dw.abs()
    tol_x = e_r @ wd.abs() + (k * V + 1) * U32 * (r.abs() @ wd.abs()) + \
        half * dx.abs()
    db = r.sum(0)
    # (the bias' gradient is summed before r is rounded)
    e_b = p.abs() * (2 * e_logit + e_sum)[:, None] + \
        (2 + N) * U32 * (p.abs() + hot.abs())
    tiny = 1e-37                     # results below float32's smallest
    return (lp, [dw, dx, db]), (tol_lp, [tol_w + tiny, tol_x + tiny,
                                         e_b.sum(0) + tiny])


def within(got, ref, tol, what=''):
    got = got.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (
        what, int(bad.sum()), 'of', bad.numel(), 'worst',
        float((off / tol.clamp_min(1e-300)).max()), 'of its bound')


def problem(N, D, V, dtype, seed=0, bias=False, ignore=None, device='cuda'):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=gen) * 2 / math.sqrt(D)).to(dtype)
    X = torch.randn(N, D, generator=gen).to(dtype)
    y = torch.randint(V, (N,), generator=gen)
    if ignore is not None and N > 1:
        y[::3] = ignore
    b = torch.randn(V, generator=gen) if bias else None
    g = 0.5 + torch.rand(N, generator=gen)
    return tuple(None if t is None else t.to(device)
                 for t in (w, X, y, b, g))


def quantized(x):
    """(whole numbers, scale) of rows of x: float32 by definition."""
    x = x.detach().float()
    most = x.abs().amax(-1, keepdim=True)
    s = most / torch.full_like(most, 127.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    return torch.round(x / s).clamp(-127, 127), s
