"""What zs.linear_categorical_log_prob is off by, as independent roundings.  float32
operands are float32 to the last bit that a float32 evaluation has: rows, features and upstream gradients of
very different sizes, rare classes, infinite and extreme weights.

helpers_class_logits bounds the worst case, K roundings of a sum of K terms all one
way, in which a lost part of a product can hide.  Here the roundings are independent:
their variances are added up (`spread`), and the root mean square of the error, over a
result or over each of its rows, is at most 4 times the root of the sum's mean.  u =
2^-24; a rounding is at most u of its value, so its variance is at most u^2 of its square.
  a sum of K products t_k, one after the other: its partial sums are at most of the
    size of k independent terms and of k / K of the whole, so that K roundings
    add u^2 K (sum t^2 / 2 + (sum t)^2 / 3), at u^2 / 3 a rounding that is spread
    evenly; K u^2 / 4 of both is more.  (Taken in blocks it is less.)
  e^x as 2^(x log2 e): the product and its constant are 2 u |x| off, the power 2 u;
  the softmax' sum: 64 terms one after the other, the rest in trees;
  r: four roundings of its two parts; every result one more."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
IGNORE = -100


def ours(w, X, y, b=None, g=None, ignore=None):
    leaves = [t.detach().clone().requires_grad_() for t in (w, X, b)
              if t is not None]
    lp = zs.linear_categorical_log_prob(
        leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None,
        ignore_label=ignore)
    return [lp.detach()] + list(torch.autograd.grad(lp, leaves, g))


def plain(w, X, y, b, g, dtype):
    """The definition in torch operations of `dtype`."""
    w, X, g = w.to(dtype), X.to(dtype), g.to(dtype)
    l = X @ w.t()
    if b is not None:
        l = l + b.to(dtype)
    m = l.amax(1, keepdim=True)
    lse = m + (l - m).exp().sum(1, keepdim=True).log()
    lp = (l.gather(1, y[:, None]) - lse)[:, 0]
    r = (l - lse).exp() * -g[:, None]
    r.scatter_add_(1, y[:, None], g[:, None])
    out = [lp, r.t() @ X, r @ w]
    return out if b is None else out + [r.sum(0)]


def spread(w, X, y, b, g):
    """Variances of log_prob, dw, dX and db, see above.  bfloat16 operands: r, dw
    and dX are rounded to it, half a step, 2^-8, at most (db sums r before that)."""
    half = 2.0 ** 32 if w.dtype == torch.bfloat16 else 0.
    w, X, g = w.double(), X.double(), g.double()[:, None]
    N, D = X.shape
    V = w.shape[0]
    l = X @ w.t()
    v_l = D / 4 * ((X * X) @ (w * w).t() + l * l)
    if b is not None:
        l = l + b.double()
        v_l = v_l + torch.where(l.isinf(), torch.zeros_like(l), l * l)
    hot = torch.zeros_like(l).scatter_(1, y[:, None], 1.)
    m = l.amax(1, keepdim=True)
    v_e = torch.where(l.isinf(), torch.zeros_like(l),
                      (2 + 2 * (l - m).abs()).square())
    p = (l - torch.logsumexp(l, 1, keepdim=True)).exp()
    v_lse = (p * p * (v_l + v_e)).sum(1, keepdim=True) + 64 + 8
    at = l.gather(1, y[:, None])
    lp = at - m - (l - m).exp().sum(1, keepdim=True).log()
    v_lp = v_l.gather(1, y[:, None]) + v_lse + (at - m).square() + \
        lp.square()
    r = g * (hot - p)
    v_p = v_l + v_e + v_lse
    v_r = (g * p).square() * v_p + 4 * g * g * (hot + p * p)
    x2, w2, r2 = X * X, w * w, r * r
    dw, dx, db = r.t() @ X, r @ w, r.sum(0)
    v_b = v_r.sum(0) + N / 4 * (r2.sum(0) + db * db) + db * db
    v_r = v_r + half * r2
    v_w = v_r.t() @ x2 + N / 4 * (r2.t() @ x2 + dw * dw) + (1 + half) * dw * dw
    # (a row's log-sum-exp is off for all of its classes alike)
    v_x = v_r @ w2 + V / 4 * (r2 @ w2 + dx * dx) + (1 + half) * dx * dx + \
        v_lse * ((g * p) @ w).square()
    return [2.0 ** -48 * v for v in (v_lp[:, 0], v_w, v_x, v_b)]


def as_good_as_float32(got, w, X, y, b, g, rows=False):
    ref = plain(w, X, y, b, g, torch.float64)
    for name, a, r, v in zip(('log_prob', 'w', 'X', 'bias'), got, ref,
                             spread(w, X, y, b, g)):
        off, var = (a.double() - r).square(), v
        if rows and r.dim() == 2:
            off, var = off.mean(1), var.mean(1)
        elif not rows:
            off, var = off.mean(), var.mean()
        ratio = (off / (var + 1e-74)).sqrt()
        assert bool((ratio <= 4).all()), (
            name, int((~(ratio <= 4)).sum()), 'of', ratio.numel(), 'worst',
            float(ratio.max()))


def check(w, X, y, b, g, rows=False):
    as_good_as_float32(ours(w, X, y, b, g), w, X, y, b, g, rows)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N,D,V', [
    (20, 96, 700),                   # 32 rows a tile
    (60, 96, 700),                   # 64
    (70, 1200, 130),                 # few tiles
    (81, 64, 300), (129, 72, 4099), (270, 100, 12419), (600, 130, 1000),
    (700, 256, 4000), (1021, 784, 1237), (2000, 300, 20000),
    (9001, 64, 15001)])              # pieces
def test_no_part_of_a_product_is_lost(N, D, V, dtype):
    for bias in (False, True):
        check(*problem(N, D, V, dtype, N + D, bias))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N,D,V', [(7, 2816, 1029), (300, 2500, 130),
                                   (700, 2048, 260)])
def test_no_part_is_lost_of_many_features(N, D, V, dtype):
    check(*problem(N, D, V, dtype, N + D, True))


@pytest.mark.parametrize('N', [60, 300, 900])
@pytest.mark.parametrize('size', [1e9, 1e25])
def test_a_row_far_larger_than_the_others_and_w(N, size):
    """It moves two classes' rows of dw; the others' are what they are
    without it."""
    w, X, y, _, g = problem(N, 96, 700, torch.float32, 57)
    X2 = X.clone()
    X2[7] *= size
    got = ours(w, X2, y, None, g)
    touched = torch.zeros(700, dtype=torch.bool, device='cuda')
    touched[y[7]] = True
    touched[(X2[7].double() @ w.double().t()).argmax()] = True
    keep = torch.arange(N, device='cuda') != 7
    args = (w, X[keep], y[keep], None, g[keep])
    ref = plain(*args, torch.float64)[1]
    off = (got[1].double() - ref).square().mean(1)
    var = spread(*args)[1].mean(1)
    assert bool((off <= 16 * var)[~touched].all()), float(
        (off / var)[~touched].max())
    as_good_as_float32([got[0][keep], ref, got[2][keep]], *args)


@pytest.mark.parametrize('N', [60, 300, 900])
def test_an_upstream_gradient_far_larger_than_the_others(N):
    w, X, y, _, g = problem(N, 96, 700, torch.float32, 58)
    g[5] *= 2.0 ** 24
    check(w, X, y, None, g, rows=True)
    g[5] *= 2.0 ** 30
    check(w, X, y, None, g, rows=True)


@pytest.mark.parametrize('N', [60, 300, 900])
def test_rare_classes_keep_their_rows(N):
    """A peaked softmax: classes of probability 1e-7 to 1e-35, whose rows of dw
    an optimiser that normalises by row or element sees at full size."""
    w, X, y, b, g = problem(N, 96, 700, torch.float32, 59, True)
    b[350:] -= torch.linspace(10., 80., 350, device='cuda')
    y = y % 350
    check(w, X, y, b, g, rows=True)


@pytest.mark.parametrize('N', [60, 300, 900])
def test_features_of_very_different_sizes(N):
    """Features from 2^-40 to 2^40 with the weights that make up for it."""
    w, X, y, _, g = problem(N, 96, 700, torch.float32, 60)
    s = torch.tensor([2.0 ** (k % 9 * 10 - 40) for k in range(96)],
                     device='cuda')
    got, ref = ours(w / s, X * s, y, None, g), ours(w, X, y, None, g)
    # powers of two: the same roundings
    assert torch.equal(got[0], ref[0])
    assert torch.equal(got[1], ref[1] * s) and torch.equal(got[2], ref[2] / s)


@pytest.mark.parametrize('N', [60, 300, 900])
def test_classes_of_very_different_sizes(N):
    """A class 2^40 larger in w changes no bit of the others' logits."""
    w, X, y, b, g = problem(N, 96, 700, torch.float32, 61, True)
    w2 = w.clone()
    w2[5] *= 2.0 ** 40
    b2 = b.clone()
    b2[5] = b[5] = -float('inf')
    y = torch.where(y == 5, torch.zeros_like(y), y)
    got, ref = ours(w2, X, y, b2, g), ours(w, X, y, b, g)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize('N', [60, 300, 900])
def test_sizes_whose_product_float32_does_not_hold(N):
    """Largest values of 2^100 and 2^60 that never meet, with logits of 0 and
    of ordinary size."""
    w, X, y, _, g = problem(N, 96, 700, torch.float32, 63)
    X, w = X.clone(), w.clone()
    X[:, :32] = 2.0 ** 100
    w[:, :32] = 0
    w[0] = 0
    X[:, 32:64] *= 2.0 ** -60
    w[:, 32:64] *= 2.0 ** 60
    lp, gw, gx = ours(w, X, y, None, g)
    (ref, _), (tol, _) = class_log_prob(w, X, y, g=g)
    within(lp, ref, tol)
    ref = plain(w, X, y, None, g, torch.float64)
    var = spread(w, X, y, None, g)
    for a, r, v in ((gw, ref[1], var[1]), (gx, ref[2], var[2])):
        for part in (slice(0, 32), slice(32, 64), slice(64, 96)):
            off = (a.double() - r)[:, part].square().mean()
            assert bool(off <= 16 * v[:, part].mean() + 1e-74), part


def test_through_a_categorical():
    N, D, V = 3000, 40, 1500
    w, X, y, _, g = problem(N, D, V, torch.float32, 64)
    leaf = w.clone().requires_grad_()
    lp = zs.distributions.Categorical(
        zs.linear_class_logits(leaf, X)).log_prob(y.int())
    gw, = torch.autograd.grad(lp, leaf, g)
    as_good_as_float32([lp.detach(), gw], w, X, y, None, g)


# Sums of one product each, in operands of 24 bits: a part of the product that is
# lost, 2^-18 of it and more, cannot hide in the roundings of a long sum.
ONE = [(20, 300), (60, 300), (129, 700), (300, 700), (600, 1000), (1021, 1237),
       (2100, 20000)]


def off(got, ref, rel, extra=0.):
    bad = (got.double() - ref).abs() > rel * ref.abs() + extra
    assert not bool(bad.any()), (int(bad.sum()), float(
        ((got.double() - ref).abs() / ref.abs()).nan_to_num(0.).max()))


def diagonal(N, dtype=torch.float32, seed=0):
    """[N, N] with random values on the diagonal, and N random numbers."""
    gen = torch.Generator().manual_seed(seed)
    x = (0.5 + torch.rand(N, generator=gen)).to(dtype)
    return torch.diag(x).cuda(), (0.5 + torch.rand(N, generator=gen)).cuda(), \
        torch.randperm(1 << 20, generator=gen)[:N].cuda()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N,V', ONE)
def test_single_products_in_the_logits(N, V, dtype):
    """Row n has one feature; its label's class a weight of about -1000 there,
    the others 0, so that log_prob is that product less log(V - 1): a rounding
    of the product, of its difference to 0 and of log_prob, at most 6 u with what
    the planes leave out, and log(V - 1) < 16 from a sum that is exact."""
    X, v, y = diagonal(N, dtype)
    y = y % V
    w = torch.zeros(V, N, device='cuda')
    w[y, torch.arange(N, device='cuda')] = -1000 * v
    w = w.to(dtype)
    lp = zs.linear_categorical_log_prob(w, X, y)
    l = X.diagonal().double() * w[y, torch.arange(N, device='cuda')].double()
    ref = l - torch.log(V - 1 + l.exp())
    off(lp, ref, 6 * 2.0 ** -24, 16 * 2.0 ** -23)


@pytest.mark.parametrize('N,V', ONE)
def test_single_products_in_the_gradient_of_w(N, V):
    """w = 0: r = g ([v == y] - 1 / V), four roundings; dw has one product an
    element, at most 2 u with what the planes leave out, and one rounding."""
    X, g, y = diagonal(N, seed=1)
    y = y % V
    w = torch.zeros(V, N, device='cuda', requires_grad=True)
    dw, = torch.autograd.grad(zs.linear_categorical_log_prob(w, X, y), w, g)
    r = torch.full((N, V), -1. / V, dtype=torch.float64, device='cuda')
    r[torch.arange(N, device='cuda'), y] += 1
    off(dw, (r * (g.double() * X.diagonal().double())[:, None]).t(),
        8 * 2.0 ** -24)


@pytest.mark.parametrize('N,V', ONE)
def test_single_products_in_the_gradient_of_X(N, V):
    """X = 0, and each feature has a weight in one class."""
    gen = torch.Generator().manual_seed(2)
    D = 200
    at = torch.randperm(V, generator=gen)[:D].cuda()
    w = torch.zeros(V, D, device='cuda')
    w[at, torch.arange(D, device='cuda')] = (
        0.5 + torch.rand(D, generator=gen)).cuda()
    _, g, y = diagonal(N, seed=3)
    y = y % V
    X = torch.zeros(N, D, device='cuda', requires_grad=True)
    dx, = torch.autograd.grad(zs.linear_categorical_log_prob(w, X, y), X, g)
    r = torch.full((N, V), -1. / V, dtype=torch.float64, device='cuda')
    r[torch.arange(N, device='cuda'), y] += 1
    ref = g.double()[:, None] * r[:, at] * w[
        at, torch.arange(D, device='cuda')].double()
    off(dx, ref, 8 * 2.0 ** -24)
