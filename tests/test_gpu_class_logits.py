"""zs.linear_categorical_log_prob (csrc/class_logits.hip) against its plain
form in 64 bits, with the element-wise bounds of helpers_class_logits."""
import math

import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import U32, class_log_prob, problem, within

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]
IGNORE = -100


def run(w, X, y, b, g, ignore=None):
    leaves = [t.detach().clone(memory_format=torch.preserve_format)
              .requires_grad_() if t.is_contiguous() else
              t.detach().requires_grad_() for t in (w, X, b) if t is not None]
    lp = zs.linear_categorical_log_prob(
        leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None,
        ignore_label=ignore)
    return lp, torch.autograd.grad(lp, leaves, g)


def check(w, X, y, b, g, ignore=None):
    lp, grads = run(w, X, y, b, g, ignore)
    (ref, refs), (tol, tols) = class_log_prob(w, X, y, b, ignore, g)
    within(lp, ref, tol, 'log_prob')
    for name, got, r, t in zip(('w', 'X', 'bias'), grads, refs, tols):
        within(got, r, t, name)
    return lp, grads


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('N,D,V', [
    (1, 1, 1), (1, 64, 128), (2, 7, 3), (5, 8, 257), (31, 64, 300),
    (32, 130, 129), (33, 128, 500), (64, 100, 777), (65, 200, 1000), (129, 72, 4099),
    (81, 64, 300), (100, 128, 12419), (260, 60, 1000), (300, 256, 40000),
    (1021, 784, 1237)])
def test_log_prob_and_gradients(N, D, V, dtype):
    for bias, ignore in ((False, None), (True, IGNORE)):
        w, X, y, b, g = problem(N, D, V, dtype, N + D + V, bias, ignore)
        check(w, X, y, b, g, ignore)


@pytest.mark.parametrize('dtype,N,V', [(torch.bfloat16, 8192, 20000),
                                       (torch.float32, 6001, 9001)])
def test_several_pieces_of_the_vocabulary(dtype, N, V):
    w, X, y, b, g = problem(N, 64, V, dtype, 3, True, IGNORE)
    check(w, X, y, b, g, IGNORE)


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('N,D,V', [
    (1, 1024, 5), (7, 2816, 1029), (32, 1000, 500), (33, 1539, 640),
    (128, 2048, 300), (300, 1200, 130)])
def test_few_logits_of_many_features(N, D, V, dtype):
    """Logits in parts, a share of the features each."""
    for bias, ignore in ((False, None), (True, IGNORE)):
        w, X, y, b, g = problem(N, D, V, dtype, N + D, bias, ignore)
        if bias:
            b[V // 2] = -float('inf')
            y[y == V // 2] = 0
            X[y == IGNORE] = float('nan')
        check(w, X, y, b, g, ignore)


@pytest.mark.parametrize('dtype', BOTH)
def test_ignored_rows_may_hold_anything(dtype):
    w, X, y, b, g = problem(70, 96, 333, dtype, 5, True, IGNORE)
    clean = run(w, X, y, b, g, IGNORE)
    X2 = X.clone()
    X2[y == IGNORE] = float('nan')
    X2[0] = float('inf')
    g2 = g.clone()
    g2[y == IGNORE] = float('nan')
    lp, grads = run(w, X2, y, b, g2, IGNORE)
    assert torch.equal(lp, clean[0])
    for a, c in zip(grads, clean[1]):
        assert torch.equal(a, c)
    assert bool((lp[y == IGNORE] == 0).all())
    assert bool((grads[1][y == IGNORE] == 0).all())


@pytest.mark.parametrize('N', [70, 300])
@pytest.mark.parametrize('dtype', BOTH)
def test_ignored_rows_set_no_scale(dtype, N):
    """Finite, but 1e30 times the others."""
    w, X, y, b, g = problem(N, 96, 333, dtype, 5, True, IGNORE)
    X = X.clone()
    X[y == IGNORE] = 1e30
    g[y == IGNORE] = 1e30
    check(w, X, y, b, g, IGNORE)


def test_rows_of_different_sizes():
    """float32 rows from 2^-12 to 2^12 times the others, in X, w and g: every
    result within its own row's bound (float16 planes hold 2^-38 of an
    operand's largest value)."""
    for N in (60, 300):
        w, X, y, b, g = problem(N, 96, 700, torch.float32, 55)
        k = torch.arange(N, device='cuda') % 5 - 2
        X = X * 2.0 ** (4 * k[:, None].clamp(max=0)).float()
        g = g * 2.0 ** (6 * k).float()
        w = w * 2.0 ** (4.0 * (torch.arange(700, device='cuda') % 4 - 3)
                        )[:, None].float()
        check(w, X, y, b, g)


def test_a_row_far_larger_than_the_others():
    """One row of 1e25: the others' log-probabilities, and their rows of dX,
    are what they are without it."""
    w, X, y, b, g = problem(300, 96, 700, torch.float32, 57, bias=True)
    X2 = X.clone()
    X2[7] *= 1e25
    others = torch.arange(300, device='cuda') != 7
    got = []
    for x in (X, X2):
        x = x.clone().requires_grad_()
        lp = zs.linear_categorical_log_prob(w, x, y, bias=b)
        got.append((lp.detach()[others],
                    torch.autograd.grad(lp, x, g)[0][others]))
    assert torch.equal(got[0][0], got[1][0])
    assert torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize('dtype', BOTH)
def test_every_row_ignored(dtype):
    w, X, y, b, g = problem(20, 64, 100, dtype, 6, True)
    y = torch.full_like(y, 7)
    lp, grads = run(w, X, y, b, g, ignore=7)
    assert bool((lp == 0).all())
    assert all(bool((t == 0).all()) for t in grads)


@pytest.mark.parametrize('dtype', BOTH)
def test_masked_classes(dtype):
    """A bias of -inf takes a class out: its probability and its gradients are
    zero; a row whose label it is has -inf; float32's lowest does the same."""
    w, X, y, b, g = problem(40, 64, 600, dtype, 7, True)
    b[256:520] = -float('inf')          # whole tiles among them
    b[3] = torch.finfo(torch.float32).min
    y = (y % 200) + 4                   # labels that stay
    lp, grads = check(w, X, y, b, g)
    assert bool((grads[0][256:520] == 0).all())
    assert bool((grads[2][256:520] == 0).all())
    y2 = y.clone()
    y2[5] = 300
    lp2, _ = run(w, X, y2, b, g)
    assert float(lp2[5]) == -float('inf')
    keep = torch.arange(40, device='cuda') != 5
    assert torch.equal(lp2[keep], lp[keep])
    b[:] = -float('inf')                # nothing is left: no distribution
    lp3 = zs.linear_categorical_log_prob(w, X, y, bias=b)
    assert bool(lp3.isnan().all())


@pytest.mark.parametrize('dtype', BOTH)
def test_labels_outside(dtype):
    w, X, y, b, g = problem(40, 64, 300, dtype, 8)
    ref = run(w, X, y, b, g)
    y2 = y.clone()
    y2[3], y2[35] = 300, -1
    lp, (gw, gx) = run(w, X, y2, b, g)
    bad = torch.zeros(40, dtype=torch.bool, device='cuda')
    bad[3] = bad[35] = True
    assert torch.equal(lp.isnan(), bad)
    assert torch.equal(gx.isnan().all(1), bad)
    assert torch.equal(lp[~bad], ref[0][~bad])
    assert torch.equal(gx[~bad], ref[1][1][~bad])
    assert bool(gw.isnan().all())


@pytest.mark.parametrize('dtype', BOTH)
def test_nonfinite_rows_stay_their_own(dtype):
    w, X, y, b, g = problem(34, 64, 300, dtype, 9)
    ref = run(w, X, y, b, g)
    X2 = X.clone()
    X2[2, 5] = float('nan')
    lp, (gw, gx) = run(w, X2, y, b, g)
    bad = torch.zeros(34, dtype=torch.bool, device='cuda')
    bad[2] = True
    assert torch.equal(lp.isnan(), bad) and torch.equal(lp[~bad], ref[0][~bad])
    assert torch.equal(gx[~bad], ref[1][1][~bad])


@pytest.mark.parametrize('dtype', BOTH)
def test_strides_alignment_and_shapes(dtype):
    w, X, y, b, g = problem(60, 96, 410, dtype, 10, True)
    ref = run(w, X, y, b, g)

    def same(w_, X_, y_, b_):
        lp, grads = run(w_, X_, y_, b_, g.reshape(y_.shape))
        assert torch.equal(lp.reshape(-1), ref[0])
        for a, c in zip(grads, ref[1]):
            assert torch.equal(a.reshape(c.shape), c)
    wide = torch.full((60, 250), float('nan'), device='cuda', dtype=dtype)
    for off in (0, 1, 8, 77):           # rows inside a wider buffer, NaN around
        wide[:] = float('nan')
        wide[:, off:off + 96] = X
        same(w, wide[:, off:off + 96], y, b)
    ww = torch.full((2, 410, 99), float('nan'), device='cuda', dtype=dtype)
    ww[1, :, 3:] = w
    same(ww[1, :, 3:], X, y, b)
    same(w.t().contiguous().t(), X.t().contiguous().t(), y.int(), b)
    same(w, X.reshape(5, 12, 96), y.reshape(5, 12), b)
    yy = torch.stack([y, y], 1)
    bb = torch.stack([b, b], 1)
    same(w, X, yy[:, 0], bb[:, 1])
    # one row used for all: the gradient of the shared row is the sum
    one = X[:1].detach().clone().requires_grad_()
    lp = zs.linear_categorical_log_prob(w, one.expand(60, 96), y, bias=b)
    gx, = torch.autograd.grad(lp, one, g)
    (_, refs), (_, tols) = class_log_prob(w, X[:1].expand(60, 96), y, b, None,
                                          g)
    # (torch adds the 60 rows in their own type)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    within(gx[0], refs[1].sum(0),
           tols[1].sum(0) + 60 * half * refs[1].abs().sum(0), 'shared row')


def test_bias_of_the_operands_type_and_partial_gradients():
    w, X, y, b, g = problem(33, 64, 200, torch.bfloat16, 11, True)
    bh = b.bfloat16().requires_grad_()
    lp = zs.linear_categorical_log_prob(w, X, y, bias=bh)
    gb, = torch.autograd.grad(lp, bh, g)
    assert gb.dtype == torch.bfloat16
    full = run(w, X, y, bh.detach().float(), g)
    assert torch.equal(lp, full[0]) and torch.equal(gb, full[1][2].bfloat16())
    for leaf, k in ((w, 0), (X, 1)):    # one gradient alone
        t = leaf.clone().requires_grad_()
        args = (t, X) if k == 0 else (w, t)
        lp = zs.linear_categorical_log_prob(*args, y, bias=bh.detach())
        got, = torch.autograd.grad(lp, t, g)
        assert torch.equal(got, full[1][k])
    with torch.no_grad():
        assert torch.equal(zs.linear_categorical_log_prob(w, X, y, bias=bh),
                           lp)


@pytest.mark.parametrize('dtype', BOTH)
def test_empty(dtype):
    w, X, y, b, g = problem(4, 33, 101, dtype, 12, True)
    lp, grads = run(w, X[:0], y[:0], b, g[:0])
    assert lp.shape == (0,) and grads[1].shape == (0, 33)
    assert bool((grads[0] == 0).all()) and bool((grads[2] == 0).all())


def test_gradients_against_differences():
    """(f(x + h) - f(x - h)) / 2h in float32: off by 2 E / 2h for a function
    known to E, and by h^2 / 6 times the third derivative, at most |w_d|^3 (for
    X; third cumulants of a variable within +-a are below 2 a^3, those of an
    indicator below 1)."""
    w, X, y, b, g = problem(3, 10, 50, torch.float32, 13, True)
    _, (tol, (_, tol_x, tol_b)) = class_log_prob(
        w, X, y, b, None, torch.ones(3, device='cuda'))
    lp, (gw, gx, gb) = run(w, X, y, b, torch.ones(3, device='cuda'))
    h = 2.0 ** -6
    for d in range(10):
        e = torch.zeros(10, device='cuda')
        e[d] = h
        up = zs.linear_categorical_log_prob(w, X + e, y, bias=b)
        dn = zs.linear_categorical_log_prob(w, X - e, y, bias=b)
        m = 2 * w[:, d].abs().max().double() ** 3
        # (X +- h is itself rounded: at most 2^-24 |X +- h| |w| off)
        slack = 2 ** -23 * (X[:, d].abs() + h).double() * \
            w[:, d].abs().max().double()
        assert bool(((up.double() - dn.double()) / (2 * h) -
                     gx[:, d].double()).abs().le(
            (2 * tol + 2 * slack) / (2 * h) + h * h / 6 * m +
            tol_x[:, d]).all())
    for v in (0, 17, 49):
        e = torch.zeros(50, device='cuda')
        e[v] = h
        up = zs.linear_categorical_log_prob(w, X, y, bias=b + e).double().sum()
        dn = zs.linear_categorical_log_prob(w, X, y, bias=b - e).double().sum()
        t = float(tol.sum()) + 3 * 2 ** -23 * (float(b[v].abs()) + h)
        assert abs(float((up - dn) / (2 * h) - gb[v].double())) <= \
            2 * t / (2 * h) + 3 * h * h / 6 + float(tol_b[v])


@pytest.mark.parametrize('dtype', BOTH)
def test_same_bits_again_and_on_another_stream(dtype):
    w, X, y, b, g = problem(200, 128, 3000, dtype, 14, True)
    ref = run(w, X, y, b, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(w, X, y, b, g)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip((got[0],) + got[1], (ref[0],) + ref[1]):
        assert torch.equal(a, c)


@pytest.mark.parametrize('dtype', BOTH)
def test_captured_and_replayed(dtype):
    """Forward and gradient in one graph, replayed over new inputs with other
    work between."""
    w, X, y, b, g = problem(150, 64, 2000, dtype, 15, True, IGNORE)
    w, X, b = (t.requires_grad_() for t in (w, X, b))

    def step():
        lp = zs.linear_categorical_log_prob(w, X, y, bias=b,
                                            ignore_label=IGNORE)
        return (lp.detach(),) + torch.autograd.grad(lp, (w, X, b), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        w2, X2, y2, b2, g2 = problem(150, 64, 2000, dtype, 20 + seed, True,
                                     IGNORE)
        with torch.no_grad():
            for dst, src in ((w, w2), (X, X2), (y, y2), (b, b2), (g, g2)):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, step()):
            assert torch.equal(a, c)
        torch.randn(1000, 1000, device='cuda').sum().item()


def test_two_graphs_replayed_in_turn():
    """Two captured calls of different sizes, replayed interleaved and on two
    streams: neither's workspace is the other's."""
    sets = [problem(150, 64, 2000, torch.float32, 60, True, IGNORE),
            problem(300, 96, 1200, torch.bfloat16, 61, True, IGNORE)]
    graphs, outs, refs = [], [], []
    for w, X, y, b, g in sets:
        w, X, b = (t.requires_grad_() for t in (w, X, b))

        def step():
            lp = zs.linear_categorical_log_prob(w, X, y, bias=b,
                                                ignore_label=IGNORE)
            return (lp.detach(),) + torch.autograd.grad(lp, (w, X, b), g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            refs.append([t.clone() for t in step()])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            for a, c in zip(out, ref):
                assert torch.equal(a, c)


def test_units_of_operands_at_both_ends_of_the_range():
    """float32 operands whose product is an ordinary number while each is near
    the end of its range, either way round, and second derivatives refused."""
    w, X, y, b, g = problem(300, 96, 700, torch.float32, 62)
    for k in (2.0 ** 110, 2.0 ** -90):
        lp, grads = run(w * k, X / k, y, None, g)
        ref, refs = run(w, X, y, None, g)
        # powers of two: nothing rounds differently, but for results below
        # 2^-126, which float32 holds in multiples of 2^-149: 2^-150 off, in
        # each of at most 64 parts that are joined
        assert torch.equal(lp, ref)
        for got, c, r in ((grads[0], k, refs[0]), (grads[1], 1 / k, refs[1])):
            off = (got.double() * c - r.double()).abs()
            assert bool((off <= 64 * 2.0 ** -150 * c).all())
    X = X.requires_grad_()
    lp = zs.linear_categorical_log_prob(w, X, y)
    gx, = torch.autograd.grad(lp.sum(), X, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.square().sum(), X)


def test_categorical_over_many_classes_takes_them_in_pieces():
    """Categorical(linear_class_logits(w, X)) of two chains: log_prob and its
    gradients, without the [2, N, V] logits."""
    N, D, V = 3000, 40, 1500
    cases = [problem(N, D, V, torch.float32, 30 + c) for c in range(2)]
    X = cases[0][1].requires_grad_()
    y = cases[0][2]
    w = torch.stack([c[0] for c in cases]).requires_grad_()
    for labels in (y.to(torch.int32), y.float(), y[None],
                   torch.stack([y, y])):
        dist = zs.distributions.Categorical(zs.linear_class_logits(w, X),
                                            group_ndims=1)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        lp = dist.log_prob(labels)
        assert lp.shape == (2,)
        gw, gx = torch.autograd.grad(lp.sum(), (w, X))
        assert dist._logits_dense is None
        assert torch.cuda.max_memory_allocated() - before < 2 * N * V * 4
        tol_x = ref_x = 0
        for c in range(2):
            # (w's gradient: row by row, as if the other chain were not there)
            (lp64, (dw, dx, _)), (tol, (tw, tx, _)) = class_log_prob(
                w[c], X, y, g=torch.ones(N, device='cuda'))
            # N rows' sum in float32, in any order
            within(lp[c], lp64.sum(), tol.sum() + N * U32 * lp64.abs().sum())
            within(gw[c], dw, tw)
            ref_x, tol_x = ref_x + dx, tol_x + tx + U32 * dx.abs()
        within(gx, ref_x, tol_x + U32 * ref_x.abs())
    # labels of a shape of their own: the logits are written out
    dist = zs.distributions.Categorical(zs.linear_class_logits(w, X))
    with torch.no_grad():
        lp3 = dist.log_prob(y.expand(3, 1, N))
        one = zs.linear_categorical_log_prob(w[1], X, y)
    assert lp3.shape == (3, 2, N)
    # (float32 sums of D terms either way, and two log-sum-exps)
    lp64, tol = class_log_prob(w[1], X, y)
    within(lp3[2, 1], lp64, 2 * tol)
    within(one, lp64, tol)
    with pytest.raises(ValueError):
        dist.log_prob(y[:-1])


def test_sampler_of_a_softmax_regression_over_many_classes():
    """A model with a [V, D] latent a chain, its logits spelled X @ w^T:
    log_joint and its gradient, and transitions of the sampler."""
    N, D, V, C = 2100, 24, 2048, 2
    w0, X, y, _, _ = problem(N, D, V, torch.float32, 41)
    w1 = problem(N, D, V, torch.float32, 42)[0]

    @zs.meta_bayesian_net()
    def model():
        bn = zs.BayesianNet()
        w = bn.normal('w', torch.zeros(V, D, device='cuda'), std=1.,
                      n_samples=C, group_ndims=2)
        bn.categorical('y', X.unsqueeze(0) @ w.tensor.transpose(-1, -2),
                       group_ndims=1)
        return bn

    labels = y.to(torch.int32)
    leaf = torch.stack([w0, w1]).requires_grad_()
    lj = model().observe(w=leaf, y=labels).log_joint()
    assert lj.shape == (C,)
    got, = torch.autograd.grad(lj.sum(), leaf)
    for c in range(C):
        wc = leaf[c].detach()
        (lp, (dw, _, _)), (tol, (tw, _, _)) = class_log_prob(
            wc, X, y, g=torch.ones(N, device='cuda'))
        within(got[c], dw - wc.double(),
               tw + 4 * U32 * (dw.abs() + wc.abs()))
        prior = -0.5 * wc.double().square() - 0.5 * math.log(2 * math.pi)
        within(lj[c], lp.sum() + prior.sum(), tol.sum() + U32 * (
            N * lp.abs().sum() + (V * D + 8) * prior.abs().sum()))

    q = torch.zeros(C, V, D, device='cuda')
    hmc = zs.HMC(step_size=1e-3, n_leapfrogs=2)
    op, info = hmc.sample(model(), {'y': labels}, {'w': q})
    assert hmc.plan_kind == 'generic'
    for _ in range(3):
        op.run()
    assert bool(torch.isfinite(info.log_prob).all())
    assert bool(q.isfinite().all()) and float(q.abs().max()) > 0
