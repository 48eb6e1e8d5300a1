"""float32 operands in planes (more than 512 rows, 256 with gradients): odd
sizes, strides and alignments, other streams, captured and replayed."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import class_log_prob, problem, within

pytestmark = pytest.mark.gpu
IGNORE = -100


def run(w, X, y, b, g, ignore=None):
    leaves = [t.detach().requires_grad_() for t in (w, X, b)
              if t is not None]
    lp = zs.linear_categorical_log_prob(
        leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None,
        ignore_label=ignore)
    return (lp.detach(),) + torch.autograd.grad(lp, leaves, g)


@pytest.mark.parametrize('N,D,V', [
    (257, 1, 1), (513, 1, 5), (513, 7, 3), (600, 65, 257), (700, 33, 513),
    (640, 64, 4096), (1000, 3, 5000)])
def test_odd_sizes(N, D, V):
    for bias, ignore in ((False, None), (True, IGNORE)):
        w, X, y, b, g = problem(N, D, V, torch.float32, N + D + V, bias,
                                ignore)
        got = run(w, X, y, b, g, ignore)
        (ref, refs), (tol, tols) = class_log_prob(w, X, y, b, ignore, g)
        within(got[0], ref, tol, 'log_prob')
        for name, a, r, t in zip(('w', 'X', 'bias'), got[1:], refs, tols):
            within(a, r, t, name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    N, D, V = 600, 96, 410
    w, X, y, b, g = problem(N, D, V, dtype, 10, True, IGNORE)
    ref = run(w, X, y, b, g, IGNORE)

    def same(w_, X_):
        for a, c in zip(run(w_, X_, y, b, g, IGNORE), ref):
            assert torch.equal(a, c)
    wide = torch.full((N, 250), float('nan'), device='cuda', dtype=dtype)
    tall = torch.full((V, 131), float('nan'), device='cuda', dtype=dtype)
    for off in (0, 1, 8, 35):
        wide[:], tall[:] = float('nan'), float('nan')
        wide[:, off:off + D] = X
        tall[:, off:off + D] = w
        same(w, wide[:, off:off + D])
        same(tall[:, off:off + D], wide[:, off:off + D])
    same(w.t().contiguous().t(), X.t().contiguous().t())
    end = torch.empty(N * D + 3, device='cuda', dtype=dtype)[3:].view(N, D)
    end.copy_(X)                     # up to the last element of an allocation
    same(w, end)


def test_on_another_stream_and_again():
    args = problem(900, 128, 3000, torch.float32, 14, True, IGNORE)
    ref = run(*args, ignore=IGNORE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*args, ignore=IGNORE)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(got, ref):
        assert torch.equal(a, c)


def test_two_graphs_replayed_in_turn():
    """Over new inputs, of other units too, with eager calls between."""
    sizes = [(600, 64, 2000), (1100, 96, 1200)]
    sets = [problem(*s, torch.float32, 60, True, IGNORE) for s in sizes]
    graphs, outs = [], []
    for w, X, y, b, g in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(w, X, y, b, g, IGNORE)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(w, X, y, b, g, IGNORE))
        graphs.append(graph)
    for seed in range(3):
        for size, held in zip(sizes, sets):
            new = problem(*size, torch.float32, 70 + seed, True, IGNORE)
            for dst, src, k in zip(held, new, (8. ** seed, 0.5 ** seed, 1, 1,
                                               0.01 ** seed)):
                dst.copy_(src * k)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, held in zip(outs, sets):
            for a, c in zip(out, run(*held, ignore=IGNORE)):
                assert torch.equal(a, c)
        torch.randn(1000, 1000, device='cuda').sum().item()
