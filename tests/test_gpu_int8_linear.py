"""zs.quantize_rows / quantized_linear (csrc/int8_linear.hip) against their
plain forms: equal where the definition is exact, within counted roundings
elsewhere."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import HALF, U32, quantized, within

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


def rand(*shape, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen) * torch.exp(
        torch.randn(*shape[:-1], 1, generator=gen))
    return x.to(dtype)


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('shape', [(1, 1), (3, 5), (1, 4096), (7, 127), (9, 128),
                                   (130, 784), (2, 3, 65), (5,), (33, 10001),
                                   (3000, 64)])
def test_quantize_rows(shape, dtype):
    x = rand(*shape, dtype=dtype)
    q, s = quantized(x)                       # on the CPU
    got = zs.quantize_rows(x.cuda())
    assert got.values.dtype == torch.int8 and got.shape == x.shape
    assert torch.equal(got.values.cpu().float(), q)
    assert torch.equal(got.scale.cpu(), s[..., 0])
    assert torch.equal(got.dequantize().cpu(), q * s)
    assert torch.equal(got.dequantize(torch.bfloat16).cpu(),
                       (q * s).bfloat16())


@pytest.mark.parametrize('dtype', BOTH)
def test_quantize_special_rows(dtype):
    x = rand(9, 200, dtype=dtype)
    x[1] = 0
    x[2, 7] = float('nan')
    x[3, 150] = float('inf')
    x[4, 0] = -float('inf')
    x[5] = torch.where(torch.arange(200) % 2 == 0, 127.0, 0.5).to(dtype)  # ties
    x[6] = torch.finfo(dtype).max
    x[7] *= 1e-38
    x[8] = -0.0
    got = zs.quantize_rows(x.cuda())
    q, s = quantized(x)
    bad = [2, 3, 4]
    ok = [0, 1, 5, 6, 7, 8]
    assert bool(got.scale[bad].isnan().all())
    assert bool((got.values[bad] == 0).all())
    assert bool(got.dequantize()[bad].isnan().all())
    assert torch.equal(got.scale.cpu()[ok], s[ok, 0])
    assert torch.equal(got.values.cpu()[ok].float(), q[ok])
    assert float(got.scale[1]) == 1.0 and float(got.scale[8]) == 1.0
    assert bool((got.values[5].cpu()[1::2] == 0).all())   # 0.5 -> the even 0


def test_quantize_strided_rows():
    x = rand(40, 300, dtype=torch.bfloat16).cuda()
    for v in (x[:, 3:204], x[::2, :100], x.t(), x[5:6, 7:], x[:, ::2]):
        a, b = zs.quantize_rows(v), zs.quantize_rows(v.contiguous())
        assert torch.equal(a.values, b.values) and torch.equal(a.scale, b.scale)
    e = zs.quantize_rows(x[:0])
    assert e.values.shape == (0, 300) and e.dequantize().shape == (0, 300)


def reference(xq, wq, bias, dtype):
    """The exact sum; float32 roundings: of the sum (above 2^24), of the scales'
    product, of its product with the sum, of the sum with the bias."""
    acc = xq.values.cpu().long() @ wq.values.cpu().long().t()
    assert int(acc.abs().max()) < 2 ** 31
    ref = acc.double() * xq.scale.cpu().double()[..., None] * \
        wq.scale.cpu().double()
    tol = 3 * U32 * ref.abs()
    if bias is not None:
        ref = ref + bias.cpu().double()
        tol = tol + U32 * ref.abs()
    return ref, tol + HALF[dtype] * ref.abs() * 1.01


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('M,K,V', [
    (1, 1, 1), (1, 64, 128), (2, 15, 3), (7, 1000, 1219), (16, 128, 129),
    (17, 4096, 300), (32, 130, 257), (33, 129, 500), (64, 2048, 70),
    (200, 784, 1241), (513, 96, 4097), (4100, 200, 4200)])
def test_quantized_linear(M, K, V, dtype):
    for bias in (None, rand(1, V, seed=3)[0].cuda()):
        w = zs.quantize_rows(rand(V, K, seed=1).cuda())
        x = rand(M, K, dtype=dtype, seed=2).cuda()
        xq = zs.quantize_rows(x)
        for out_dtype in BOTH:
            ref, tol = reference(xq, w, bias, out_dtype)
            got = zs.quantized_linear(w, x, bias=bias, dtype=out_dtype)
            assert got.dtype == out_dtype
            within(got.cpu(), ref, tol, 'tensor')
            assert torch.equal(got, zs.quantized_linear(
                w, xq, bias=bias, dtype=out_dtype))
    assert zs.quantized_linear(w, x).dtype == dtype
    assert zs.quantized_linear(w, xq).dtype == torch.float32


def test_largest_sum():
    """131 072 products of 127 * 127 stay inside an int32."""
    one = torch.ones(3, 131072, device='cuda')
    w = zs.quantize_rows(one * torch.tensor([[1.], [-1.], [2.]],
                                            device='cuda'))
    for rows in (1, 3, 40):
        got = zs.quantized_linear(w, one[:1].expand(rows, -1))
        ref = torch.tensor([131072., -131072., 262144.], dtype=torch.float64,
                           device='cuda').expand(rows, 3)
        within(got, ref, 8 * U32 * ref.abs(), rows)
    with pytest.raises(ValueError, match='131072'):
        zs.quantized_linear(zs.QuantizedRows(
            torch.zeros(2, 131073, dtype=torch.int8, device='cuda'),
            torch.ones(2, device='cuda')), torch.zeros(1, 131073,
                                                       device='cuda'))


def test_values_of_ones_own():
    """Values and scales that a program brings: any stride and alignment, with
    other bytes around them."""
    gen = torch.Generator().manual_seed(4)
    for V, K in ((50, 100), (300, 128), (33, 77), (1, 13)):
        v = torch.randint(-127, 128, (V, K), generator=gen,
                          dtype=torch.int8).cuda()
        s = torch.rand(V, generator=gen).cuda()
        x = rand(5, K, seed=5).cuda()
        ref = zs.quantized_linear(zs.QuantizedRows(v, s), x)
        tol = reference(zs.quantize_rows(x), zs.QuantizedRows(v, s), None,
                        torch.float32)
        within(ref.cpu(), *tol)
        for pitch, off in ((K + 3, 1), ((K + 15) // 16 * 16 + 32, 16),
                           ((K + 15) // 16 * 16, 0)):
            room = torch.full((V * pitch + off + K + 64,), 99,
                              dtype=torch.int8, device='cuda')
            view = room[off:].as_strided((V, K), (pitch, 1))
            view.copy_(v)
            q = zs.QuantizedRows(view, s)
            assert torch.equal(q.values, v)
            assert torch.equal(zs.quantized_linear(q, x), ref)
            # ... as the left operand, whose tail must count as zeros
            left = zs.QuantizedRows(view, s)
            right = zs.quantize_rows(x)
            a = zs.quantized_linear(right, left)
            within(a.cpu(), *reference(left, right, None, torch.float32))
        # at the very end of an allocation
        tail = torch.zeros(V * K, dtype=torch.int8, device='cuda')
        t = tail.view(V, K)
        t.copy_(v)
        assert torch.equal(zs.quantized_linear(zs.QuantizedRows(t, s), x), ref)
        assert torch.equal(zs.quantized_linear(zs.QuantizedRows(
            v.t().contiguous().t(), s), x), ref)


def test_nan_rows_and_scales_pass_through():
    w = zs.quantize_rows(rand(70, 64, seed=6).cuda())
    x = rand(5, 64, seed=7).cuda()
    ref = zs.quantized_linear(w, x)
    x[3, 9] = float('nan')
    got = zs.quantized_linear(w, x)
    bad = torch.arange(5, device='cuda') == 3
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], ref[~bad])


def test_shapes_and_empty():
    w = zs.quantize_rows(rand(70, 64, seed=6).cuda())
    x = rand(2, 3, 64, seed=7).cuda()
    assert zs.quantized_linear(w, x).shape == (2, 3, 70)
    assert torch.equal(zs.quantized_linear(w, x).reshape(6, 70),
                       zs.quantized_linear(w, x.reshape(6, 64)))
    assert zs.quantized_linear(w, x[0, 0]).shape == (70,)
    assert torch.equal(zs.quantized_linear(w, x[0, 0]),
                       zs.quantized_linear(w, x)[0, 0])
    assert zs.quantized_linear(w, x[:0]).shape == (0, 3, 70)


def test_streams_and_graph():
    w = zs.quantize_rows(rand(3000, 256, seed=8).cuda())
    x = rand(20, 256, seed=9, dtype=torch.bfloat16).cuda()
    ref = zs.quantized_linear(w, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = zs.quantized_linear(w, x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = zs.quantized_linear(w, x)
        back = zs.quantize_rows(x).dequantize()
    for seed in range(3):
        x.copy_(rand(20, 256, seed=30 + seed, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, zs.quantized_linear(w, x))
        assert torch.equal(back, zs.quantize_rows(x).dequantize())


def test_an_output_layer_trained_rounded_and_used():
    """What the operators are for, together: log-probabilities and gradients
    move a layer, its weights are rounded to 8 bits, and the rounded layer's logits
    make a Categorical that is sampled and scored."""
    gen = torch.Generator().manual_seed(1)
    V, D, N = 700, 96, 256
    truth = torch.randn(V, D, generator=gen)
    X = torch.randn(N, D, generator=gen)
    y = (X @ truth.t()).argmax(1).cuda()
    X = X.cuda()
    w = torch.zeros(V, D, device='cuda', requires_grad=True)
    b = torch.zeros(V, device='cuda', requires_grad=True)
    for _ in range(3):
        loss = -zs.linear_categorical_log_prob(w, X, y, bias=b).mean()
        gw, gb = torch.autograd.grad(loss, (w, b))
        with torch.no_grad():
            w -= 50 * gw
            b -= gb
    with torch.no_grad():
        wq = zs.quantize_rows(w)
        logits = zs.quantized_linear(wq, X, bias=b)
        exact = zs.quantize_rows(X).dequantize().double() @ \
            wq.dequantize().double().t() + b.double()
        # (what is read back from the integers is rounded once per value)
        mag = zs.quantize_rows(X).dequantize().double().abs() @ \
            wq.dequantize().double().abs().t() + b.abs()
        within(logits, exact, 8 * U32 * mag)
        d = zs.distributions.Categorical(logits)
        s = d.sample(4)
        assert s.shape == (4, N) and int(s.min()) >= 0 and int(s.max()) < V
        lp = d.log_prob(y)
        ref = torch.log_softmax(logits.double(), 1).gather(1, y[:, None])[:, 0]
        within(lp, ref, 64 * 2.0 ** -24 * (1 + logits.abs().double().amax(1)))


def test_no_gradient_is_refused():
    w = zs.quantize_rows(torch.randn(20, 16, device='cuda'))
    X = torch.randn(3, 16, device='cuda')
    b = torch.randn(20, device='cuda')
    ref = zs.quantized_linear(w, X, bias=b)
    for kw in (dict(X=X.clone().requires_grad_()),
               dict(bias=b.clone().requires_grad_())):
        kw = dict(dict(X=X, bias=b), **kw)
        with pytest.raises(RuntimeError, match='gradient'):
            zs.quantized_linear(w, **kw)
        with torch.no_grad():
            assert torch.equal(zs.quantized_linear(w, **kw), ref)


def test_a_categorical_answers_from_8_bit_rows():
    """Categorical(linear_class_logits(quantize_rows(w), X)): its logits are
    quantized_linear's, and labels are scored and drawn from them."""
    gen = torch.Generator().manual_seed(3)
    w = torch.randn(300, 96, generator=gen).cuda()
    X = torch.randn(40, 96, generator=gen).cuda()
    y = torch.randint(300, (40,), generator=gen, dtype=torch.int32).cuda()
    q = zs.quantize_rows(w)
    dist = zs.distributions.Categorical(zs.linear_class_logits(q, X),
                                        group_ndims=1)
    logits = zs.quantized_linear(q, X)
    assert dist.get_batch_shape() == (40,)
    assert torch.equal(dist.logits, logits)
    plain = zs.distributions.Categorical(logits, group_ndims=1)
    assert torch.equal(dist.log_prob(y), plain.log_prob(y))
    drawn = dist.sample(7)
    assert drawn.shape == (7, 40)
    assert int(drawn.min()) >= 0 and int(drawn.max()) < 300
    with pytest.raises(ValueError):
        zs.linear_class_logits(q, X[:, :95])
    with pytest.raises(ValueError):
        zs.linear_class_logits(zs.quantize_rows(w.reshape(2, 150, 96)), X)
