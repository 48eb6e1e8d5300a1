"""8-bit values that a program brings: the smallest one, and rows further apart
than the product's kernels take."""
import pytest
import torch

import zhusuan_amd as zs

pytestmark = pytest.mark.gpu


def lowest(rows, K):
    return zs.QuantizedRows(torch.full((rows, K), -128, dtype=torch.int8,
                                       device='cuda'),
                            torch.ones(rows, device='cuda'))


def test_products_of_the_lowest_value():
    """K products of 2^14 are exact up to K = 131071, and refused where their
    sum, 2^31, is no int32."""
    K = 131071
    got = zs.quantized_linear(lowest(3, K), lowest(2, K))
    assert torch.equal(got, torch.full_like(got, float(K * 2 ** 14)))
    with pytest.raises(ValueError, match='131071'):
        zs.quantized_linear(lowest(3, K + 1), lowest(2, K + 1))
    # one side rounded here stays within 127 * 128
    one = torch.ones(2, K + 1, device='cuda')
    for X in (one, zs.quantize_rows(one)):
        got = zs.quantized_linear(lowest(3, K + 1), X) * 127
        ref = torch.full_like(got, -127. * 128 * (K + 1))
        # (1 / 127 as the scale, and two products with it)
        assert bool(((got - ref).abs() <= 4 * 2.0 ** -24 * ref.abs()).all())
    got = zs.quantized_linear(zs.quantize_rows(one), lowest(3, K + 1)) * 127
    assert bool(((got + 127. * 128 * (K + 1)).abs() <=
                 4 * 2.0 ** -24 * 127. * 128 * (K + 1)).all())


def test_rows_far_apart():
    """16-byte aligned rows 8 MB apart: copied closer together."""
    room = torch.zeros(5 * (8 << 20), dtype=torch.int8, device='cuda')
    view = room.as_strided((5, 64), (8 << 20, 1))
    gen = torch.Generator().manual_seed(0)
    values = torch.randint(-127, 128, (5, 64), generator=gen,
                           dtype=torch.int8).cuda()
    view.copy_(values)
    scale = torch.rand(5, device='cuda')
    x = torch.randn(3, 64, device='cuda')
    far, near = zs.QuantizedRows(view, scale), zs.QuantizedRows(values, scale)
    assert torch.equal(far.values, values)
    assert torch.equal(zs.quantized_linear(far, x),
                       zs.quantized_linear(near, x))
    assert torch.equal(zs.quantized_linear(near, far),
                       zs.quantized_linear(near, near))
    assert torch.equal(far.dequantize(), near.dequantize())
