"""8-bit values that a program brings: rows further apart
than the product's kernels take."""
import pytest
import torch

import zhusuan_amd as zs

pytestmark = pytest.mark.gpu


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
