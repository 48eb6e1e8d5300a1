"""More rows than one launch takes (2^24 workgroups of 256 threads)."""
import pytest
import torch

import zhusuan_amd as zs
from helpers_class_logits import quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_quantize_rows(dtype):
    n = 2 ** 26 + 4097
    gen = torch.Generator(device='cuda')
    gen.manual_seed(0)
    x = torch.randn(n, 4, generator=gen, device='cuda').to(dtype)
    got = zs.quantize_rows(x)
    most = x.float().abs().amax(1)
    assert torch.equal(got.scale, most / torch.full_like(most, 127.))
    for at in (0, 2 ** 25 - 50, 2 ** 26 - 50, n - 100):
        q, s = quantized(x[at:at + 100].cpu())
        assert torch.equal(got.values[at:at + 100].cpu().float(), q)
    back = got.dequantize(dtype)
    for at in (0, 2 ** 25 - 50, n - 100):
        q, s = quantized(x[at:at + 100].cpu())
        assert torch.equal(back[at:at + 100].cpu(), (q * s).to(dtype))
