"""Scales at the ends of their type's range, outputs that the call before wrote, and fp32 rows to their last bits."""
import numpy as np
import pytest
import torch

from tests.test_gpu_w4_linear import make
from tests.w4_reference import as64, checkpoint, dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('scale_dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('offset', [0, 1])
def test_dequantize_scales_of_every_size(dtype, scale_dtype, zeros, offset):
    """(code - zero) * scale has at most 4 + 11 bits: exact in 64 bits, so one rounding (to fp32 and on to 16 bits it
    is one too: 15 bits are exact in fp32 down to 2^-135, and a bf16's steps end at 2^-133 with 8 bits of scale)."""
    from micro_vllm_b200.w4_linear import pack_w4, w4_dequantize
    n, k, group = 96, 256, 32
    codes, _, zero = checkpoint(n, k, group, zeros, scale_dtype, seed=1)
    low, high = (-24, 15) if scale_dtype == torch.float16 else (-133, 127)
    exponents = torch.arange(n * (k // group)).view(n, -1) % (high - low + 1) + low
    mantissa = 1 + torch.rand(exponents.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    scales = (mantissa * 2.0 ** exponents.double()).float().clamp(max=torch.finfo(scale_dtype).max).to(scale_dtype)
    weight = pack_w4(codes.cuda(), scales.cuda(), None if zero is None else zero.cuda(), group_size=group)
    wide = torch.empty((n, k + offset), dtype=dtype, device='cuda')
    got = w4_dequantize(weight, out=wide[:, offset:])
    expected = torch.from_numpy(dense(codes, scales, zero, group)).to(torch.float32).to(dtype)
    assert torch.equal(got.cpu(), expected)
    if not offset:
        assert torch.equal(w4_dequantize(weight, dtype).cpu(), expected)
