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


@pytest.mark.parametrize('k', [2048, 2056])
def test_dequantize_reads_what_the_call_before_wrote(k):
    """Records rewritten between calls on one stream, with no wait of the host, by torch's copies and between this
    library's own launches, which may start before the kernel ahead of them ends."""
    from micro_vllm_b200.w4_linear import W4Weight, w4_dequantize, w4_linear
    pairs = [make(2048, k, 64, True, seed=s) for s in (3, 4)]
    a = pairs[0][0]
    live = W4Weight(torch.empty_like(a.records), a.shape, a.group_size, a.has_zeros, a.scale_dtype)
    expected = [torch.from_numpy(w).float().to(torch.bfloat16).cuda() for _, w in pairs]
    out = torch.empty((2048, k), dtype=torch.bfloat16, device='cuda')
    x = torch.ones((16, k), dtype=torch.bfloat16, device='cuda')
    products = [w4_linear(x, weight) for weight, _ in pairs]
    for turn in range(20):
        live.records.copy_(pairs[turn % 2][0].records)
        w4_dequantize(live, out=out)
        assert torch.equal(out, expected[turn % 2])
        assert torch.equal(w4_linear(x, live), products[turn % 2])
        live.records.copy_(pairs[1 - turn % 2][0].records)
        w4_linear(x, live)
        assert torch.equal(w4_dequantize(live, torch.bfloat16), expected[1 - turn % 2])


@pytest.mark.parametrize('m', [1, 5, 20])
def test_fp32_rows_are_multiplied_to_their_last_bits(m):
    """One number of x per row and group: y is its product with a weight, over one group a sum of one term.

    x is the exact sum of three bf16 numbers. Their products with a code's distance (at most 4 bits) are exact, three
    are added (each addition off by at most 2^-23 of the largest), then scaled and joined by at most three more
    roundings of 2^-24: below 2^-20 of the value. Without its third number x would be off by up to 2^-16."""
    from micro_vllm_b200.w4_linear import w4_linear
    n, k = 130, 512
    weight, w = make(n, k, 64, False, seed=5)
    gen = torch.Generator().manual_seed(6)
    x = torch.zeros((m, k))
    column = torch.randint(0, k, (m,), generator=gen)
    # Mantissas whose last eight bits are all ones: what the first two bf16 numbers leave is nearly 2^-16.
    bits = torch.randint(0, 1 << 15, (m,), generator=gen, dtype=torch.int32) << 8 | 0xff | 127 << 23
    x[torch.arange(m), column] = bits.view(torch.float32)
    y = as64(w4_linear(x.cuda(), weight))
    expected = as64(x[torch.arange(m), column])[:, None] * w.T[column.numpy()]
    assert (np.abs(y - expected) <= 2.0 ** -20 * np.abs(expected)).all()
    two = as64((x[torch.arange(m), column].view(torch.int32) & -256).view(torch.float32))[:, None] * w.T[column.numpy()]
    assert not (np.abs(two - expected) <= 2.0 ** -20 * np.abs(expected)).all()  # what the bound would catch
