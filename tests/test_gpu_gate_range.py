"""silu_mul_quant at gates over the whole range of fp32's exponential.

Tolerance. The exponent's argument, at most 2^7, is off by half of its step (2^-18) and by 1.4e-8 of itself (2^-19)
for log2 e's own rounding, so the exponential by ln 2 of that, below 2^-18; exp, the reciprocal and the products add
at most eight units of 2^-23. All in all a value, and with it its row's scale, is within 2^-17 of itself.
"""
import numpy as np
import pytest
import torch

from tests.w4_reference import as64, assert_quantized

pytestmark = pytest.mark.gpu

EIGHT = [torch.int8, torch.float8_e4m3fn]
GATE_OFF = 2.0 ** -17


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('width', [1, 8, 264, 1001])
def test_gates_down_to_the_end_of_the_exponentials_range(quant, width):
    """exp(-g) is finite in fp32 down to -88.72: what g / (1 + exp(-g)) gives there is a normal number."""
    from micro_vllm_b200.row_ops import silu_mul_quant
    gates = torch.tensor([-1.0, -20.0, -60.0, -80.0, -86.9, -87.2, -87.3, -87.4, -87.5, -88.0, -88.4, -88.5, -88.7])
    u = torch.linspace(0.5, 1.5, width) * 1e30
    x = torch.cat([gates[:, None].expand(-1, width), u.expand(len(gates), -1)], dim=-1)
    q, scale = silu_mul_quant(x.cuda(), quant_dtype=quant)
    x64 = as64(x)
    g64, u64 = x64[:, :width], x64[:, width:]
    assert_quantized(q, scale, g64 / (1 + np.exp(-g64)) * u64, quant, GATE_OFF)
    assert (scale > 0).all()


@pytest.mark.parametrize('quant', EIGHT)
def test_gates_beyond_the_exponentials_range_are_zeros(quant):
    from micro_vllm_b200.row_ops import silu_mul_quant
    x = torch.tensor([[-88.8, 1e30], [-100.0, 1e30], [-3e38, 3e38], [-200.0, 1.0]])
    q, scale = silu_mul_quant(x.cuda(), quant_dtype=quant)
    assert not q.float().any() and not scale.any()


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('quant', EIGHT)
def test_many_gates_of_every_size(dtype, quant):
    from micro_vllm_b200.row_ops import silu_mul_quant
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((500, 2 * 96), generator=gen) * 3
    x[:, ::7] *= 8  # gates down to some -80
    x = x.to(dtype)
    q, scale = silu_mul_quant(x.cuda(), quant_dtype=quant)
    x64 = as64(x)
    g64, u64 = x64[:, :96], x64[:, 96:]
    assert_quantized(q, scale, g64 / (1 + np.exp(-g64)) * u64, quant, GATE_OFF)
