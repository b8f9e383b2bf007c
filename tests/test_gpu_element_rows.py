"""Many rows that can only be read element by element, at the widths where a warp's row becomes a CTA's.

Tolerances as in test_gpu_quant_rows.py: the norm's sum has at most 64 terms a thread and a tree behind it, below
2^-18 of y; the gate's values, for gates up to 12, stay within 2^-18.
"""
import numpy as np
import pytest
import torch

from tests.test_gpu_quant_rows import NORM_OFF, norm64, norm_inputs
from tests.w4_reference import HALF_STEP, as64, assert_quantized

pytestmark = pytest.mark.gpu


def at_odd_offset(t):
    """The same rows as columns 1.. of wider ones, which no vector access can read."""
    wide = torch.full((t.shape[0], t.shape[1] + 2), float('nan'), dtype=t.dtype, device='cuda')
    wide[:, 1:-1] = t.cuda()
    return wide[:, 1:-1]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,width,offset', [(400, 1001, 0), (400, 1000, 1), (301, 513, 0), (700, 512, 1), (700, 511, 0),
                                               (500, 257, 0), (500, 256, 1), (320, 1024, 1), (320, 1025, 0)])
def test_rows_read_by_element(dtype, rows, width, offset):
    from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant, silu_mul_quant
    x, r, w = norm_inputs((rows, width), dtype, 8)
    s, y = norm64(x, r, w, 1e-6)
    place = at_odd_offset if offset else torch.Tensor.cuda
    out, total = add_rms_norm(place(x), place(r), w.cuda(), 1e-6)
    assert torch.equal(total.cpu(), s)
    subnormal = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert (np.abs(as64(out) - y) <= (HALF_STEP[dtype] * (1 + 2.0 ** -8) + NORM_OFF) * np.abs(y) + subnormal).all()
    for quant in (torch.int8, torch.float8_e4m3fn):
        q, scale, total = add_rms_norm_quant(place(x), place(r), w.cuda(), 1e-6, quant_dtype=quant)
        assert torch.equal(total.cpu(), s)
        assert_quantized(q, scale, y, quant, NORM_OFF)
        both = torch.cat([x, r], dim=-1)
        g64, u64 = as64(x), as64(r)
        q, scale = silu_mul_quant(place(both), quant_dtype=quant)
        assert np.abs(g64).max() < 12
        assert_quantized(q, scale, g64 / (1 + np.exp(-g64)) * u64, quant, 2.0 ** -18)
