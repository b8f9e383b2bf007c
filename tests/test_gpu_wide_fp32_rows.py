"""fp32 rows at both sides of what the norm's threads hold.

The sum of squares: at most width / 448 additions a thread and twenty more, each off by half of fp32's step, halved by
the root; then a handful of roundings.
"""
import numpy as np
import pytest
import torch

from tests.test_gpu_quant_rows import norm64, norm_inputs
from tests.w4_reference import HALF_STEP, as64, assert_quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows', [1, 300])
@pytest.mark.parametrize('width', [14336, 14344, 16384, 16392, 24576, 32776])
def test_wide_fp32_rows(rows, width):
    from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant
    x, r, w = norm_inputs((rows, width), torch.float32, 9)
    s, y = norm64(x, r, w, 1e-6)
    off = (width / 448 / 2 + 24) * 2.0 ** -24
    place = x.cuda()
    out, total = add_rms_norm(place, r.cuda(), w.cuda(), 1e-6, residual_out=place)
    assert torch.equal(total.cpu(), s)
    assert (np.abs(as64(out) - y) <= (HALF_STEP[torch.float32] + off) * np.abs(y)).all()
    for quant in (torch.int8, torch.float8_e4m3fn):
        q, scale, total = add_rms_norm_quant(x.cuda(), r.cuda(), w.cuda(), 1e-6, quant_dtype=quant)
        assert torch.equal(total.cpu(), s)
        assert_quantized(q, scale, y, quant, off)
