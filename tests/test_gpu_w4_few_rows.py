"""Both sides of the rule between the two product kernels, at each of its sizes, in every type and group.

Tolerances as in test_gpu_w4_linear.py.
"""
import pytest
import torch

from tests.test_gpu_w4_linear import activations, assert_linear
from tests.w4_reference import checkpoint, dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('group,zeros', [(32, True), (64, True), (128, False)])
@pytest.mark.parametrize('k,n', [(384, 320), (1280, 6336), (1280, 6400), (2304, 6400), (2304, 6464), (4096, 8128), (4096, 8192), (8192, 8128),
                                 (8192, 8256), (16384, 16448)])
def test_few_rows_at_every_size_of_the_rule(dtype, group, zeros, k, n):
    from micro_vllm_b200.w4_linear import pack_w4, w4_linear
    codes, scales, zero = checkpoint(n, k, group, zeros, torch.bfloat16, seed=60)
    weight = pack_w4(codes.cuda(), scales.cuda(), None if zero is None else zero.cuda(), group_size=group)
    x, scale = activations(9, k, dtype, seed=61)
    rows = [0, 1, 63, 64, n // 2, n - 65, n - 64, n - 1]  # of the weight: first, last and at tiles' borders
    w = dense(codes[rows], scales[rows], None if zero is None else zero[rows], group)
    for m in (2, 3, 4, 5, 7, 8, 9):
        y = w4_linear(x[:m].cuda(), weight, x_scale=None if scale is None else scale[:m].cuda(), out_dtype=torch.float32)
        assert y.shape == (m, n)
        assert_linear(y[:, rows], x[:m], None if scale is None else scale[:m], w, group=group)
        assert torch.isfinite(y).all() or dtype == torch.float8_e4m3fn
