"""The 8-bit rows' values where their rounding shows: numbers halfway between two 8-bit ones, at scales of every size.

Where the row's values and scale are exact in fp32 the results are equal to the formula's, ties to even.
"""
import numpy as np
import pytest
import torch

from tests.w4_reference import TOP, as64

pytestmark = pytest.mark.gpu

EIGHT = [torch.int8, torch.float8_e4m3fn]


def ties(quant):
    """The numbers halfway between neighbours of the 8-bit type, with the largest first, and what they round to."""
    if quant == torch.int8:
        numbers = np.arange(-127.0, 128.0)
        halves, nearest = (numbers[1:] + numbers[:-1]) / 2, np.round((numbers[1:] + numbers[:-1]) / 2)
    else:  # e4m3: bit patterns 0 to 0x7e are its numbers from 0 to 448, in order; the even pattern wins a tie
        numbers = torch.arange(0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
        halves = (numbers[1:] + numbers[:-1]) / 2
        nearest = np.where(np.arange(0x7e) % 2 == 0, numbers[:-1], numbers[1:])
        halves, nearest = np.concatenate([halves, -halves]), np.concatenate([nearest, -nearest])
    return np.concatenate([[TOP[quant]], halves]), np.concatenate([[TOP[quant]], nearest])


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('rows', [1, 2, 400])
def test_ties_of_the_norm_round_to_even(quant, rows):
    """Rows of ones have the mean square 1, so y is the weight; with the largest |y| top * c the scale is c."""
    from micro_vllm_b200.row_ops import add_rms_norm_quant
    values, nearest = ties(quant)
    x = torch.ones((rows, len(values)), device='cuda')
    for c in range(1, 256, 2):  # at most 8 bits, and a tie at most 8 (int8) or 5: y is exact in fp32
        weight = torch.from_numpy(values * c).float().cuda()
        q, scale, _ = add_rms_norm_quant(x, None, weight, 0.0, quant_dtype=quant)
        assert (scale == c).all()
        assert np.array_equal(as64(q.float()), np.broadcast_to(nearest, x.shape)), c


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('exponent', [-130, -100, -60, 0, 60, 110])
def test_ties_of_the_gate_round_to_even(quant, exponent):
    """A gate of 64 is its own silu, so y = 64 u, exactly: the ties are multiples of 2^-10, u of 2^-146 at least."""
    from micro_vllm_b200.row_ops import silu_mul_quant
    values, nearest = ties(quant)
    rows = np.array([1.0, 3.0, 5.0, 7.0, 11.0, 13.0, 77.0, 101.0, 127.0])
    u = torch.from_numpy(values * rows[:, None] * 2.0 ** (exponent - 6)).float()
    q, scale = silu_mul_quant(torch.cat([torch.full_like(u, 64.0), u], dim=-1).cuda(), quant_dtype=quant)
    assert np.array_equal(as64(scale), rows * 2.0 ** exponent)
    assert np.array_equal(as64(q.float()), np.broadcast_to(nearest, u.shape))
