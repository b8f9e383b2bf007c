"""CPU checks of which outputs of the row operations may lie over an input."""
import pytest
import torch

from micro_vllm_b200 import row_ops


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('quant', [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('rows', [1, 4])
def test_an_8_bit_output_is_never_the_input_itself(dtype, quant, rows):
    """Its address and its strides, counted in elements, are the input's, but its row r lies over an earlier row."""
    x = torch.zeros((rows, 64), dtype=dtype)
    out = x.view(torch.uint8).view(-1)[:rows * 64].view(rows, 64).view(quant)
    assert out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    with pytest.raises(RuntimeError, match='itself'):
        row_ops._disjoint(out, (x, None), same=(x,))
    row_ops._disjoint(x, (x, None), same=(x,))
    row_ops._disjoint(torch.zeros((rows, 64), dtype=quant), (x, None), same=(x,))


@pytest.mark.parametrize('rows', [1, 4])
def test_an_output_of_the_inputs_type_is_it_only_at_the_same_address_and_strides(rows):
    buffer = torch.zeros((rows + 1, 64))
    x = buffer[:rows]
    for out in (buffer[1:], buffer.view(-1)[32:rows * 64 + 32].view(rows, 64)):
        with pytest.raises(RuntimeError, match='itself'):
            row_ops._disjoint(out, (x,), same=(x,))
    row_ops._disjoint(buffer[:rows], (x,), same=(x,))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,width', [(1, 64), (4, 64), (1, 40000)])
def test_the_norm_and_the_gate_refuse_an_8_bit_output_over_their_input(dtype, rows, width):
    x = torch.ones((rows, width), dtype=dtype, device='cuda')
    w = torch.ones(width, dtype=dtype, device='cuda')
    out = x.view(torch.int8).view(-1)[:rows * width].view(rows, width)
    with pytest.raises(RuntimeError, match='itself'):
        row_ops.add_rms_norm_quant(x, None, w, 1e-6, out=out)
    with pytest.raises(RuntimeError, match='itself'):
        row_ops.add_rms_norm_quant(torch.ones_like(x), x, w, 1e-6, out=out)
    with pytest.raises(RuntimeError, match='itself'):
        row_ops.silu_mul_quant(x, out=x.view(torch.int8).view(-1)[:rows * width // 2].view(rows, width // 2))
    assert (x == 1).all()
