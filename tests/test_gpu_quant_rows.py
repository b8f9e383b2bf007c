"""add_rms_norm, add_rms_norm_quant and silu_mul_quant on the GPU against their formulas in 64 bits.

Tolerances. The norm's sum of squares has at most C = 64 terms per thread and 16 per
tree and loop behind it, each addition off by 2^-24 of the (positive) sum, so rsqrt
of the mean is off by less than 128 * 2^-24 / 2, and five more roundings (the two
products, rsqrt's two units, the division) stay below 2^-20 in all. silu_mul's exp
argument is rounded once (2^-24 of |g| <= 90 in the exponent) and exp, the division
and two products add a few 2^-23: below 2^-16 of the value for |g| up to 90, below
2^-19 up to 8. Rows wider than 32768 are summed by 512 threads in up to 32 turns of 8.
"""
import numpy as np
import pytest
import torch

from tests.w4_reference import HALF_STEP, TOP, as64, assert_quantized

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
EIGHT = [torch.int8, torch.float8_e4m3fn]
NORM_OFF = 2.0 ** -18
SHAPES = [(1, 8), (1, 1), (3, 7), (2, 33), (5, 257), (4, 896), (1, 3584), (700, 512), (2, 8192), (2, 8200), (3, 14336),
          (2, 16400), (400, 1000), (2, 28672), (1, 40000), (2, 16391), (301, 2047)]


def norm_inputs(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x, r = torch.randn(shape, generator=gen) * 2, torch.randn(shape, generator=gen) * 3
    w = 1 + 0.3 * torch.randn(shape[-1], generator=gen)
    return x.to(dtype), r.to(dtype), w.to(dtype)


def norm64(x, r, w, eps):
    s = (x.float() + r.float()).to(x.dtype) if r is not None else x
    s64 = as64(s)
    return s, as64(w) * s64 / np.sqrt((s64 ** 2).mean(-1, keepdims=True) + eps)


@pytest.mark.parametrize('dtype', FLOATS)
@pytest.mark.parametrize('shape', SHAPES)
def test_add_rms_norm(dtype, shape):
    from micro_vllm_b200.row_ops import add_rms_norm
    x, r, w = norm_inputs(shape, dtype, 1)
    out, total = add_rms_norm(x.cuda(), r.cuda(), w.cuda(), 1e-6)
    s, y = norm64(x, r, w, 1e-6)
    assert torch.equal(total.cpu(), s)
    subnormal = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert (np.abs(as64(out) - y) <= (HALF_STEP[dtype] * (1 + 2.0 ** -8) + NORM_OFF) * np.abs(y) + subnormal).all()


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('dtype', FLOATS)
@pytest.mark.parametrize('shape', SHAPES)
def test_add_rms_norm_quant(dtype, quant, shape):
    from micro_vllm_b200.row_ops import add_rms_norm_quant
    x, r, w = norm_inputs(shape, dtype, 2)
    q, scale, total = add_rms_norm_quant(x.cuda(), r.cuda(), w.cuda(), 1e-5, quant_dtype=quant)
    assert q.dtype == quant and scale.shape == shape[:-1]
    s, y = norm64(x, r, w, 1e-5)
    assert torch.equal(total.cpu(), s)
    assert_quantized(q, scale, y, quant, NORM_OFF)
    # Without a residual: s is x itself.
    q, scale, same = add_rms_norm_quant(x.cuda().contiguous(), None, w.cuda(), 1e-5, quant_dtype=quant)
    assert_quantized(q, scale, norm64(x, None, w, 1e-5)[1], quant, NORM_OFF)
    assert torch.equal(same.cpu(), x)


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('dtype', FLOATS)
@pytest.mark.parametrize('shape', SHAPES)
def test_silu_mul_quant(dtype, quant, shape):
    from micro_vllm_b200.row_ops import silu_mul_quant
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn((shape[0], 2 * shape[1]), generator=gen) * 2).to(dtype)
    q, scale = silu_mul_quant(x.cuda(), quant_dtype=quant)
    x64 = as64(x)
    g, u = x64[:, :shape[1]], x64[:, shape[1]:]
    assert np.abs(g).max() < 12
    assert_quantized(q, scale, g / (1 + np.exp(-g)) * u, quant, 2.0 ** -18)


@pytest.mark.parametrize('quant', EIGHT)
def test_far_gates(quant):
    from micro_vllm_b200.row_ops import silu_mul_quant
    g = torch.tensor([[-200.0, -90.0, -89.0, -30.0, 0.0, 30.0, 89.0, 200.0]])
    u = torch.tensor([[1e30, 1.0, 1e30, 2.0, 5.0, -3.0, 1.0, -1.0]])
    for row in range(8):  # each gate alone: values of every size
        x = torch.cat((g[:, row:row + 1], u[:, row:row + 1]), dim=-1)
        q, scale = silu_mul_quant(x.cuda(), quant_dtype=quant)
        g64, u64 = float(g[0, row]), float(u[0, row])
        y = np.array([[g64 / (1 + np.exp(-g64)) * u64]])
        if abs(y[0, 0]) < 2.0 ** -120 or g64 < -88:  # 1 + exp(-g) leaves fp32's range: a zero
            assert float(scale[0]) * abs(float(q.float()[0, 0])) <= abs(y[0, 0]) * (1 + 2.0 ** -12)
        else:
            assert_quantized(q, scale, y, quant, 2.0 ** -16)


@pytest.mark.parametrize('quant', EIGHT)
@pytest.mark.parametrize('width', [16, 17])
def test_rows_of_zeros_nan_infinities_and_tiny_values(quant, width):
    from micro_vllm_b200.row_ops import add_rms_norm_quant, silu_mul_quant
    x = torch.randn((7, width))
    x[0] = 0
    x[1, 3], x[2, 5], x[3, 6] = float('nan'), float('inf'), float('-inf')
    x[4] = 0
    x[4, 1] = 1e-42
    x[5] *= 1e-38
    w = torch.ones(width)
    q, scale, _ = add_rms_norm_quant(x.cuda(), None, w.cuda(), 0.0, quant_dtype=quant)
    q, scale = q.float().cpu(), scale.cpu()
    # Row 0 is 0 * rsqrt(0) = NaN with eps 0; rows 1 to 3 hold what is not finite.
    assert torch.isnan(scale[:4]).all() and not q[:4].any()
    q, scale, _ = add_rms_norm_quant(x.cuda(), None, w.cuda(), 1e-6, quant_dtype=quant)
    assert scale[0] == 0 and not q[0].float().any()
    assert torch.isnan(scale[1:4]).all() and not q[1:4].float().any()
    # Tiny rows keep their direction: y = 1e3 x, its scale a number that fp32 still holds.
    assert q[4].float().abs().max() == TOP[quant] and scale[4] > 0
    assert_quantized(q[6:], scale[6:], norm64(x[6:], None, w, 1e-6)[1], quant, NORM_OFF)
    q5 = as64(q[5].float())
    y5 = norm64(x[5:6], None, w, 1e-6)[1][0]
    assert (np.abs(q5 - y5 / np.abs(y5).max() * TOP[quant]) <= (0.51 if quant == torch.int8 else 18.0)).all()

    gate = torch.randn((3, 2 * width))
    gate[0, 1], gate[1, width + 2] = float('nan'), float('inf')
    q, scale = silu_mul_quant(gate.cuda(), quant_dtype=quant)
    assert torch.isnan(scale[:2]).all() and not q[:2].float().any() and torch.isfinite(scale[2])
    q, scale = silu_mul_quant(torch.zeros((2, 2 * width), device='cuda'), quant_dtype=quant)
    assert not scale.any() and not q.float().any()


@pytest.mark.parametrize('dtype', FLOATS)
def test_strided_rows_in_place_and_what_lies_around(dtype):
    from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant, silu_mul_quant
    x, r, w = norm_inputs((6, 264), dtype, 5)
    s, y = norm64(x, r, w, 1e-6)
    expected, total = add_rms_norm(x.cuda(), r.cuda(), w.cuda(), 1e-6)
    for offset in (0, 8, 3):
        wide = torch.zeros((6, 300), dtype=dtype, device='cuda')
        wide[:, offset:offset + 264] = x.cuda()
        stream = torch.full((6, 301), 9.0, dtype=dtype, device='cuda')
        stream[:, 2:266] = r.cuda()
        view = wide[:, offset:offset + 264]
        out, got = add_rms_norm(view, stream[:, 2:266], w.cuda(), 1e-6, out=view, residual_out=stream[:, 2:266])
        bound = (HALF_STEP[dtype] * 1.01 + NORM_OFF) * np.abs(y) + 2.0 ** -25
        assert (np.abs(as64(view) - y) <= bound).all() and torch.equal(got.cpu(), s)
        assert (stream[:, :2] == 9).all() and (stream[:, 266:] == 9).all() and not wide[:, offset + 264:].any()
        q = torch.full((6, 280), 1, dtype=torch.int8, device='cuda')
        scale = torch.empty(6, device='cuda')
        add_rms_norm_quant(x.cuda(), r.cuda(), w.cuda(), 1e-6, out=q[:, 5:269], scales=scale)
        assert_quantized(q[:, 5:269], scale, y, torch.int8, NORM_OFF)
        assert (q[:, :5] == 1).all() and (q[:, 269:] == 1).all()
    place = x.cuda()
    out, got = add_rms_norm(place, r.cuda(), w.cuda(), 1e-6, residual_out=place)
    assert got is place and torch.equal(place.cpu(), s) and torch.equal(out, expected)
    q, scale = silu_mul_quant(torch.randn((2, 3, 64), device='cuda').to(dtype))
    assert q.shape == (2, 3, 32) and scale.shape == (2, 3)


@pytest.mark.parametrize('width', [40000, 40001])
def test_wide_rows_in_place(width):
    """Rows that no thread's registers hold are read twice: the sum may already lie over an input."""
    from micro_vllm_b200.row_ops import add_rms_norm
    x, r, w = norm_inputs((2, width), torch.bfloat16, 6)
    s, y = norm64(x, r, w, 1e-6)
    for target in ('x', 'r', None):
        dx, dr = x.cuda(), r.cuda()
        out, total = add_rms_norm(dx, dr, w.cuda(), 1e-6, residual_out={'x': dx, 'r': dr, None: None}[target])
        assert torch.equal(total.cpu(), s)
        assert (np.abs(as64(out) - y) <= (HALF_STEP[torch.bfloat16] * 1.01 + NORM_OFF) * np.abs(y)).all()


def test_refusals():
    from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant, silu_mul_quant
    x = torch.zeros((4, 64), device='cuda', dtype=torch.bfloat16)
    w = torch.ones(64, device='cuda', dtype=torch.bfloat16)
    for call, message in [
        (lambda: add_rms_norm(x, None, w, 1e-6), 'residual'),
        (lambda: add_rms_norm(x, x[:3], w, 1e-6), 'match'),
        (lambda: add_rms_norm(x, x.float(), w, 1e-6), 'match'),
        (lambda: add_rms_norm(x, x.clone(), w[:63], 1e-6), 'weight'),
        (lambda: add_rms_norm(x, x.clone(), w, -1.0), 'eps'),
        (lambda: add_rms_norm(x, x.clone(), w, float('nan')), 'eps'),
        (lambda: add_rms_norm(x, x.clone().requires_grad_(), w, 1e-6), 'gradients'),
        (lambda: add_rms_norm(x.cpu(), x.cpu(), w.cpu(), 1e-6), 'CUDA'),
        (lambda: add_rms_norm(x, x.clone(), w, 1e-6, out=x[:2]), 'out'),
        (lambda: add_rms_norm(x, x.clone(), w, 1e-6, out=x, residual_out=x), 'itself'),
        (lambda: add_rms_norm(x, x.clone(), w, 1e-6, residual_out=torch.zeros_like(x[:1]).expand(4, 64)), 'overlap'),
        (lambda: add_rms_norm_quant(x, None, w, 1e-6, quant_dtype=torch.uint8), 'quant_dtype'),
        (lambda: add_rms_norm_quant(x, None, w, 1e-6, residual_out=x), 'residual'),
        (lambda: add_rms_norm_quant(x, None, w, 1e-6, out=torch.zeros_like(x)), 'out'),
        (lambda: add_rms_norm_quant(x, None, w, 1e-6, scales=torch.zeros(3, device='cuda')), 'scales'),
        (lambda: silu_mul_quant(x[:, :63].contiguous()), 'halves'),
        (lambda: silu_mul_quant(x, quant_dtype=torch.bfloat16), 'quant_dtype'),
        (lambda: silu_mul_quant(x, out=x.view(torch.int8)[:, :32]), 'itself|memory'),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
    buffer = torch.zeros((6, 64), device='cuda', dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='itself'):
        add_rms_norm(buffer[:4], x, w, 1e-6, residual_out=buffer[1:5])
    empty = add_rms_norm_quant(x[:0], None, w, 1e-6)
    assert empty[0].shape == (0, 64) and empty[1].shape == (0,)


def test_replayed_graph_and_streams_give_the_same_bits():
    from micro_vllm_b200.row_ops import add_rms_norm_quant, silu_mul_quant
    x, r, w = (t.cuda() for t in norm_inputs((300, 896), torch.bfloat16, 7))
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, scale, total = add_rms_norm_quant(static, r, w, 1e-6)
        q2, scale2 = silu_mul_quant(total)
    for v in (x * 2, x):
        static.copy_(v)
        graph.replay()
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            eager = add_rms_norm_quant(v, r, w, 1e-6)
            eager2 = silu_mul_quant(eager[2])
        torch.cuda.synchronize()
        for a, b in zip((q, scale, total, q2, scale2), eager + eager2):
            assert torch.equal(a, b)
