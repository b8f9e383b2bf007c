"""w4_linear and w4_dequantize on the GPU against their formulas in 64 bits.

Tolerances. Products of the kernel are exact (a code's distance from its zero
point is a small integer). What is left is addition: the tensor core adds 16 or 32
products to an fp32 number at a time and may drop bits below 2^-23 of the largest
addend, so a sum of `steps` additions is within steps * 2^-22 * sum|x w| (a factor
of two for the addends' own size), and the last rounding is half a step of the
result's type.
"""
import numpy as np
import pytest
import torch

from tests.w4_reference import HALF_STEP, as64, checkpoint, dense

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def activations(m, k, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=gen)
    if dtype == torch.int8:
        return torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8), torch.rand(m, generator=gen) + 0.01
    if dtype == torch.float8_e4m3fn:
        return (x * 100).to(dtype), torch.rand(m, generator=gen) + 0.01
    return x.to(dtype), None


def assert_linear(y, x, x_scale, w, bias=None, residual=None, group=32):
    x64 = as64(x.float()) * (1.0 if x_scale is None else as64(x_scale)[:, None])
    expected, size = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    for more in (bias, residual):
        if more is not None:
            expected = expected + as64(more)
            size = size + np.abs(as64(more))
    planes = 3 if x.dtype == torch.float32 else 1
    steps = planes * (-(-w.shape[1] // 16)) + -(-w.shape[1] // group) + 32 + 3
    bound = steps * 2.0 ** -22 * size + HALF_STEP[y.dtype] * np.abs(expected) * (1 + 2.0 ** -8) + 2.0 ** -126
    if y.dtype == torch.float16:
        bound += 2.0 ** -25  # half a step of a subnormal
    actual, nan = as64(y).reshape(expected.shape), np.isnan(expected)  # a value past e4m3's largest is a NaN in x
    assert np.array_equal(np.isnan(actual), nan)
    error, bound = np.abs(actual - expected)[~nan], bound[~nan]
    assert (error <= bound).all(), (float((error / bound).max()), int((error > bound).sum()))


def make(n, k, group=128, zeros=False, scale_dtype=torch.bfloat16, seed=0):
    from micro_vllm_b200.w4_linear import pack_w4
    codes, scales, zero = checkpoint(n, k, group, zeros, scale_dtype, seed)
    weight = pack_w4(codes.cuda(), scales.cuda(), None if zero is None else zero.cuda(), group_size=group)
    return weight, dense(codes, scales, zero, group)


@pytest.mark.parametrize('dtype', FLOATS + [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('m,k,n', [(1, 128, 64), (3, 200, 70), (8, 1024, 192), (13, 640, 64), (31, 520, 130)])
def test_every_type_group_and_zero_point(dtype, group, zeros, m, k, n):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(n, k, group, zeros, torch.float16 if group == 64 else torch.bfloat16, seed=m)
    x, scale = activations(m, k, dtype, seed=k)
    out_dtype = dtype if dtype in FLOATS else torch.float32
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=out_dtype)
    assert y.shape == (m, n) and y.dtype == out_dtype
    assert_linear(y, x, scale, w, group=group)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('m', [1, 2, 7, 8, 9, 15, 16, 17, 32, 33, 63, 64, 65, 100, 129, 257])
def test_token_counts(dtype, m):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(100, 384, seed=m)
    x, scale = activations(m, 384, dtype, seed=m)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.bfloat16)
    assert_linear(y, x, scale, w, group=128)


@pytest.mark.parametrize('dtype', FLOATS + [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('m', [12, 30, 33, 64, 65, 128, 130])
@pytest.mark.parametrize('k', [840, 1153])
def test_groups_at_every_token_block(dtype, group, zeros, m, k):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(200, k, group, zeros, seed=m + k)
    x, scale = activations(m, k, dtype, seed=k)
    out_dtype = dtype if dtype in FLOATS else torch.bfloat16
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=out_dtype)
    assert_linear(y, x, scale, w, group=group)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.int8])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('m', [16, 64, 128])
def test_long_columns_of_every_group_and_token_block(dtype, group, m):
    """Many turns of every buffer and barrier, with bias and residual."""
    from micro_vllm_b200.w4_linear import w4_linear
    k, n = 14336, 384
    gen = torch.Generator().manual_seed(m)
    weight, w = make(n, k, group, True, seed=m)
    x, scale = activations(m, k, dtype, seed=group)
    bias, residual = torch.randn(n, generator=gen).bfloat16(), torch.randn((m, n), generator=gen).bfloat16()
    y = w4_linear(x.cuda(), weight, bias.cuda(), residual.cuda(), x_scale=None if scale is None else scale.cuda())
    assert_linear(y, x, scale, w, bias, residual, group=group)


@pytest.mark.parametrize('dtype', FLOATS + [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('k', [1, 2, 7, 8, 31, 33, 127, 129, 255, 1001, 4097])
@pytest.mark.parametrize('n', [1, 63, 65])
def test_odd_sizes(dtype, k, n):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(n, k, 32, True, torch.float16, seed=k)
    x, scale = activations(5, k, dtype, seed=n)
    out_dtype = dtype if dtype in FLOATS else torch.float16
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=out_dtype)
    assert_linear(y, x, scale, w)


@pytest.mark.parametrize('k,n,m', [(3584, 4608, 1), (14336, 3584, 16), (18000, 72, 4), (128, 20000, 2), (896, 1152, 64)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.int8])
def test_splits_of_long_columns_and_many_rows(dtype, k, n, m):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(n, k, seed=3)
    x, scale = activations(m, k, dtype, seed=4)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.bfloat16)
    assert_linear(y, x, scale, w, group=128)


@pytest.mark.parametrize('out_dtype', FLOATS)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.int8])
def test_bias_and_residual(dtype, out_dtype):
    from micro_vllm_b200.w4_linear import w4_linear
    gen = torch.Generator().manual_seed(9)
    weight, w = make(201, 300, seed=1)
    x, scale = activations(6, 300, dtype, seed=2)
    bias, residual = torch.randn(201, generator=gen).to(out_dtype), torch.randn((6, 201), generator=gen).to(out_dtype)
    args = dict(x_scale=None if scale is None else scale.cuda())
    y = w4_linear(x.cuda(), weight, bias.cuda(), residual.cuda(), **args)
    assert y.dtype == out_dtype
    assert_linear(y, x, scale, w, bias, residual, group=128)
    # In place over the residual: the same bits.
    place = residual.cuda()
    assert w4_linear(x.cuda(), weight, bias.cuda(), place, out=place, **args) is place
    assert torch.equal(place, y)
    assert_linear(w4_linear(x.cuda(), weight, bias.cuda(), out_dtype=out_dtype, **args), x, scale, w, bias, group=128)


def test_strided_rows_and_what_lies_around_them():
    """Rows of wider tensors, at offsets that allow no vector load; nothing beside the output changes."""
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(130, 256, 64, True, seed=5)
    for offset in (0, 1, 8):
        wide = torch.full((9, 300), float('nan'), dtype=torch.bfloat16)
        x, _ = activations(9, 256, torch.bfloat16, seed=6)
        wide[:, offset:offset + 256] = x
        out = torch.full((9, 200), 7.0, dtype=torch.bfloat16, device='cuda')
        residual = torch.randn((9, 260)).to(torch.bfloat16)
        y = w4_linear(wide.cuda()[:, offset:offset + 256], weight, residual=residual.cuda()[:, 3:133],
                      out=out[:, 11:141])
        assert (out[:, :11] == 7).all() and (out[:, 141:] == 7).all()
        assert_linear(y, x, None, w, residual=residual[:, 3:133], group=64)


def test_broadcast_rows_and_leading_dimensions():
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(64, 128, seed=7)
    x, _ = activations(1, 128, torch.bfloat16, seed=8)
    y = w4_linear(x.cuda().expand(4, 128), weight)
    assert torch.equal(y, w4_linear(x.cuda(), weight).expand(4, 64))
    assert_linear(y[:1], x, None, w, group=128)
    x3, _ = activations(6, 128, torch.bfloat16, seed=8)
    y3 = w4_linear(x3.view(2, 3, 128).cuda(), weight)
    assert y3.shape == (2, 3, 64) and torch.equal(y3.view(6, 64), w4_linear(x3.cuda(), weight))
    assert w4_linear(x.cuda()[0], weight).shape == (64,)
    assert w4_linear(torch.empty((0, 128), device='cuda', dtype=torch.bfloat16), weight).shape == (0, 64)


@pytest.mark.parametrize('dtype', FLOATS + [torch.float8_e4m3fn])
def test_rows_with_nan_and_infinities_leave_the_others_alone(dtype):
    from micro_vllm_b200.w4_linear import w4_linear
    n, k = 64, 256
    weight, w = make(n, k, 128, True, seed=11)
    x, scale = activations(4, k, dtype, seed=12)
    x = x.float()
    x[1, 77] = float('nan')
    if dtype != torch.float8_e4m3fn:
        x[2, 5] = float('inf')
    x = x.to(dtype)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.float32).cpu()
    assert torch.isnan(y[1]).all()
    if dtype != torch.float8_e4m3fn:  # an infinity times W[:, 5]: its sign, NaN where the weight is zero
        expected = torch.where(torch.from_numpy(w[:, 5]) == 0, torch.nan, torch.from_numpy(np.sign(w[:, 5])) * torch.inf)
        assert torch.equal(torch.nan_to_num(y[2].double(), nan=5.0), torch.nan_to_num(expected, nan=5.0))
    keep = [0, 3]
    assert_linear(y[keep], x[keep], None if scale is None else scale[keep], w, group=128)


def test_large_values_of_fp32_and_fp16_rows():
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(64, 128, seed=13)
    x = torch.zeros((2, 128))
    x[0, 3], x[1, 4] = torch.finfo(torch.float32).max / 4, 2.0 ** -120
    y = w4_linear(x.cuda(), weight)
    assert_linear(y, x, None, w, group=128)
    half = torch.full((1, 128), 65504.0, dtype=torch.float16)
    assert_linear(w4_linear(half.cuda(), weight, out_dtype=torch.float32), half, None, w, group=128)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.int8])
def test_same_bits_for_every_call_alone_replayed_and_on_other_streams(dtype):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(512, 4096, seed=14)
    x, scale = activations(16, 4096, dtype, seed=15)
    xs = [x.cuda(), (x.float() * 0.5).to(dtype).cuda()]
    kw = dict(x_scale=None if scale is None else scale.cuda(), out_dtype=torch.bfloat16)
    expected = [w4_linear(v, weight, **kw) for v in xs]
    assert_linear(expected[0], x, scale, w, group=128)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for turn in range(6):  # two calls at once
        with torch.cuda.stream(streams[turn % 3]):
            outs.append((turn % 2, w4_linear(xs[turn % 2], weight, **kw)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, expected[i]) for i, y in outs)
    static, out = xs[0].clone(), torch.empty_like(expected[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        w4_linear(static, weight, out=out, **kw)
        w4_linear(static, weight, out=out, **kw)
    for i in (1, 0, 1):
        static.copy_(xs[i])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected[i])


def test_a_weight_that_the_call_before_wrote_is_the_one_that_is_read():
    """The launch may start before the kernel ahead of it ends; what that kernel wrote must be seen."""
    from micro_vllm_b200.w4_linear import W4Weight, w4_linear
    a, wa = make(4096, 2048, seed=16)
    b, wb = make(4096, 2048, seed=17)
    records = torch.empty_like(a.records)
    live = W4Weight(records, a.shape, a.group_size, a.has_zeros, a.scale_dtype)
    x, _ = activations(4, 2048, torch.bfloat16, seed=18)
    x = x.cuda()
    expected = [w4_linear(x, a), w4_linear(x, b)]
    assert_linear(expected[1], x, None, wb, group=128)
    for turn in range(20):
        records.copy_((a, b)[turn % 2].records)
        y = w4_linear(x, live)
        assert torch.equal(y, expected[turn % 2])


@pytest.mark.parametrize('dtype', FLOATS)
@pytest.mark.parametrize('group,zeros', [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize('n,k', [(1, 1), (64, 128), (65, 129), (70, 1000), (200, 333), (3, 8)])
def test_dequantize_is_the_formula_rounded_once(dtype, group, zeros, n, k):
    from micro_vllm_b200.w4_linear import w4_dequantize
    for scale_dtype in (torch.float16, torch.bfloat16):
        weight, w = make(n, k, group, zeros, scale_dtype, seed=n + k)
        # (code - zero) * scale has at most 4 + 11 bits: exact in fp32 and 64 bits, so the rounding is the only one.
        expected = torch.from_numpy(w).to(torch.float32).to(dtype)
        assert torch.equal(w4_dequantize(weight, dtype).cpu(), expected)
        wide = torch.full((n, k + 9), 3.0, dtype=dtype, device='cuda')
        w4_dequantize(weight, out=wide[:, 1:k + 1])
        assert torch.equal(wide[:, 1:k + 1].cpu(), expected)
        assert (wide[:, 0] == 3).all() and (wide[:, k + 1:] == 3).all()
    assert w4_dequantize(weight).dtype == torch.bfloat16


def test_offsets_past_32_bits():
    """Records and outputs of more than 2^32 bytes: the last rows against the formula."""
    from micro_vllm_b200.w4_linear import W4Weight, w4_dequantize, w4_linear
    n, k = 70000, 131072  # 4.7 GB of records
    tile, w = make(64, k, seed=20)
    tiles = -(-n // 64)
    records = tile.records.expand(tiles, -1, -1).contiguous()
    records[:-1, :, 4096:] = 0  # scales of all but the last tile: zero
    weight = W4Weight(records, (n, k), 128, False, tile.scale_dtype)
    x, _ = activations(2, k, torch.bfloat16, seed=21)
    y = w4_linear(x.cuda(), weight, out_dtype=torch.float32)
    last = (tiles - 1) * 64
    assert (y[:, :last] == 0).all()
    assert_linear(y[:, last:], x, None, w[:n - last], group=128)
    out = w4_dequantize(weight, torch.bfloat16)  # 18 GB
    assert torch.equal(out[last:].cpu(), torch.from_numpy(w[:n - last]).float().to(torch.bfloat16))
    assert not out[last - 64:last].any()


def test_quantize_then_linear_equals_the_dequantized_product():
    from micro_vllm_b200.w4_linear import quantize_w4, w4_dequantize, w4_linear
    gen = torch.Generator(device='cuda').manual_seed(22)
    for zeros in (False, True):
        dense_weight = torch.randn((300, 700), generator=gen, device='cuda').to(torch.bfloat16)
        weight = quantize_w4(dense_weight, group_size=64, zeros=zeros)
        w = w4_dequantize(weight, torch.float32)
        x, _ = activations(3, 700, torch.bfloat16, seed=23)
        assert_linear(w4_linear(x.cuda(), weight), x, None, as64(w), group=64)


def test_refusals_on_cuda_tensors():
    from micro_vllm_b200.w4_linear import w4_dequantize, w4_linear
    weight, _ = make(64, 128)
    x = torch.zeros((2, 128), device='cuda', dtype=torch.bfloat16)
    scale = torch.ones(2, device='cuda')
    out = torch.zeros((2, 64), device='cuda', dtype=torch.bfloat16)
    bad = [
        (dict(x=x[:, :64]), 'features'),
        (dict(x=x.to(torch.float64)), 'float32, float16'),
        (dict(x=x.to(torch.int8)), 'x_scale|out_dtype'),
        (dict(x=x.to(torch.int8), out_dtype=torch.bfloat16), 'x_scale'),
        (dict(x=x.to(torch.int8), x_scale=scale), 'out_dtype'),
        (dict(x=x, x_scale=scale[:1]), 'one per row'),
        (dict(x=x, x_scale=scale.to(torch.float16)), 'float32'),
        (dict(x=x.t().contiguous().t()), 'stride 1'),
        (dict(x=x.clone().requires_grad_()), 'gradients'),
        (dict(x=x, bias=torch.zeros(63, device='cuda', dtype=torch.bfloat16)), 'bias'),
        (dict(x=x, bias=torch.zeros(64, device='cuda'), out_dtype=torch.bfloat16), 'bias'),
        (dict(x=x, residual=out[:1]), 'residual'),
        (dict(x=x, out=out[:1]), 'out must'),
        (dict(x=x, out=out[:1].expand(2, 64)), 'overlap'),
        (dict(x=x, out=out, residual=out[:, :].flip(0).as_strided((2, 64), (64, 1), 0)), None),
        (dict(x=x, out=x[:, :64]), 'alias'),
        (dict(x=x, residual=torch.zeros((4, 64), device='cuda', dtype=torch.bfloat16)[1:3]), None),
        (dict(x=x.cpu()), 'CUDA'),
        (dict(x=x, out_dtype=torch.int8), 'out_dtype'),
    ]
    for kw, message in bad:
        if message is None:
            w4_linear(kw.pop('x'), weight, **kw)
            continue
        with pytest.raises(RuntimeError, match=message):
            w4_linear(kw.pop('x'), weight, **kw)
    buffer = torch.zeros((4, 64), device='cuda', dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='residual itself'):
        w4_linear(x, weight, residual=buffer[:2], out=buffer[1:3])
    with pytest.raises(RuntimeError, match='dtype'):
        w4_dequantize(weight, torch.int8)
    with pytest.raises(RuntimeError, match='out must'):
        w4_dequantize(weight, torch.bfloat16, out=out)
