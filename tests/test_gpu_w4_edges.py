"""The 4-bit layer where its callers meet it: more rows than a grid has blocks for, rows that TMA cannot copy,
first calls inside a capture, neighbours on other streams, memory that the call before wrote, copies of a weight.

Tolerances as in test_gpu_w4_linear.py.
"""
import copy
import ctypes
import pickle
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.test_gpu_w4_linear import FLOATS, activations, assert_linear, make

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.int8])
def test_more_rows_than_a_launch_takes(dtype):
    """A launch takes 65535 * 8 rows: the rows after them are those of a second one."""
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(8, 32, 32, seed=30)
    m = 65535 * 8 + 5
    x, scale = activations(m, 32, dtype, seed=31)
    residual = torch.randn((m, 8), generator=torch.Generator().manual_seed(32))
    y = w4_linear(x.cuda(), weight, residual=residual.cuda(), x_scale=None if scale is None else scale.cuda())
    for rows in (slice(0, 40), slice(65535 * 8 - 20, m)):
        assert_linear(y[rows], x[rows], None if scale is None else scale[rows], w, residual=residual[rows], group=32)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('m', [9, 33, 65])
@pytest.mark.parametrize('offset,width', [(0, 272), (16, 272), (1, 271), (8, 264), (3, 272)])
def test_rows_of_wider_tensors_at_every_token_block(dtype, m, offset, width):
    """k = 200: a last chunk of 72 columns, beside which the wider rows hold NaN (or 127)."""
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(130, 200, 64, True, seed=33)
    x, scale = activations(m, 200, dtype, seed=34)
    wide = torch.full((m, width), 127.0 if dtype == torch.int8 else float('nan')).to(dtype)
    wide[:, offset:offset + 200] = x
    y = w4_linear(wide.cuda()[:, offset:offset + 200], weight, out_dtype=torch.float32,
                  x_scale=None if scale is None else scale.cuda())
    assert_linear(y, x, scale, w, group=64)


@pytest.mark.parametrize('m', [12, 40, 100])
def test_broadcast_and_overlapping_rows_in_place_and_around(m):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(200, 256, seed=35)
    x, _ = activations(1, 256, torch.bfloat16, seed=36)
    y = w4_linear(x.cuda().expand(m, 256), weight)
    assert torch.equal(y, y[:1].expand(m, 200))
    assert_linear(y[:1], x, None, w, group=128)
    line, _ = activations(1, 256 + 8 * m, torch.bfloat16, seed=37)  # rows that start 8 apart
    sliding = line.flatten().as_strided((m, 256), (8, 1))
    assert_linear(w4_linear(line.cuda().flatten().as_strided((m, 256), (8, 1)), weight), sliding, None, w, group=128)
    around = torch.full((m + 2, 210), 7.0, dtype=torch.bfloat16, device='cuda')
    place = around[1:m + 1, 5:205]
    residual = torch.randn((m, 200), generator=torch.Generator().manual_seed(38)).to(torch.bfloat16)
    place.copy_(residual)
    assert w4_linear(sliding.cuda(), weight, residual=place, out=place) is place
    assert_linear(place, sliding, None, w, residual=residual, group=128)
    place.fill_(7.0)
    assert (around == 7).all()
    one = residual[:1].cuda()
    y = w4_linear(sliding.cuda(), weight, residual=one.expand(m, 200))
    assert_linear(y, sliding, None, w, residual=residual[:1].expand(m, 200), group=128)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize('m', [12, 40, 100])
def test_rows_with_nan_leave_the_others_alone_at_every_token_block(dtype, m):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(128, 384, 128, True, seed=39)
    x, scale = activations(m, 384, dtype, seed=40)
    x = x.float().nan_to_num(0.0)
    x[3, 77] = float('nan')
    x = x.to(dtype)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.float32).cpu()
    assert torch.isnan(y[3]).all()
    keep = [i for i in range(m) if i != 3]
    assert_linear(y[keep], x[keep], None if scale is None else scale[keep], w, group=128)


@pytest.mark.parametrize('m', [4, 16, 48, 128])
def test_what_the_calls_before_wrote_is_what_is_read(m):
    """Weights and rows rewritten between calls on one stream, with no wait of the host."""
    from micro_vllm_b200.w4_linear import W4Weight, w4_linear
    pairs = [make(2048, 2048, seed=s) for s in (41, 42)]
    a = pairs[0][0]
    live = W4Weight(torch.empty_like(a.records), a.shape, a.group_size, a.has_zeros, a.scale_dtype)
    x = [activations(m, 2048, torch.bfloat16, seed=s)[0].cuda() for s in (43, 44)]
    rows = torch.empty_like(x[0])
    expected = [w4_linear(x[i], pairs[i][0]) for i in (0, 1)]
    assert_linear(expected[1], x[1].cpu(), None, pairs[1][1], group=128)
    for turn in range(20):
        live.records.copy_(pairs[turn % 2][0].records)
        rows.copy_(x[turn % 2])
        assert torch.equal(w4_linear(rows, live), expected[turn % 2])
    # A chain in which each call reads what the one before wrote, and overwrites what it read.
    chain = [x[0].clone(), torch.empty_like(x[0])]
    for turn in range(6):
        w4_linear(chain[turn % 2], pairs[turn % 2][0], out=chain[1 - turn % 2])
    z = x[0].clone()
    for turn in range(6):
        torch.cuda.synchronize()
        z = w4_linear(z, pairs[turn % 2][0])
    assert torch.equal(z, chain[0])


def test_tensor_memory_is_shared_with_other_streams_kernels():
    """Products of 512 and of 256 tensor-memory columns and a prompt's attention, at once on four streams."""
    from micro_vllm_b200.cuda_attention import paged_chunk_attention
    from micro_vllm_b200.w4_linear import w4_linear
    weight, _ = make(4096, 4096, seed=45)
    xs = [activations(m, 4096, torch.bfloat16, seed=m)[0].cuda() for m in (16, 64, 128)]
    gen = torch.Generator().manual_seed(46)
    q = torch.randn((2, 8, 256, 128), generator=gen).to(torch.bfloat16).cuda()
    k, v = (torch.randn((32, 2, 16, 128), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    table = torch.randperm(32, generator=gen).view(2, 16).to(torch.int32).cuda()
    lens = torch.full((2,), 256, dtype=torch.int32, device='cuda')

    def attention():
        return paged_chunk_attention(q, k, v, table, lens, max_context_len=256)

    calls = [lambda x=x: w4_linear(x, weight) for x in xs] + [attention]
    expected = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [[] for _ in calls]
    for _ in range(10):
        for call, stream, out in zip(calls, streams, outs):
            with torch.cuda.stream(stream):
                out.append(call())
    torch.cuda.synchronize()
    for out, right in zip(outs, expected):
        assert all(torch.equal(y, right) for y in out)


def test_first_calls_inside_a_capture():
    """In a process whose every first call of a kernel is captured, the replay gives what eager calls give."""
    code = '''
import sys
sys.path.insert(0, 'micro-vllm_b200')
import torch
from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant, silu_mul_quant
from micro_vllm_b200.w4_linear import pack_w4, w4_dequantize, w4_linear
gen = torch.Generator().manual_seed(0)
weight = pack_w4(torch.randint(0, 16, (512, 256), generator=gen, dtype=torch.uint8).cuda(),
                 torch.rand((512, 2), generator=gen).half().cuda())
x = [torch.randn((m, 256), generator=gen).bfloat16().cuda() for m in (2, 16, 128)]
g = torch.ones(256, dtype=torch.bfloat16, device='cuda')
def calls():
    out = [w4_linear(v, weight) for v in x] + [w4_dequantize(weight), *add_rms_norm(x[1], x[1], g, 1e-6)]
    q, s, _ = add_rms_norm_quant(x[1], None, g, 1e-6)
    q2, s2 = silu_mul_quant(out[1])
    return out + [q, s, q2, s2, w4_linear(q, weight, x_scale=s, out_dtype=torch.bfloat16)]
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    captured = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, calls()))
'''
    run = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


def test_copies_of_a_weight_have_their_own_records():
    from micro_vllm_b200.w4_linear import w4_dequantize, w4_linear
    weight, w = make(100, 200, 32, True, seed=47)
    x, _ = activations(3, 200, torch.float32, seed=48)
    y = w4_linear(x.cuda(), weight)
    for other in (copy.copy(weight), copy.deepcopy(weight), pickle.loads(pickle.dumps(weight)),
                  weight.to('cpu').to('cuda')):
        assert other.fixed[0] == other.records.data_ptr() and other.shape == weight.shape
        assert torch.equal(w4_linear(x.cuda(), other), y)
        assert torch.equal(w4_dequantize(other), w4_dequantize(weight))


def test_device_status_stays_clear_and_a_bad_device_leaves_no_error_behind():
    from micro_vllm_b200 import _native, _quant_native
    from micro_vllm_b200.w4_linear import w4_linear
    lib = _quant_native.library()
    weight, _ = make(256, 1024, seed=49)
    status = ctypes.c_uint32(5)
    _quant_native.check(lib.mvq_clear_device_status(0))
    for m in (1, 16, 128):
        w4_linear(torch.ones((m, 1024), device='cuda:0', dtype=torch.bfloat16), weight)
    _quant_native.check(lib.mvq_device_status(0, ctypes.byref(status)))
    assert status.value == 0
    with pytest.raises(_native.NativeError):
        _quant_native.check(lib.mvq_device_status(1000, ctypes.byref(status)))
    with pytest.raises(_native.NativeError):
        _quant_native.check(lib.mvq_clear_device_status(1000))
    assert torch.ones(3, device='cuda').sum().item() == 3  # torch finds no error of ours
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize('dtype', FLOATS)
def test_calls_that_the_short_way_leaves_to_the_checked_one_agree_with_it(dtype):
    """Subclasses, inference tensors, parameters without gradients, whole-number eps, 3-D residuals."""
    from micro_vllm_b200.row_ops import add_rms_norm
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(96, 160, seed=50)
    x, _ = activations(12, 160, dtype, seed=51)
    residual = torch.randn((12, 96), generator=torch.Generator().manual_seed(52)).to(dtype)
    y = w4_linear(x.cuda(), weight, residual=residual.cuda())
    assert_linear(y, x, None, w, residual=residual, group=128)
    assert torch.equal(w4_linear(torch.nn.Parameter(x.cuda(), requires_grad=False), weight, residual=residual.cuda()), y)
    with torch.no_grad():
        assert torch.equal(w4_linear(torch.nn.Parameter(x.cuda()), weight, residual=residual.cuda()), y)
    with torch.inference_mode():
        assert torch.equal(w4_linear(x.cuda(), weight, residual=residual.cuda()), y)
    assert torch.equal(w4_linear(x.cuda().view(3, 4, 160), weight, residual=residual.cuda().view(3, 4, 96)),
                       y.view(3, 4, 96))
    g = torch.ones(96, dtype=dtype, device='cuda')
    a, b = add_rms_norm(y, y, g, 1), add_rms_norm(y, y, g, 1.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('m', [4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize('k,n', [(2048, 128), (2176, 4160), (2176, 64)])
def test_both_sides_of_the_rule_between_the_two_kernels(dtype, m, k, n):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(n, k, 128, True, seed=53)
    x, scale = activations(m, k, dtype, seed=54)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.float32)
    assert_linear(y, x, scale, w, group=128)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize('m', [17, 40, 100, 250])
@pytest.mark.parametrize('k,n', [(2048, 64), (256, 19072), (1152, 9500)])
def test_few_and_many_weight_rows_at_every_count_of_tokens(dtype, m, k, n):
    """Few weight rows take narrow passes over many tokens, many weight rows wide ones."""
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(n, k, 64, False, seed=55)
    x, scale = activations(m, k, dtype, seed=56)
    y = w4_linear(x.cuda(), weight, x_scale=None if scale is None else scale.cuda(), out_dtype=torch.float32)
    assert_linear(y, x, scale, w, group=64)


@pytest.mark.parametrize('m', [9, 16, 33, 70, 128])
@pytest.mark.parametrize('group', [32, 128])
def test_e4m3_rows_over_long_columns_give_the_same_bits_each_time(m, group):
    from micro_vllm_b200.w4_linear import w4_linear
    weight, w = make(300, 8256, group, True, seed=57)
    x, scale = activations(m, 8256, torch.float8_e4m3fn, seed=58)
    args = dict(x_scale=scale.cuda(), out_dtype=torch.float32)
    x_gpu = x.cuda()
    y = w4_linear(x_gpu, weight, **args)
    assert_linear(y, x, scale, w, group=group)
    for _ in range(30):
        again = w4_linear(x_gpu, weight, **args)
        assert torch.equal(torch.nan_to_num(again, nan=0.5), torch.nan_to_num(y, nan=0.5))


@pytest.mark.parametrize('rows', [1, 700])
@pytest.mark.parametrize('width', [12344, 14336, 14344, 16384])
def test_wide_rows_at_the_border_of_what_a_thread_holds(rows, width):
    from micro_vllm_b200.row_ops import add_rms_norm_quant, silu_mul_quant
    from tests.w4_reference import as64, assert_quantized
    gen = torch.Generator().manual_seed(59)
    x, r = (torch.randn((rows, width), generator=gen).to(torch.bfloat16) for _ in range(2))
    weight = torch.randn(width, generator=gen).to(torch.bfloat16)
    q, scales, total = add_rms_norm_quant(x.cuda(), r.cuda(), weight.cuda(), 1e-6)
    s = (x.float() + r.float()).to(torch.bfloat16)
    assert torch.equal(total.cpu(), s)
    s64 = as64(s)
    y = as64(weight) * s64 / ((s64 ** 2).mean(-1, keepdims=True) + 1e-6) ** 0.5
    # The sum of squares: a tree of at most width / 32 additions a thread and ten more, each off by half of
    # fp32's step, halved by the root; then a handful of roundings.
    assert_quantized(q, scales, y, torch.int8, (width / 32 / 2 + 16) * 2.0 ** -24)
    g = torch.cat([x, r], dim=-1)
    q, scales = silu_mul_quant(g.cuda())
    g64, u64 = as64(x), as64(r)
    # The exponent's argument (up to 2^3) is off by 2^-24 of itself, exp and division by two units each.
    assert_quantized(q, scales, g64 / (1 + np.exp(-g64)) * u64, torch.int8, 16 * 2.0 ** -23)
