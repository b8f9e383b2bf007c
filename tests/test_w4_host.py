"""CPU checks of the 4-bit weights' layout, quantisation and refusals, and of libmvquant.so's C ABI."""
import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.w4_reference import as64, checkpoint, dense, unpack_records

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / 'include' / 'mvquant.h'


def _library():
    from micro_vllm_b200 import _quant_native, build
    if build.is_stale():
        build.build()
    return _quant_native.library()


@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('n,k', [(1, 1), (64, 128), (65, 129), (130, 333)])
def test_records_hold_the_codes_as_the_header_says(group, zeros, n, k):
    from micro_vllm_b200.w4_linear import pack_w4
    scale_dtype = torch.float16 if group == 64 else torch.bfloat16
    codes, scales, zero = checkpoint(n, k, group, zeros, scale_dtype, seed=n + k)
    kept = codes.clone()
    weight = pack_w4(codes, scales, zero, group_size=group)
    assert torch.equal(codes, kept) and weight.shape == (n, k) and weight.scale_dtype == scale_dtype
    got_codes, got_scales, got_zeros = unpack_records(weight)
    assert np.array_equal(got_codes, codes.numpy())
    assert torch.equal(got_scales, scales)
    assert np.array_equal(got_zeros, zero.numpy() if zeros else np.full(scales.shape, 8))
    assert weight.nbytes == -(-n // 64) * -(-k // 128) * (4096 + 128 // group * (192 if zeros else 128))
    assert weight.to('cpu') is weight and 'group_size' in repr(weight)


@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_rounds_to_the_nearest_code(zeros, dtype):
    """Every value is within half a step of its weight (with the scale's own rounding, at the range's ends)."""
    from micro_vllm_b200.w4_linear import quantize_w4
    gen = torch.Generator().manual_seed(3)
    w = (torch.randn((70, 300), generator=gen) + (0.5 if zeros else 0.0)).to(dtype)
    w[3, 64:128] = 0
    weight = quantize_w4(w, group_size=64, zeros=zeros)
    codes, scales, zero = unpack_records(weight)
    codes = torch.from_numpy(codes)
    got = dense(codes, scales, torch.from_numpy(zero), 64)
    step = as64(scales)[:, np.arange(300) // 64]
    # The scale is rounded by at most 2^-8 (bf16), so the range's ends move by 15 * 2^-8 steps, and the zero
    # point's rounding moves what lies at an end of the range by another half step.
    slack = 0.5 + 15 * 2.0 ** -8 + (0.5 if zeros else 0.0)
    assert (np.abs(got - as64(w)) <= slack * step).all()
    assert not got[3, 64:128].any()
    assert weight.scale_dtype == (torch.float16 if dtype == torch.float32 else dtype)


def test_quantize_of_representable_weights_is_exact():
    from micro_vllm_b200.w4_linear import quantize_w4
    gen = torch.Generator().manual_seed(4)
    codes = torch.randint(-7, 8, (5, 256), generator=gen).float()
    codes[:, ::128] = 7
    weight = quantize_w4(codes * 0.25, scale_dtype=torch.float16)
    got, scales, _ = unpack_records(weight)
    assert np.array_equal(got.astype(np.int64) - 8, codes.numpy().astype(np.int64)) and (scales == 0.25).all()


def test_refusals_of_packing():
    from micro_vllm_b200.w4_linear import pack_w4, quantize_w4, w4_dequantize, w4_linear
    codes, scales, zeros = checkpoint(8, 128, 64, True, torch.float16, 0)
    for call, message in [
        (lambda: pack_w4(codes, scales, group_size=48), 'group_size'),
        (lambda: pack_w4(codes.int(), scales, group_size=64), 'uint8'),
        (lambda: pack_w4(codes[0], scales, group_size=64), 'N, K'),
        (lambda: pack_w4(codes[:0], scales[:0], group_size=64), 'nonempty'),
        (lambda: pack_w4(codes, scales[:, :1], group_size=64), 'scales'),
        (lambda: pack_w4(codes, scales.float(), group_size=64), 'scales'),
        (lambda: pack_w4(codes + 1, scales, group_size=64), '0..15'),
        (lambda: pack_w4(codes, scales, zeros[:, :1], group_size=64), 'zeros'),
        (lambda: pack_w4(codes, scales, zeros + 16, group_size=64), '0..15'),
        (lambda: quantize_w4(torch.full((2, 32), float('inf'))), 'finite'),
        (lambda: quantize_w4(torch.full((2, 32), 1e30), scale_dtype=torch.float16), 'overflow'),
        (lambda: quantize_w4(torch.zeros((2, 32), dtype=torch.int32)), 'float'),
        (lambda: quantize_w4(torch.zeros((2, 32)), scale_dtype=torch.float32), 'scale_dtype'),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
    weight = pack_w4(codes, scales, zeros, group_size=64)
    with pytest.raises(RuntimeError, match='CUDA'):
        w4_linear(torch.zeros((1, 128)), weight)
    with pytest.raises(RuntimeError, match='CUDA'):
        w4_dequantize(weight)


def declared_functions():
    return re.findall(r'^MVQ_API\s+[\w\s\*]+?\b(mvq_\w+)\s*\(', HEADER.read_text(), flags=re.MULTILINE)


def test_header_library_and_binding_agree():
    from micro_vllm_b200 import _quant_native
    lib = _library()
    assert set(declared_functions()) == set(_quant_native.EXPORTED_SYMBOLS)
    out = subprocess.run(['nm', '-D', '--defined-only', str(_quant_native.LIB_PATH)], capture_output=True, text=True,
                         check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if ' T ' in line}
    assert {name for name in exported if name.startswith('mv')} == set(declared_functions())
    constants = {name: int(value) for name, value in
                 re.findall(r'^#define\s+(MVQ_[A-Z0-9_]+)\s+(\d+)\b', HEADER.read_text(), flags=re.MULTILINE)}
    assert lib.mvq_abi_version() == constants['MVQ_ABI_VERSION'] == _quant_native.MVQ_ABI_VERSION
    for name in ('F32', 'F16', 'BF16', 'I8', 'E4M3'):
        assert constants[f'MVQ_DTYPE_{name}'] == getattr(_quant_native, f'DTYPE_{name}')


@pytest.mark.parametrize('struct,fields', [('MvqLinearArgs', 'LINEAR_FIELDS'), ('MvqNormArgs', 'NORM_FIELDS'),
                                           ('MvqDequantizeArgs', 'DEQUANTIZE_FIELDS'), ('MvqSiluArgs', 'SILU_FIELDS')])
def test_argument_structs_match_the_header(struct, fields):
    from micro_vllm_b200 import _quant_native
    body = re.search(r'typedef struct %s \{(.*?)\} %s;' % (struct, struct), HEADER.read_text(), re.S).group(1)
    declared = [re.findall(r'(\w+)\s*$', d.strip())[0] for d in body.replace('\n', ' ').split(';') if d.strip()]
    kinds = [d.strip().split()[0] for d in body.replace('\n', ' ').split(';') if d.strip()]
    assert declared == list(getattr(_quant_native, fields))
    assert all((kind == 'double') == (name == 'eps') for kind, name in zip(kinds, declared))


def test_argument_errors_are_reported_without_a_gpu():
    from micro_vllm_b200 import _native, _quant_native as q
    lib = _library()

    def linear(**changes):
        values = dict(x=64, x_stride_row=128, x_scale=0, records=64, n=64, k=128, group=128, has_zeros=0,
                      scale_dtype=q.DTYPE_BF16, bias=0, residual=0, residual_stride_row=0, out=64, out_stride_row=64,
                      m=2, x_dtype=q.DTYPE_BF16, out_dtype=q.DTYPE_BF16)
        values.update(changes)
        return lib.mvq_w4_linear(q.pack_linear(*(values[f] for f in q.LINEAR_FIELDS)), None)

    for changes, message in [
        (dict(records=0), 'NULL'), (dict(records=72), 'aligned'), (dict(n=0), 'positive'), (dict(k=-1), 'positive'),
        (dict(k=1 << 31), '2\\^30'), (dict(group=16), 'group'), (dict(scale_dtype=0), 'scale_dtype'),
        (dict(x=0), 'NULL'), (dict(out=0), 'NULL'), (dict(m=0), 'positive'), (dict(x_dtype=9), 'x_dtype'),
        (dict(out_dtype=q.DTYPE_I8), 'out_dtype'), (dict(out_stride_row=63), 'stride'), (dict(x_stride_row=-1), 'stride'),
    ]:
        with pytest.raises(_native.NativeError, match=message):
            q.check(linear(**changes))
    assert lib.mvq_w4_linear(None, None) == 1 and b'NULL' in lib.mvq_last_error()
    norm = dict(x=64, x_stride_row=8, residual=0, residual_stride_row=0, weight=64, out=64, out_stride_row=8, scales=0,
                residual_out=0, residual_out_stride_row=0, rows=2, hidden=8, eps=1e-6, dtype=2, out_dtype=2)
    for changes, message in [(dict(eps=float('nan')), 'eps'), (dict(eps=float('inf')), 'eps'), (dict(scales=64), 'scales'),
                             (dict(out_dtype=3), 'scales'), (dict(out_dtype=1), 'out_dtype'), (dict(rows=0), 'positive'),
                             (dict(hidden=0), 'positive'), (dict(weight=0), 'NULL'), (dict(dtype=3), 'dtype'),
                             (dict(out_stride_row=7), 'overlap')]:
        with pytest.raises(_native.NativeError, match=message):
            q.check(lib.mvq_add_rms_norm(q.pack_norm(*({**norm, **changes}[f] for f in q.NORM_FIELDS)), None))
    silu = dict(gate_up=64, stride_row=16, out=64, out_stride_row=8, scales=64, rows=2, width=8, dtype=2, out_dtype=3)
    for changes, message in [(dict(out_dtype=2), 'out_dtype'), (dict(scales=0), 'NULL'), (dict(out_stride_row=1), 'overlap')]:
        with pytest.raises(_native.NativeError, match=message):
            q.check(lib.mvq_silu_mul_quant(q.pack_silu(*({**silu, **changes}[f] for f in q.SILU_FIELDS)), None))
    deq = dict(records=64, n=64, k=128, group=32, has_zeros=0, scale_dtype=1, out=64, out_stride_row=128, out_dtype=0)
    for changes, message in [(dict(out_dtype=4), 'out_dtype'), (dict(out=0), 'NULL'), (dict(out_stride_row=9), 'overlap')]:
        with pytest.raises(_native.NativeError, match=message):
            q.check(lib.mvq_w4_dequantize(q.pack_dequantize(*({**deq, **changes}[f] for f in q.DEQUANTIZE_FIELDS)), None))


def test_import_loads_no_native_code_and_a_missing_library_fails_loudly(tmp_path, monkeypatch):
    import sys
    code = ('import sys; sys.path.insert(0, "micro-vllm_b200"); '
            'from micro_vllm_b200 import w4_linear, row_ops, _quant_native; '
            'assert _quant_native.library.cache_info().currsize == 0')
    run = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
    from micro_vllm_b200 import _quant_native
    monkeypatch.setattr(_quant_native, 'LIB_PATH', tmp_path / 'absent.so')
    _quant_native.library.cache_clear()
    try:
        with pytest.raises(RuntimeError, match='not built'):
            _quant_native.library()
    finally:
        _quant_native.library.cache_clear()


def test_copies_of_a_weight_point_at_their_own_records():
    import copy
    import pickle

    from micro_vllm_b200.w4_linear import pack_w4
    codes, scales, zero = checkpoint(70, 130, 64, True, torch.float16, seed=3)
    weight = pack_w4(codes, scales, zero, group_size=64)
    for other in (copy.copy(weight), copy.deepcopy(weight), pickle.loads(pickle.dumps(weight))):
        assert torch.equal(other.records, weight.records) and repr(other) == repr(weight)
        assert other.fixed == (other.records.data_ptr(), *weight.fixed[1:]) and other.index == weight.index
    assert copy.deepcopy(weight).fixed[0] != weight.fixed[0]


def test_checkpoints_may_be_strided():
    from micro_vllm_b200.w4_linear import pack_w4, quantize_w4
    codes, scales, _ = checkpoint(128, 256, 64, False, torch.float16, seed=4)
    kept = codes.clone()
    records = pack_w4(codes, scales, group_size=64).records
    assert torch.equal(codes, kept)
    strided = pack_w4(codes.t().contiguous().t(), scales.t().contiguous().t(), group_size=64)
    assert torch.equal(strided.records, records)
    one = pack_w4(codes[:1].expand(128, 256), scales[:1].expand(128, 4), group_size=64)
    assert torch.equal(one.records, pack_w4(codes[:1].repeat(128, 1), scales[:1].repeat(128, 1), group_size=64).records)
    matrix = torch.randn((128, 256), generator=torch.Generator().manual_seed(5))
    assert torch.equal(quantize_w4(matrix.t().contiguous().t()).records, quantize_w4(matrix).records)


def test_pointers_off_their_elements_are_refused_without_a_gpu():
    from micro_vllm_b200 import _native, _quant_native as q
    lib = _library()
    linear = dict(x=64, x_stride_row=128, x_scale=0, records=64, n=64, k=128, group=128, has_zeros=0,
                  scale_dtype=q.DTYPE_BF16, bias=0, residual=0, residual_stride_row=0, out=64, out_stride_row=64, m=2,
                  x_dtype=q.DTYPE_BF16, out_dtype=q.DTYPE_F32)
    norm = dict(x=64, x_stride_row=8, residual=0, residual_stride_row=0, weight=64, out=64, out_stride_row=8, scales=64,
                residual_out=0, residual_out_stride_row=0, rows=2, hidden=8, eps=1e-6, dtype=2, out_dtype=3)
    silu = dict(gate_up=64, stride_row=16, out=64, out_stride_row=8, scales=64, rows=2, width=8, dtype=0, out_dtype=3)
    deq = dict(records=64, n=64, k=128, group=32, has_zeros=0, scale_dtype=1, out=64, out_stride_row=128, out_dtype=0)
    for entry, pack, names, good, bad in [
        (lib.mvq_w4_linear, q.pack_linear, q.LINEAR_FIELDS, linear,
         dict(x=65, x_scale=66, bias=66, residual=66, out=66)),
        (lib.mvq_add_rms_norm, q.pack_norm, q.NORM_FIELDS, norm, dict(x=65, residual=65, weight=65, scales=66)),
        (lib.mvq_silu_mul_quant, q.pack_silu, q.SILU_FIELDS, silu, dict(gate_up=66, scales=66)),
        (lib.mvq_w4_dequantize, q.pack_dequantize, q.DEQUANTIZE_FIELDS, deq, dict(out=66)),
    ]:
        for name, value in bad.items():
            with pytest.raises(_native.NativeError, match='aligned to their elements'):
                q.check(entry(pack(*({**good, name: value}[f] for f in names)), None))
