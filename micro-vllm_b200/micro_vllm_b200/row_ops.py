"""Fused row operations of the batched runtime's decode step (libmvdecode.so).

``rms_norm`` is the reference's RMSNorm (src/micro_vllm/model.py:25-41: fp32
statistics, normalised values cast back, then the scale) as one kernel per
call instead of a chain of elementwise launches; ``silu_mul`` is
``F.silu(gate) * up`` (model.py:150-165) on one fused gate/up projection
output, rounded step by step as the reference expression is.

``add_rms_norm`` adds the residual first and returns both the norm and the sum
(the residual stream); ``add_rms_norm_quant`` and ``silu_mul_quant`` end in 8
bits with one fp32 scale per row, the input of ``w4_linear`` (libmvquant.so).
"""
import torch

from . import _native, _quant_native
from ._tensors import DTYPE_CODES, current_stream_raw, storage_overlaps

QUANT_CODES = {torch.int8: _quant_native.DTYPE_I8, torch.float8_e4m3fn: _quant_native.DTYPE_E4M3}


def _check(condition, message):
    if not condition:
        raise RuntimeError(message)


def _rows(t):
    _check(t.is_cuda and t.dtype in DTYPE_CODES and t.dim() >= 1 and t.stride(-1) == 1,
           'row operations take CUDA float tensors with feature stride 1')
    _check(t.dim() == 2 or t.is_contiguous(), 'tensors other than [rows, width] must be contiguous')
    flat = t.view(-1, t.shape[-1]) if t.dim() != 2 else t
    _check(flat.dim() == 2 and (flat.shape[0] <= 1 or flat.stride(0) >= flat.shape[1]),
           'rows must not overlap')
    return flat


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """weight * to_dtype(x * rsqrt(mean(x^2, -1) + eps)) over the last dimension."""
    rows = _rows(x)
    _check(weight.shape == (x.shape[-1],) and weight.dtype == x.dtype and weight.is_contiguous()
           and weight.device == x.device, 'weight must be a contiguous [hidden] tensor of the input dtype')
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    o = _rows(out)
    _check(o.shape == rows.shape, 'out must match x')
    _native.check(_native.library().mv_rms_norm(
        rows.data_ptr(), rows.stride(0), weight.data_ptr(), o.data_ptr(), o.stride(0), rows.shape[0],
        rows.shape[1], float(eps), DTYPE_CODES[x.dtype], current_stream_raw(x.device.index)))
    return out


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(g) * u for the last dimension split as [g | u]."""
    rows = _rows(gate_up)
    _check(rows.shape[1] % 2 == 0, 'the last dimension must hold gate and up halves')
    width = rows.shape[1] // 2
    if out is None:
        out = torch.empty(gate_up.shape[:-1] + (width,), dtype=gate_up.dtype, device=gate_up.device)
    o = _rows(out)
    _check(o.shape == (rows.shape[0], width), 'out must be [..., width]')
    _native.check(_native.library().mv_silu_mul(
        rows.data_ptr(), rows.stride(0), o.data_ptr(), o.stride(0), rows.shape[0], width,
        DTYPE_CODES[gate_up.dtype], current_stream_raw(gate_up.device.index)))
    return out


def _no_grad(*tensors):
    _check(not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors),
           'row operations do not support gradients')


def _output_rows(t, shape, dtype, device, name):
    """A given output, checked, as [rows, width]."""
    _check(isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == device,
           f'{name} must have the shape {tuple(shape)}, dtype {dtype} and the device of the input')
    _no_grad(t)
    _check(t.dim() == 2 or t.is_contiguous(), f'{name}: tensors other than [rows, width] must be contiguous')
    flat = t if t.dim() == 2 else t.view(-1, shape[-1])
    _check(shape[-1] == 1 or flat.stride(1) == 1, f'{name} requires feature stride 1')
    _check(flat.shape[0] <= 1 or flat.stride(0) >= shape[-1], f'rows of {name} must not overlap')
    return flat


def _disjoint(out, others, same=()):
    """An output may be one of ``same`` exactly, and may share no memory with anything else."""
    for other in others:
        if other is None or not storage_overlaps(out, other):
            continue
        exact = any(other is t for t in same) and out.data_ptr() == other.data_ptr() and (
            out.stride() == other.stride() or out.numel() <= out.shape[-1])
        _check(exact, 'an output must be the input itself or share no memory with it')


def _launch(entry, packed, index):
    stream = current_stream_raw(index)
    if torch.cuda.current_device() == index:
        return _quant_native.check(entry(packed, stream))
    with torch.cuda.device(index):
        return _quant_native.check(entry(packed, stream))


def _add_rms_norm(x, residual, weight, eps, out, out_dtype, scales, residual_out):
    rows = _rows(x)
    hidden, device = x.shape[-1], x.device
    _check(rows.shape[1] > 0, 'rows must not be empty')
    _check(weight.shape == (hidden,) and weight.dtype == x.dtype and weight.is_contiguous()
           and weight.device == device, 'weight must be a contiguous [hidden] tensor of the input dtype')
    _no_grad(x, residual, weight)
    residual_at = residual_stride = sum_at = sum_stride = scales_at = 0
    if residual is not None:
        _check(residual.shape == x.shape and residual.dtype == x.dtype and residual.device == device,
               'residual must match x')
        flat = _rows(residual)
        residual_at, residual_stride = flat.data_ptr(), flat.stride(0)
        fresh = residual_out is None
        if fresh:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=device)
        flat = _output_rows(residual_out, x.shape, x.dtype, device, 'residual_out')
        if not fresh:
            _disjoint(residual_out, (x, residual, weight), same=(x, residual))
        sum_at, sum_stride = flat.data_ptr(), flat.stride(0)
    else:
        _check(residual_out is None, 'residual_out needs a residual')
    fresh = out is None
    if fresh:
        out = torch.empty(x.shape, dtype=out_dtype, device=device)
    flat = _output_rows(out, x.shape, out_dtype, device, 'out')
    if not fresh:
        _disjoint(out, (x, residual, weight, residual_out), same=(x,) if residual_out is not x else ())
    if out_dtype in QUANT_CODES:
        if scales is None:
            scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
        else:
            _check(scales.shape == x.shape[:-1] and scales.dtype == torch.float32 and scales.is_contiguous()
                   and scales.device == device, 'scales must be contiguous float32, one per row')
            _disjoint(scales, (x, residual, weight, out, residual_out))
        scales_at = scales.data_ptr()
    if rows.shape[0]:
        _launch(_quant_native.library().mvq_add_rms_norm, _quant_native.pack_norm(
            rows.data_ptr(), rows.stride(0), residual_at, residual_stride, weight.data_ptr(), flat.data_ptr(),
            flat.stride(0), scales_at, sum_at, sum_stride, rows.shape[0], hidden, float(eps), DTYPE_CODES[x.dtype],
            QUANT_CODES[out_dtype] if out_dtype in QUANT_CODES else DTYPE_CODES[out_dtype]), device.index)
    return out, scales, x if residual is None else residual_out


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                 out: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """s = x + residual (in x's dtype); (weight * s * rsqrt(mean(s^2, -1) + eps), s), over the last dimension.

    fp32 statistics, the norm rounded once (``rms_norm`` rounds the normalised value
    before the scale too, as the reference does). residual_out may be x or residual,
    out may be x.
    """
    _check(residual is not None, 'add_rms_norm needs a residual')
    out, _, total = _add_rms_norm(x, residual, weight, eps, out, x.dtype, None, residual_out)
    return out, total


def add_rms_norm_quant(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                       quant_dtype: torch.dtype = torch.int8, out: torch.Tensor | None = None,
                       scales: torch.Tensor | None = None, residual_out: torch.Tensor | None = None):
    """``add_rms_norm`` with its norm y in 8 bits: (q, scales, s).

    scales [...] fp32 = max|y| / 127 (int8) or / 448 (float8_e4m3fn) over each row,
    q = round(y / scale); a row of zeros has scale 0 and zeros, a row with a NaN or an
    infinity a NaN scale and zeros. residual None: s is x itself, which is not copied.
    """
    _check(quant_dtype in QUANT_CODES, 'quant_dtype must be int8 or float8_e4m3fn')
    return _add_rms_norm(x, residual, weight, eps, out, quant_dtype, scales, residual_out)


def silu_mul_quant(gate_up: torch.Tensor, *, quant_dtype: torch.dtype = torch.int8, out: torch.Tensor | None = None,
                   scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """silu(g) * u in 8 bits, the last dimension split as [g | u]: (q, scales) as in ``add_rms_norm_quant``.

    The product stays in fp32 until its one rounding (``silu_mul`` rounds each step).
    """
    _check(quant_dtype in QUANT_CODES, 'quant_dtype must be int8 or float8_e4m3fn')
    rows = _rows(gate_up)
    _check(rows.shape[1] % 2 == 0 and rows.shape[1] > 0, 'the last dimension must hold gate and up halves')
    _no_grad(gate_up)
    width, device = rows.shape[1] // 2, gate_up.device
    shape = gate_up.shape[:-1] + (width,)
    fresh = out is None
    if fresh:
        out = torch.empty(shape, dtype=quant_dtype, device=device)
    flat = _output_rows(out, shape, quant_dtype, device, 'out')
    if not fresh:
        _disjoint(out, (gate_up,))
    if scales is None:
        scales = torch.empty(gate_up.shape[:-1], dtype=torch.float32, device=device)
    else:
        _check(scales.shape == gate_up.shape[:-1] and scales.dtype == torch.float32 and scales.is_contiguous()
               and scales.device == device, 'scales must be contiguous float32, one per row')
        _disjoint(scales, (gate_up, out))
    if rows.shape[0]:
        _launch(_quant_native.library().mvq_silu_mul_quant, _quant_native.pack_silu(
            rows.data_ptr(), rows.stride(0), flat.data_ptr(), flat.stride(0), scales.data_ptr(), rows.shape[0], width,
            DTYPE_CODES[gate_up.dtype], QUANT_CODES[quant_dtype]), device.index)
    return out, scales
