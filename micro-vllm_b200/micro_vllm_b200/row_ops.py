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


_strided = torch.strided
_grad_enabled = torch.is_grad_enabled


def _input_rows(t, shape, dtype, index, name):
    """Row stride of an input [..., width] of this shape, dtype and device, seen as [rows, width]."""
    if not (t.is_cuda and t.get_device() == index and t.dtype is dtype and t.shape == shape and t.layout is _strided
            and not t.is_neg()):
        _check(False, f'{name} must match the input: a strided CUDA tensor of its shape, dtype and device')
    if t.requires_grad and _grad_enabled():
        _check(False, 'row operations do not support gradients')
    if t.is_contiguous():
        return shape[-1]
    if len(shape) == 2:
        row, feature = t.stride()
        _check(feature == 1 or shape[1] == 1, f'{name} requires feature stride 1')
        _check(shape[0] <= 1 or row >= shape[1], f'rows of {name} must not overlap')
        return row
    return _check(False, f'{name}: tensors other than [rows, width] must be contiguous')


def _fresh(like, shape, dtype):
    """An uninitialised contiguous tensor (`like`, where it has the shape, is the cheaper way to say so)."""
    if like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)
    return torch.empty(shape, dtype=dtype, device=like.device)


def _fresh_scales(shape, device):
    if len(shape) == 2:
        return torch.empty(shape[0], dtype=torch.float32, device=device)
    return torch.empty(shape[:-1], dtype=torch.float32, device=device)


def _check_scales(scales, shape, index):
    _check(scales.is_cuda and scales.shape == shape and scales.dtype == torch.float32 and scales.is_contiguous()
           and scales.get_device() == index and not (scales.requires_grad and _grad_enabled()),
           'scales must be contiguous float32, one per row, on the device of the input')


def _disjoint(out, others, same=()):
    """An output may be one of ``same`` exactly, and may share no memory with anything else."""
    for other in others:
        if other is None or not storage_overlaps(out, other):
            continue
        # Strides count elements: at another element size, rows of the same strides lie over other rows.
        exact = any(other is t for t in same) and out.dtype is other.dtype and out.data_ptr() == other.data_ptr() and (
            out.stride() == other.stride() or out.numel() <= out.shape[-1])
        _check(exact, 'an output must be the input itself or share no memory with it')


def _launch(entry, packed, index):
    """Enqueue on the current stream of device `index`, with that device current."""
    if torch.cuda.current_device() == index:
        status = entry(packed, current_stream_raw(index))
    else:
        with torch.cuda.device(index):
            status = entry(packed, current_stream_raw(index))
    if status:
        _quant_native.check(status)


def _add_rms_norm(x, residual, weight, eps, out, out_dtype, scales, residual_out):
    """What the binding's ``norm`` does, for every call: all is checked, and refused with its reason, here."""
    if x.is_cuda:
        _quant_native.refuse_transforms(x, residual, weight, out, scales, residual_out)
    dtype, shape = x.dtype, x.shape
    code = DTYPE_CODES.get(dtype)
    _check(x.is_cuda and code is not None and shape, 'row operations take CUDA float tensors')
    index, device, hidden = x.get_device(), x.device, shape[-1]
    _check(hidden > 0, 'rows must not be empty')
    x_stride = _input_rows(x, shape, dtype, index, 'x')
    if weight.shape != (hidden,) or weight.dtype is not dtype or not weight.is_contiguous() or \
            weight.get_device() != index:
        _check(False, 'weight must be a contiguous [hidden] tensor of the input dtype')
    _check(not (weight.requires_grad and _grad_enabled()), 'row operations do not support gradients')
    residual_at = residual_stride = sum_at = sum_stride = scales_at = 0
    given_out, given_sum = out is not None, residual_out is not None
    if residual is not None:
        residual_stride = _input_rows(residual, shape, dtype, index, 'residual')
        residual_at = residual.data_ptr()
        if given_sum:
            sum_stride = _input_rows(residual_out, shape, dtype, index, 'residual_out')
            _disjoint(residual_out, (x, residual, weight), same=(x, residual))
        else:
            residual_out, sum_stride = _fresh(x, shape, dtype), hidden
        sum_at = residual_out.data_ptr()
    else:
        _check(not given_sum, 'residual_out needs a residual')
        residual_out = x
    if given_out:
        out_stride = _input_rows(out, shape, out_dtype, index, 'out')
        _disjoint(out, (x, residual, weight, residual_out if residual is not None else None),
                  same=(x,) if residual is None or residual_out is not x else ())
    else:
        out, out_stride = _fresh(x, shape, out_dtype), hidden
    out_code = QUANT_CODES.get(out_dtype)
    if out_code is None:
        out_code = code
    elif scales is None:
        scales = _fresh_scales(shape, device)
        scales_at = scales.data_ptr()
    else:
        _check_scales(scales, shape[:-1], index)
        _disjoint(scales, (x, residual, weight, out, residual_out))
        scales_at = scales.data_ptr()
    rows = x.numel() // hidden
    if rows:
        _launch(_quant_native.library().mvq_add_rms_norm, _quant_native.pack_norm(
            x.data_ptr(), x_stride, residual_at, residual_stride, weight.data_ptr(), out.data_ptr(), out_stride,
            scales_at, sum_at, sum_stride, rows, hidden, eps, code, out_code), index)
    return out, scales, residual_out


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                 out: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """s = x + residual (in x's dtype); (weight * s * rsqrt(mean(s^2, -1) + eps), s), over the last dimension.

    fp32 statistics, the norm rounded once (``rms_norm`` rounds the normalised value
    before the scale too, as the reference does). residual_out may be x or residual,
    out may be x.
    """
    _check(residual is not None, 'add_rms_norm needs a residual')
    if out is None and residual_out is None and x.is_cuda:
        found = _quant_native.binding().norm(x, residual, weight, eps, x.dtype)
        if found is not None:
            return found[0], found[2]
    out, _, total = _add_rms_norm(x, residual, weight, eps, out, x.dtype, None, residual_out)
    return out, total


def add_rms_norm_quant(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                       quant_dtype: torch.dtype = torch.int8, out: torch.Tensor | None = None,
                       scales: torch.Tensor | None = None, residual_out: torch.Tensor | None = None):
    """``add_rms_norm`` with its norm y in 8 bits: (q, scales, s).

    scales [...] fp32 = max|y| / 127 (int8) or / 448 (float8_e4m3fn) over each row,
    q = round(y / scale), ties to even; a row of zeros has scale 0 and zeros, a row with a NaN
    or an infinity a NaN scale and zeros. residual None: s is x itself, which is not copied.
    out shares no memory with an input.
    """
    _check(quant_dtype in QUANT_CODES, 'quant_dtype must be int8 or float8_e4m3fn')
    if out is None and scales is None and residual_out is None and x.is_cuda:
        found = _quant_native.binding().norm(x, residual, weight, eps, quant_dtype)
        if found is not None:
            return found
    return _add_rms_norm(x, residual, weight, eps, out, quant_dtype, scales, residual_out)


def silu_mul_quant(gate_up: torch.Tensor, *, quant_dtype: torch.dtype = torch.int8, out: torch.Tensor | None = None,
                   scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """silu(g) * u in 8 bits, the last dimension split as [g | u]: (q, scales) as in ``add_rms_norm_quant``.

    The product stays in fp32 until its one rounding (``silu_mul`` rounds each step): off by a few
    2^-24 of itself and, for gates below zero, by |g| 2^-24. Below -88.72, where fp32 does not hold
    exp(-g), a value is zero.
    """
    out_code = QUANT_CODES.get(quant_dtype)
    _check(out_code is not None, 'quant_dtype must be int8 or float8_e4m3fn')
    if out is None and scales is None and gate_up.is_cuda:
        found = _quant_native.binding().silu(gate_up, quant_dtype)
        if found is not None:
            return found
    if gate_up.is_cuda:
        _quant_native.refuse_transforms(gate_up, out, scales)
    dtype, shape = gate_up.dtype, gate_up.shape
    code = DTYPE_CODES.get(dtype)
    _check(gate_up.is_cuda and code is not None and shape, 'row operations take CUDA float tensors')
    index, device, width = gate_up.get_device(), gate_up.device, shape[-1] // 2
    _check(shape[-1] % 2 == 0 and width > 0, 'the last dimension must hold gate and up halves')
    stride = _input_rows(gate_up, shape, dtype, index, 'gate_up')
    out_shape = shape[:-1] + (width,)
    if out is None:
        out = (torch.empty(shape[0], width, dtype=quant_dtype, device=device) if len(shape) == 2
               else torch.empty(out_shape, dtype=quant_dtype, device=device))
        out_stride = width
    else:
        out_stride = _input_rows(out, out_shape, quant_dtype, index, 'out')
        _disjoint(out, (gate_up,))
    if scales is None:
        scales = _fresh_scales(shape, device)
    else:
        _check_scales(scales, shape[:-1], index)
        _disjoint(scales, (gate_up, out))
    rows = gate_up.numel() // (2 * width)
    if rows:
        _launch(_quant_native.library().mvq_silu_mul_quant, _quant_native.pack_silu(
            gate_up.data_ptr(), stride, out.data_ptr(), out_stride, scales.data_ptr(), rows, width, code, out_code), index)
    return out, scales
