"""Linear layers with 4-bit weights and group scales (libmvquant.so).

A ``W4Weight`` holds W [N, K] as 4-bit codes with one scale (and, if asked for,
one zero point) per row and per ``group_size`` columns:

    W[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group]

``quantize_w4`` makes one from a weight matrix, ``pack_w4`` from a checkpoint's
codes; both lay the codes out once in the order the kernels read them.

``w4_linear`` is the layer: x W^T with a few rows of x (a decode step's tokens),
the bias and the residual's addition in the same kernel. x is fp32, fp16 or
bf16, or int8 / e4m3 with a scale for each row (``row_ops.add_rms_norm_quant``
and ``row_ops.silu_mul_quant`` make those). ``w4_dequantize`` writes W out for
products with many rows (a prompt), which are matrix products of the library's.

The reference has no quantised layers: its linear layers are F.linear on the
checkpoint's own weights (src/micro_vllm/model.py:126-165, 189-241).
"""
import torch

from . import _quant_native as _native
from ._tensors import current_stream_raw, storage_overlaps

GROUP_SIZES = (32, 64, 128)
TILE_ROWS, CHUNK = 64, 128

FLOAT_CODES = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16,
               torch.bfloat16: _native.DTYPE_BF16}
ACTIVATION_CODES = {**FLOAT_CODES, torch.int8: _native.DTYPE_I8, torch.float8_e4m3fn: _native.DTYPE_E4M3}
SCALE_CODES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}


def _check(condition, message):
    if not condition:
        raise RuntimeError(message)


class W4Weight:
    """A [N, K] weight in 4-bit codes, laid out for the kernels (include/mvquant.h). Immutable."""

    __slots__ = ('records', 'shape', 'group_size', 'has_zeros', 'scale_dtype', 'index', 'fixed', 'packed')

    def __init__(self, records, shape, group_size, has_zeros, scale_dtype):
        shape = torch.Size(shape)
        _check(len(shape) == 2 and min(shape) > 0, 'shape must be two positive sizes')
        _check(group_size in GROUP_SIZES, 'group_size must be 32, 64 or 128')
        _check(scale_dtype in SCALE_CODES, 'scale_dtype must be float16 or bfloat16')
        _check(records.dtype == torch.uint8 and records.is_contiguous(), 'records must be a contiguous uint8 tensor')
        per_group = 2 * TILE_ROWS + (TILE_ROWS if has_zeros else 0)
        record = TILE_ROWS * CHUNK // 2 + CHUNK // group_size * per_group
        size = -(-shape[0] // TILE_ROWS) * -(-shape[1] // CHUNK) * record
        # The kernels read what the shape says: fewer bytes would be read past their end.
        _check(records.numel() == size, f'records of this weight take {size} bytes')
        self.records = records
        self.shape = shape
        self.group_size = group_size
        self.has_zeros = has_zeros
        self.scale_dtype = scale_dtype
        self.index = records.get_device()  # -1 on the CPU
        # The weight's fields of the calls' argument structs.
        self.fixed = (records.data_ptr(), *self.shape, group_size, int(has_zeros), SCALE_CODES[scale_dtype])
        self.packed = _native.pack_weight(*self.fixed)

    @property
    def device(self):
        return self.records.device

    @property
    def nbytes(self):
        return self.records.numel()

    def __reduce__(self):
        # A copy's addresses are those of its own records.
        return W4Weight, (self.records, self.shape, self.group_size, self.has_zeros, self.scale_dtype)

    def to(self, device):
        """This weight on another device (itself where it is there already)."""
        records = self.records.to(device)
        if records is self.records:
            return self
        return W4Weight(records, self.shape, self.group_size, self.has_zeros, self.scale_dtype)

    def __repr__(self):
        return (f'W4Weight(shape={tuple(self.shape)}, group_size={self.group_size}, zeros={self.has_zeros}, '
                f'scales={self.scale_dtype}, device={self.device})')


@torch.no_grad()
def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
            group_size: int = 128) -> W4Weight:
    """A ``W4Weight`` from codes [N, K] (uint8, 0..15), scales [N, ceil(K / group_size)] (fp16 or bf16)
    and zero points of the scales' shape (uint8, 0..15; without them every zero point is 8).

    The last group of a row may be partial. Values are checked here (reading them
    back once where they live on a GPU). Any device; the kernels need a CUDA one.
    """
    _check(group_size in GROUP_SIZES, 'group_size must be 32, 64 or 128')
    _check(codes.dim() == 2 and codes.numel() > 0 and codes.dtype == torch.uint8,
           'codes must be a nonempty [N, K] uint8 tensor')
    n, k = codes.shape
    groups = (k + group_size - 1) // group_size
    _check(scales.shape == (n, groups) and scales.dtype in SCALE_CODES and scales.device == codes.device,
           'scales must be a [N, ceil(K / group_size)] float16 or bfloat16 tensor on the device of the codes')
    _check(bool(codes.max() <= 15), 'codes must lie in 0..15')
    if zeros is not None:
        _check(zeros.shape == (n, groups) and zeros.dtype == torch.uint8 and zeros.device == codes.device,
               'zeros must be a uint8 tensor of the shape and device of the scales')
        _check(bool(zeros.max() <= 15), 'zeros must lie in 0..15')
    tiles, chunks, per_chunk = -(-n // TILE_ROWS), -(-k // CHUNK), CHUNK // group_size
    pad = torch.nn.functional.pad
    rows = tiles * TILE_ROWS - n
    # [tile, p, q, half, g, chunk, h, e, t, s]: row 32p + 16q + 8half + g, column 32h + 16e + 4t + s. Codes are
    # stored with their highest bit inverted (code - 8 in two's complement); columns beyond K hold code 8.
    c = pad(codes, (0, chunks * CHUNK - k, 0, rows), value=8).bitwise_xor_(8)
    c = c.view(tiles, 2, 2, 2, 8, chunks, 4, 2, 4, 4)
    c = c[:, :, :, 0] | (c[:, :, :, 1] << 4)                # [tile, p, q, g, chunk, h, e, t, s]
    c = c.permute(0, 4, 5, 1, 3, 7, 2, 6, 8)[..., [0, 2, 1, 3]].reshape(tiles, chunks, TILE_ROWS * CHUNK // 2)

    def by_group(values):  # [tile, chunk, bytes of the chunk's groups]
        values = pad(values, (0, chunks * per_chunk - groups, 0, rows))
        values = values.view(tiles, 2, 2, 2, 8, chunks, per_chunk).permute(0, 5, 6, 4, 1, 2, 3).contiguous()
        return values.view(torch.uint8).reshape(tiles, chunks, -1)

    parts = [c, by_group(scales)]
    if zeros is not None:
        parts.append(by_group(zeros.to(torch.int8) - 8))
    return W4Weight(torch.cat(parts, dim=-1), (n, k), group_size, zeros is not None, scales.dtype)


@torch.no_grad()
def quantize_w4(weight: torch.Tensor, *, group_size: int = 128, zeros: bool = False,
                scale_dtype: torch.dtype | None = None) -> W4Weight:
    """Round a float weight [N, K] to 4 bits, group by group.

    Without ``zeros``: scale = max|w| / 7 over the group, codes 1..15 around 8.
    With them: scale = (max - min) / 15 with 0 in the range, zero = round(-min /
    scale). Codes are rounded with the scale as it is stored (``scale_dtype``,
    default the weight's own 16-bit type, else float16); a group whose scale
    rounds to zero holds zeros. Weights must be finite.
    """
    _check(group_size in GROUP_SIZES, 'group_size must be 32, 64 or 128')
    _check(weight.dim() == 2 and weight.numel() > 0 and weight.dtype in FLOAT_CODES,
           'weight must be a nonempty [N, K] float tensor')
    scale_dtype = scale_dtype or (weight.dtype if weight.dtype in SCALE_CODES else torch.float16)
    _check(scale_dtype in SCALE_CODES, 'scale_dtype must be float16 or bfloat16')
    n, k = weight.shape
    groups = (k + group_size - 1) // group_size
    w = torch.nn.functional.pad(weight.float(), (0, groups * group_size - k)).view(n, groups, group_size)
    _check(bool(torch.isfinite(w).all()), 'weights must be finite')
    if zeros:
        low, high = w.amin(-1).clamp_(max=0), w.amax(-1).clamp_(min=0)
        scale = ((high - low) / 15).to(scale_dtype)
    else:
        scale = (w.abs().amax(-1) / 7).to(scale_dtype)
    _check(bool(torch.isfinite(scale).all()), f'a scale overflows {scale_dtype}')
    step = torch.where(scale > 0, scale.float(), torch.inf)
    zero = (-low / step).round_().clamp_(0, 15) if zeros else torch.full_like(step, 8.0)
    least = 0 if zeros else 1
    codes = (w / step.unsqueeze(-1)).round_().add_(zero.unsqueeze(-1)).clamp_(least, 15).to(torch.uint8)
    return pack_w4(codes.view(n, -1)[:, :k].contiguous(), scale, zero.to(torch.uint8) if zeros else None,
                   group_size=group_size)


_strided = torch.strided
_grad_enabled = torch.is_grad_enabled


def _usable(t, index):
    """A strided tensor on CUDA device `index` that asks for no gradient."""
    return (t.is_cuda and t.get_device() == index and t.layout is _strided and not t.is_neg()
            and not (t.requires_grad and _grad_enabled()))


def _refuse(t, name, index):
    _check(t.is_cuda and t.layout is _strided and not t.is_neg(), f'{name} must be a strided CUDA tensor')
    _check(not t.requires_grad or not _grad_enabled(), f'{name}: 4-bit layers do not support gradients')
    _check(t.get_device() == index, f'{name} must be on the device of x')


def _row_stride(t, width, name):
    """Row stride of t [..., width] seen as [rows, width] without copying."""
    if t.is_contiguous():
        return width
    _check(t.dim() == 2, f'{name}: tensors other than [rows, width] must be contiguous')
    row, feature = t.stride()
    _check(feature == 1 or width == 1, f'{name} requires feature stride 1')
    return row


def _launch(entry, packed, index):
    """Enqueue on the current stream of device `index`, with that device current."""
    if torch.cuda.current_device() == index:
        status = entry(packed, current_stream_raw(index))
    else:
        with torch.cuda.device(index):
            status = entry(packed, current_stream_raw(index))
    if status:
        _native.check(status)


def w4_linear(x: torch.Tensor, weight: W4Weight, bias: torch.Tensor | None = None,
              residual: torch.Tensor | None = None, *, x_scale: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x W^T (times ``x_scale`` per row) + bias + residual, over the last dimension of x.

    x: [..., K] fp32, fp16 or bf16, or int8 / float8_e4m3fn with ``x_scale``
    (fp32, one per row); rows of a 2-D x may be strided. The sums are fp32 (32-bit
    integers within a group for int8) and rounded once, to ``out_dtype``: the
    type of ``out`` or of the residual or bias, else x's own; 8-bit x needs one
    of these. bias [N] and residual [..., N] have that type; out may be residual.
    Any number of rows; made for a decode step's (up to 128). Runs on the current stream.
    """
    if out is None and x.is_cuda:
        y = _native.binding().linear(x, weight.packed, weight.index, bias, residual, x_scale, out_dtype)
        if y is not None:
            return y
    # Not the usual call: everything is checked, and refused with its reason, here.
    if x.is_cuda:
        _native.refuse_transforms(x, bias, residual, x_scale, out)
    n, k = weight.shape
    x_dtype = x.dtype
    code = ACTIVATION_CODES.get(x_dtype)
    _check(code is not None, 'x must be float32, float16, bfloat16, int8 or float8_e4m3fn')
    index = x.get_device()
    if not _usable(x, index):
        _refuse(x, 'x', index)
    if weight.index != index:
        _check(False, 'the weight must be on the device of x')
    x_shape = x.shape
    if not x_shape or x_shape[-1] != k:
        _check(False, f'x must have {k} features')
    x_stride = _row_stride(x, k, 'x')
    if len(x_shape) == 2:
        m = x_shape[0]
        shape = (m, n)
    else:
        shape = x_shape[:-1] + (n,)
        m = x.numel() // k
    if out_dtype is None:
        given = out if out is not None else residual if residual is not None else bias
        _check(given is not None or code <= 2, '8-bit x needs out_dtype, out, residual or bias')
        out_dtype = x_dtype if given is None else given.dtype
    out_code = FLOAT_CODES.get(out_dtype)
    _check(out_code is not None, 'out_dtype must be float32, float16 or bfloat16')
    scale_at = bias_at = residual_at = residual_stride = 0
    if x_scale is not None:
        if not _usable(x_scale, index):
            _refuse(x_scale, 'x_scale', index)
        if x_scale.dtype is not torch.float32 or x_scale.numel() != m or not x_scale.is_contiguous():
            _check(False, 'x_scale must be contiguous float32, one per row')
        scale_at = x_scale.data_ptr()
    elif code > 2:
        _check(False, '8-bit x needs x_scale')
    if bias is not None:
        if not _usable(bias, index):
            _refuse(bias, 'bias', index)
        if bias.dtype is not out_dtype or bias.shape != (n,) or not bias.is_contiguous():
            _check(False, 'bias must be a contiguous [N] tensor of out_dtype')
        bias_at = bias.data_ptr()
    if residual is not None:
        if not _usable(residual, index):
            _refuse(residual, 'residual', index)
        if residual.dtype is not out_dtype or residual.shape != shape:
            _check(False, 'residual must be a [..., N] tensor of out_dtype')
        residual_stride = _row_stride(residual, n, 'residual')
        residual_at = residual.data_ptr()
    if out is None:
        # Shapes given as separate numbers cost torch the least host time.
        out = torch.empty(*shape, dtype=out_dtype, device=x.device)
        out_at, out_stride = out.data_ptr(), n
    else:
        if not _usable(out, index):
            _refuse(out, 'out', index)
        _check(out.shape == shape and out.dtype is out_dtype, 'out must be a [..., N] tensor of out_dtype')
        out_at, out_stride = out.data_ptr(), _row_stride(out, n, 'out')
        _check(m <= 1 or out_stride >= n, 'rows of out must not overlap')
        for other in (x, x_scale, bias, weight.records):
            _check(other is None or not storage_overlaps(out, other), 'out must not alias an input')
        _check(residual is None or (out_at == residual_at and (m <= 1 or out_stride == residual_stride))
               or not storage_overlaps(out, residual), 'out must be the residual itself or not alias it')
    if m:
        _launch(_native.library().mvq_w4_linear, _native.pack_linear(
            x.data_ptr(), x_stride, scale_at, *weight.fixed, bias_at, residual_at, residual_stride, out_at, out_stride,
            m, code, out_code), index)
    return out


def w4_dequantize(weight: W4Weight, dtype: torch.dtype | None = None, *,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """W [N, K] written out in ``dtype`` (default: the scales'), each value rounded once.

    out: an [N, K] tensor of ``dtype``, rows may be strided. Runs on the current stream.
    """
    n, k = weight.shape
    index = weight.index
    _check(index >= 0, 'the weight must be on a CUDA device')
    dtype = dtype or (out.dtype if out is not None else weight.scale_dtype)
    if out is None:
        out = _native.binding().dequantize(weight.packed, weight.records, dtype)
        if out is not None:
            return out
    _native.refuse_transforms(weight.records, out)
    code = FLOAT_CODES.get(dtype)
    _check(code is not None, 'dtype must be float32, float16 or bfloat16')
    if out is None:
        out = torch.empty(n, k, dtype=dtype, device=weight.device)
    else:
        if not _usable(out, index):
            _refuse(out, 'out', index)
        _check(out.shape == (n, k) and out.dtype == dtype and (k == 1 or out.stride(1) == 1)
               and (n == 1 or out.stride(0) >= k), 'out must be an [N, K] tensor of dtype with feature stride 1')
        _check(not storage_overlaps(out, weight.records), 'out must not alias the weight')
    _launch(_native.library().mvq_w4_dequantize, _native.pack_dequantize(
        *weight.fixed, out.data_ptr(), out.stride(0), code), index)
    return out
