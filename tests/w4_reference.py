"""Plain 64-bit forms of the 4-bit and 8-bit operators, for the tests (numpy, CPU)."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def as64(t):
    return None if t is None else t.detach().cpu().to(torch.float64).numpy()


def dense(codes, scales, zeros, group):
    """W in 64 bits from a checkpoint's codes [N, K], scales [N, G] and zero points (None: 8)."""
    codes, scales = as64(codes), as64(scales)
    column = np.arange(codes.shape[1]) // group
    zero = 8.0 if zeros is None else as64(zeros)[:, column]
    return (codes - zero) * scales[:, column]


def checkpoint(n, k, group, with_zeros, scale_dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = (0.02 * (0.5 + torch.rand((n, groups), generator=gen))).to(scale_dtype)
    zeros = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8) if with_zeros else None
    return codes, scales, zeros


def unpack_records(weight):
    """Codes, scales and zero points read back from a W4Weight by include/mvquant.h's description."""
    n, k = weight.shape
    tiles, chunks, groups = -(-n // 64), -(-k // 128), 128 // weight.group_size
    size = 4096 + groups * (192 if weight.has_zeros else 128)
    data = weight.records.cpu().numpy().reshape(-1)
    assert data.size == tiles * chunks * size
    codes = np.full((tiles * 64, chunks * 128), 255, dtype=np.uint8)
    scales = torch.zeros((tiles * 64, chunks * groups), dtype=weight.scale_dtype)
    zeros = np.full((tiles * 64, chunks * groups), 8, dtype=np.int64)
    for i in range(tiles):
        for j in range(chunks):
            record = data[(i * chunks + j) * size:][:size]
            for h in range(4):
                for p in range(2):
                    for lane in range(32):
                        g, t = lane // 4, lane % 4
                        for word in range(4):
                            q, e = word // 2, word % 2
                            at = (((h * 2 + p) * 32 + lane) * 4 + word) * 4
                            for byte, s in enumerate((0, 2, 1, 3)):
                                value = int(record[at + byte])
                                column = j * 128 + 32 * h + 16 * e + 4 * t + s
                                row = i * 64 + 32 * p + 16 * q + g
                                codes[row, column] = (value & 15) ^ 8
                                codes[row + 8, column] = (value >> 4) ^ 8
            for group in range(groups):
                raw = torch.from_numpy(record[4096 + group * 128:][:128].copy()).view(weight.scale_dtype)
                for g in range(8):
                    for rest in range(8):
                        p, q, half = rest // 4, rest // 2 % 2, rest % 2
                        row = i * 64 + 32 * p + 16 * q + 8 * half + g
                        scales[row, j * groups + group] = raw[g * 8 + rest]
                        if weight.has_zeros:
                            byte = record[4096 + groups * 128 + group * 64 + g * 8 + rest]
                            zeros[row, j * groups + group] = int(byte.astype(np.int8)) + 8
    real = -(-k // weight.group_size)
    return codes[:n, :k], scales[:n, :real], zeros[:n, :real]


def quantized(y, quant_dtype):
    """Row scales of y and y / scale in 64 bits (zeros where the scale is zero)."""
    scale = np.abs(y).max(-1) / TOP[quant_dtype]
    with np.errstate(divide='ignore', invalid='ignore'):
        v = np.where(scale[..., None] > 0, y / scale[..., None], 0.0)
    return scale, v


def assert_quantized(q, scale, y, quant_dtype, relative):
    """q and scale against y in 64 bits; `relative`: how far the kernel's fp32 y may be off, of the row's largest."""
    expected, v = quantized(y, quant_dtype)
    np.testing.assert_allclose(as64(scale), expected, rtol=relative, atol=0)
    got = as64(q.float())
    slack = TOP[quant_dtype] * 2 * relative
    if quant_dtype == torch.int8:
        assert (np.abs(got - v) <= 0.5 + slack).all()
    else:  # half a step: 2^-4 of a normal number, 2^-10 below 2^-6; a step's border may be crossed by the slack
        assert (np.abs(got - v) <= np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10) + slack).all()
