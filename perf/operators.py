"""The 4-bit decode step's operators, measured: each as plain torch operations and as the framework's kernels.

Operators: ``w4_linear`` (a row batch against 4-bit weights with group scales; activations in 16 or 32 bits,
or in 8 bits with a scale for each row), ``w4_dequantize`` (the same weights written out, for long prompts),
``add_rms_norm`` / ``add_rms_norm_quant`` (the residual's addition and the root-mean-square norm, the
output in the model's type or in 8 bits with a scale for each row) and ``silu_mul_quant`` (the gated
activation in 8 bits).  The two chains run them as a decode step does: norm, then the projection it feeds.

Formulas.  Weights: W[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group], code and zero in
0..15 (zero 8 where there are none).  Linear: y = x W^T * x_scale + bias + residual.  Norm: s = round(x +
residual), y = w * s * rsqrt(mean(s^2) + eps).  Gate: y = g / (1 + exp(-g)) * u.  8 bits: scale = max|y| / top
over the row (top: 127 for int8, 448 for e4m3), the value round(y / scale).

Hidden sizes 896, 1536, 3584 and 8192 and the projections' widths follow from the head counts and widths that
the benchmark runs (14/2 heads of 64; 12/2, 28/4 and 64/8 heads of 128); widths of feed-forward layers that
it does not give are four times the hidden size, or 28672.
"""
import math

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32,
         'int8': torch.int8, 'e4m3': torch.float8_e4m3fn}
TOP = {'int8': 127.0, 'e4m3': 448.0}
EPS = 1e-6


def _linear(name, m, k, n, x, out, group=128, zeros=False, bias=False, residual=False):
    return {'name': name, 'op': 'linear', 'm': m, 'k': k, 'n': n, 'x': x, 'out': out, 'group': group,
            'zeros': zeros, 'bias': bias, 'residual': residual}


def _chain(name, op, m, k, n, x, out, group=128, zeros=False, bias=False, residual=False):
    return dict(_linear(name, m, k, n, x, out, group, zeros, bias, residual), op=op)


def _rows(name, op, m, k, x, out):
    return {'name': name, 'op': op, 'm': m, 'k': k, 'x': x, 'out': out}


def _dequant(name, k, n, out, group=128, zeros=False):
    return {'name': name, 'op': 'dequant', 'k': k, 'n': n, 'out': out, 'group': group, 'zeros': zeros}


def listed():
    return [
        # Q/K/V projection of the smallest model for one sequence: all latency.
        _linear('qkv_1_bf16', 1, 896, 1152, 'bf16', 'bf16', bias=True),
        # Gate/up projection of one sequence's token: the stream of the weights.
        _linear('gate_up_1_bf16', 1, 3584, 28672, 'bf16', 'bf16'),
        # Odd sizes in 32 bits with zero points and small groups: a checked or truncated model.
        _linear('ragged_5_fp32', 5, 1499, 2047, 'fp32', 'fp32', group=32, zeros=True, bias=True),
        # Down projection with the residual's addition for a batch of 64 sequences, a checkpoint with zero points.
        _linear('down_64_fp16', 64, 14336, 3584, 'fp16', 'fp16', group=64, zeros=True, residual=True),
        # Gate/up projection of the largest model with 8-bit activations, 16 sequences: the largest stream.
        _linear('gate_up_16_int8', 16, 8192, 57344, 'int8', 'bf16'),
        # The norm before a projection for one sequence: all latency.
        _rows('norm_1_e4m3', 'norm', 1, 3584, 'bf16', 'e4m3'),
        # The same for a prompt of 8192 tokens.
        _rows('norm_8192_e4m3', 'norm', 8192, 3584, 'bf16', 'e4m3'),
        # Norm into 8 bits, then the Q/K/V projection of 8 sequences: half of what a layer does before attention.
        _chain('norm_qkv_8_int8', 'norm_linear', 8, 3584, 4608, 'bf16', 'bf16', bias=True),
        # The gated activation of a prompt of 2048 tokens.
        _rows('silu_2048_e4m3', 'silu', 2048, 14336, 'bf16', 'e4m3'),
        # The gated activation into 8 bits, then the down projection: the end of a layer for 32 sequences.
        _chain('mlp_tail_32_int8', 'silu_linear', 32, 8960, 1536, 'bf16', 'bf16', residual=True),
        # Weights of a gate/up projection written out for a prompt's matrix product.
        _dequant('dequant_3584_bf16', 3584, 28672, 'bf16'),
        # A small projection's, with zero points.
        _dequant('dequant_896_fp16', 896, 1152, 'fp16', group=64, zeros=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A size of the range: a multiple of 128 in half of the cases, of 8 in a quarter, any in the rest."""
    step = rng.choice((128, 128, 8, 1))
    return max(low, _log(rng, low, high) // step * step)


def draw(rng):
    op = rng.choice(('linear', 'linear', 'linear', 'norm', 'silu', 'norm_linear', 'silu_linear', 'dequant'))
    if op in ('norm', 'silu'):
        k = _width(rng, 64, 16384)
        m = _log(rng, 1, max(1, min(8192, (8192 * 3584) // k)))
        x = rng.choice(('bf16', 'fp16', 'fp32'))
        return {'op': op, 'm': m, 'k': k, 'x': x, 'out': rng.choice(('e4m3', x)) if op == 'norm' else 'e4m3'}
    k = _width(rng, 64, 16384)
    n = _width(rng, 16, max(16, min(57344, 200_000_000 // k)))
    case = {'op': op, 'k': k, 'n': n, 'group': rng.choice((32, 64, 128)), 'zeros': rng.random() < 0.5}
    if op == 'dequant':
        case['n'] = min(n, 100_000_000 // k)
        case['out'] = rng.choice(('bf16', 'fp16', 'fp32'))
        return case
    m = _log(rng, 1, max(1, min(256, 7_000_000_000 // (n * k))))
    out = rng.choice(('bf16', 'fp16'))
    x = rng.choice(('bf16', 'fp16', 'fp32', 'int8', 'e4m3')) if op == 'linear' else out
    return dict(case, m=m, x=x, out=x if x in ('bf16', 'fp16', 'fp32') else out,
                bias=rng.random() < 0.4, residual=rng.random() < 0.4)


def _weights(case, gen, state):
    """A 4-bit checkpoint's codes (two to a byte, the lower column in the low half), scales and zero points."""
    n, k, group = case['n'], case['k'], case['group']
    groups = -(-k // group)
    kind = torch.float16 if case['out'] in ('fp16', 'fp32') else torch.bfloat16
    codes = torch.empty((n, k), dtype=torch.uint8, device='cuda')
    for at in range(0, n, 8192):
        rows = torch.randn((min(8192, n - at), k), generator=gen, device='cuda')
        codes[at:at + 8192] = rows.mul_(2.6).add_(8).round_().clamp_(0, 15).to(torch.uint8)
    scales = ((0.5 + torch.rand((n, groups), generator=gen, device='cuda')) * (0.4 / math.sqrt(k))).to(kind)
    zeros = (torch.randint(5, 11, (n, groups), generator=gen, device='cuda', dtype=torch.uint8)
             if case['zeros'] else None)
    if own:
        from micro_vllm_b200.w4_linear import pack_w4
        state['weight'] = pack_w4(codes, scales, zeros, group_size=group)
        return
    even = torch.nn.functional.pad(codes, (0, k % 2))
    state.update(packed=even[:, 0::2] | (even[:, 1::2] << 4), scales=scales, zeros=zeros)


def _package():
    """The package's root is not on the path of a program that runs in the repository's root."""
    import os
    import sys
    root = os.path.join(os.getcwd(), 'micro-vllm_b200')
    if root not in sys.path:
        sys.path.insert(0, root)


def _hidden(gen, m, k):
    """Rows of a residual stream: a few channels are much larger than the rest."""
    x = torch.randn((m, k), generator=gen, device='cuda')
    loud = torch.rand((k,), generator=gen, device='cuda') < 0.004
    return torch.where(loud, x * 12, x)


def prepare(case, seed):
    if own:
        _package()
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, k = case['op'], case['k']
    state = {'case': case}
    if 'n' in case:
        _weights(case, gen, state)
    if op == 'dequant':
        return state
    m, kind = case['m'], TYPES[case['x']]
    if op == 'linear':
        x = _hidden(gen, m, k)
        if case['x'] in TOP:
            scale = x.abs().amax(-1, keepdim=True) / TOP[case['x']]
            x = x / scale
            state['x'] = x.round().to(kind) if case['x'] == 'int8' else x.to(kind)
            state['x_scale'] = scale[:, 0].contiguous()
        else:
            state['x'], state['x_scale'] = x.to(kind), None
    elif op.startswith('norm'):
        state['x'] = _hidden(gen, m, k).to(kind)
        state['stream'] = (_hidden(gen, m, k) * 2).to(kind)
        state['norm'] = (1 + 0.1 * torch.randn((k,), generator=gen, device='cuda')).to(kind)
    else:
        state['x'] = (_hidden(gen, m, 2 * k)).to(kind)
    if 'n' in case:
        out = TYPES[case['out']]
        state['bias'] = torch.randn((case['n'],), generator=gen, device='cuda').to(out) if case['bias'] else None
        state['residual'] = (torch.randn((m, case['n']), generator=gen, device='cuda').to(out)
                             if case['residual'] else None)
    return state


# The plain forms.

def _plain_weights(state):
    case = state['case']
    k, group = case['k'], case['group']
    packed = state['packed']
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(1)[:, :k].float()
    zeros = state['zeros'].float().repeat_interleave(group, 1)[:, :k] if case['zeros'] else 8.0
    return (codes - zeros) * state['scales'].float().repeat_interleave(group, 1)[:, :k]


def _plain_linear(state, x):
    y = x @ _plain_weights(state).t()
    if state['bias'] is not None:
        y = y + state['bias'].float()
    if state['residual'] is not None:
        y = y + state['residual'].float()
    return y.to(TYPES[state['case']['out']])


def _plain_norm(state):
    kind = TYPES[state['case']['x']]
    total = (state['x'].float() + state['stream'].float()).to(kind)
    s = total.float()
    return state['norm'].float() * (s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)), total


def _plain_silu(state):
    g, u = state['x'].float().chunk(2, dim=-1)
    return g / (1 + torch.exp(-g)) * u


def _plain_quant(y, out):
    scale = y.abs().amax(-1, keepdim=True) / TOP[out]
    q = torch.where(scale > 0, y / scale, 0.0)
    return (q.round() if out == 'int8' else q).to(TYPES[out]), scale[:, 0]


def _run_plain(state):
    case = state['case']
    op = case['op']
    if op == 'dequant':
        return _plain_weights(state).to(TYPES[case['out']])
    if op == 'linear':
        x = state['x'].float()
        return _plain_linear(state, x if state['x_scale'] is None else x * state['x_scale'][:, None])
    if op.startswith('norm'):
        y, total = _plain_norm(state)
    else:
        y, total = _plain_silu(state), None
    if op in ('norm', 'silu'):
        outs = _plain_quant(y, case['out']) if case['out'] in TOP else (y.to(TYPES[case['out']]),)
    else:
        q, scale = _plain_quant(y, 'int8')
        outs = (_plain_linear(state, q.float() * scale[:, None]),)
    return outs if total is None else outs + (total,)


def _run_own(state):
    from micro_vllm_b200.row_ops import add_rms_norm, add_rms_norm_quant, silu_mul_quant
    from micro_vllm_b200.w4_linear import w4_dequantize, w4_linear
    case = state['case']
    op, out = case['op'], case.get('out')
    if op == 'linear':
        return w4_linear(state['x'], state['weight'], state['bias'], state['residual'], x_scale=state['x_scale'],
                         out_dtype=TYPES[out])
    if op == 'dequant':
        return w4_dequantize(state['weight'], TYPES[out])
    if op == 'norm' and out not in TOP:
        return add_rms_norm(state['x'], state['stream'], state['norm'], EPS)
    if op == 'norm':
        return add_rms_norm_quant(state['x'], state['stream'], state['norm'], EPS, quant_dtype=TYPES[out])
    if op == 'silu':
        return silu_mul_quant(state['x'], quant_dtype=TYPES[out])
    if op == 'norm_linear':
        q, scale, total = add_rms_norm_quant(state['x'], state['stream'], state['norm'], EPS)
    else:
        q, scale = silu_mul_quant(state['x'])
    y = w4_linear(q, state['weight'], state['bias'], state['residual'], x_scale=scale, out_dtype=TYPES[out])
    return (y, total) if op == 'norm_linear' else (y,)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'int8': 1, 'e4m3': 1}
    op, k = case['op'], case['k']
    moved = flops = 0
    if 'n' in case:
        n, groups = case['n'], -(-k // case['group'])
        moved += n * k / 2 + n * groups * (2.5 if case['zeros'] else 2)
    if op == 'dequant':
        return {'bytes': moved + n * k * size[case['out']], 'flops': 2 * n * k}
    m, x = case['m'], size[case['x']]
    if op.startswith('norm'):  # the addend and the stream in, the stream out, the norm's weights
        moved += 3 * m * k * x + k * x
        flops += 6 * m * k
    elif op.startswith('silu'):
        moved += 2 * m * k * x
        flops += 8 * m * k
    else:
        moved += m * k * x + (4 * m if case['x'] in TOP else 0)
    if 'n' in case:
        out = size[case['out']]
        moved += m * n * out * (2 if case['residual'] else 1) + (n * out if case['bias'] else 0)
        flops += 2 * m * n * k
    else:
        moved += m * k * size[case['out']] + (4 * m if case['out'] in TOP else 0)
    return {'bytes': moved, 'flops': flops}


# The definitions in 64 bits.

def _exact_product(case, x, state):
    """x W^T, a block of rows of W at a time, group by group: sum_g scale_g (x_g code_g^T - zero_g sum x_g)."""
    n, k, group = case['n'], case['k'], case['group']
    groups = -(-k // group)
    padded = torch.nn.functional.pad(x, (0, groups * group - k)).view(-1, groups, group).transpose(0, 1)
    sums = padded.sum(-1)
    blocks = []
    for at in range(0, n, 2048):
        packed = state['packed'][at:at + 2048]
        codes = torch.zeros((packed.shape[0], groups * group), dtype=torch.float64, device='cuda')
        codes[:, 0:k:2] = (packed % 16).double()
        codes[:, 1:k:2] = torch.div(packed, 16, rounding_mode='floor')[:, :k // 2].double()
        parts = torch.einsum('gmk,ngk->mng', padded, codes.view(-1, groups, group))
        zero = (state['zeros'][at:at + 2048].double() if case['zeros']
                else torch.full((packed.shape[0], groups), 8.0, dtype=torch.float64, device='cuda'))
        parts = parts - torch.einsum('ng,gm->mng', zero, sums)
        blocks.append(torch.einsum('mng,ng->mn', parts, state['scales'][at:at + 2048].double()))
    y = torch.cat(blocks, dim=1)
    for name in ('bias', 'residual'):
        if state[name] is not None:
            y = y + state[name].double()
    return y


def exact(case, seed):
    global own
    asked, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = asked
    op, k = case['op'], case['k']
    if op == 'dequant':
        group, column = case['group'], torch.arange(k, device='cuda')
        codes = (state['packed'][:, column // 2] >> (4 * (column % 2)).to(torch.uint8)) % 16
        zero = state['zeros'][:, column // group].double() if case['zeros'] else 8.0
        return (codes.double() - zero) * state['scales'][:, column // group].double()
    x = state['x'].double()
    if op == 'linear':
        if state['x_scale'] is not None:
            x = x * state['x_scale'].double().unsqueeze(-1)
        return _exact_product(case, x, state)
    total = None
    if op.startswith('norm'):
        total = x + state['stream'].double()
        s = total.to(TYPES[case['x']]).double()
        y = s / (s.square().sum(-1, keepdim=True) / k + EPS).sqrt() * state['norm'].double()
    else:
        y = x[:, :k] * x[:, k:] / (1 + torch.exp(-x[:, :k]))
    if op in ('norm', 'silu') and case['out'] not in TOP:
        return (y, total)
    scale = y.abs().max(-1).values / TOP[case['out'] if op in ('norm', 'silu') else 'int8']
    q = torch.nan_to_num(y / scale.unsqueeze(-1), nan=0.0)
    if op in ('norm', 'silu'):
        outs = (q, scale)  # 8-bit values before their rounding: the nearest ones are the answer
    else:
        outs = (_exact_product(case, q.round() * scale.unsqueeze(-1), state),)
    return outs if total is None else outs + (total,)
