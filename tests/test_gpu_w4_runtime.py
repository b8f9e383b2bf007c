"""The batched runtime on 4-bit projections: prefill, decode steps, graphs and the greedy loop.

The same model with its operators replaced by their plain forms (64-bit sums,
rounded where the operators round) is the reference. Both see the same codes.
What differs is fp32 summation (2^-20 of a projection's size, see
test_gpu_w4_linear.py) and where that crosses a rounding's border: in fp32 nothing
is rounded to fewer bits, so logits of three layers stay within 2^-12 of the
largest; with int8 rows one value of a row may come out one step (1/127 of the
row's largest) apart, which moves a projection's result by 1/127 of one product
of hundreds, below 2^-8 of the logits' size for a handful of them.
"""
import pytest
import torch
import torch.nn.functional as F

from tests.golden.model_cases import MODEL_CASES, make_prompts, make_weights, model_config

pytestmark = pytest.mark.gpu


def model_of(name, dtype, **kw):
    from micro_vllm_b200.runtime import prepare_model
    weights = {k: torch.from_numpy(v).to(dtype).cuda() for k, v in make_weights(name).items()}
    return prepare_model(weights, model_config(name), **kw)


def plain_linear(x, weight, bias=None, residual=None, *, x_scale=None, out_dtype=None, out=None):
    from micro_vllm_b200.w4_linear import w4_dequantize
    y = x.double() if x.dtype != torch.int8 else x.double() * x_scale.double().unsqueeze(-1)
    y = y @ w4_dequantize(weight, torch.float32).double().t()
    for more in (bias, residual):
        y = y if more is None else y + more.double()
    return y.to(out_dtype or x.dtype)


def plain_norm(x, residual, weight, eps):
    s = x if residual is None else x + residual
    s64 = s.double()
    return weight.double() * s64 * torch.rsqrt((s64 * s64).mean(-1, keepdim=True) + eps), s


def plain_quant(y):
    scale = y.abs().amax(-1) / 127
    return (y / scale.unsqueeze(-1)).round().to(torch.int8), scale.float()


def plain_operators(monkeypatch):
    from micro_vllm_b200 import runtime

    def norm(x, residual, weight, eps):
        y, s = plain_norm(x, residual, weight, eps)
        return y.to(x.dtype), s

    def norm_quant(x, residual, weight, eps):
        y, s = plain_norm(x, residual, weight, eps)
        return (*plain_quant(y), s)

    def silu_quant(gate_up):
        g, u = gate_up.double().chunk(2, dim=-1)
        return plain_quant(g / (1 + torch.exp(-g)) * u)

    monkeypatch.setattr(runtime, 'w4_linear', plain_linear)
    monkeypatch.setattr(runtime, 'add_rms_norm', norm)
    monkeypatch.setattr(runtime, 'add_rms_norm_quant', norm_quant)
    monkeypatch.setattr(runtime, 'silu_mul_quant', silu_quant)


def logits_of(model, name, steps=4, batch=None):
    """Prefill logits and those of some decode steps on fixed tokens."""
    prompts = torch.from_numpy(make_prompts(name)).cuda()
    if batch:
        prompts = prompts.repeat(batch, 1)[:batch]
    cache = model.allocate_cache(prompts.shape[0], prompts.shape[1] + steps, shuffle_seed=3)
    model.bind(cache)
    found = [model.prefill(prompts, cache)]
    for step in range(steps):
        lens = cache.lengths + 1
        found.append(model.decode(prompts[:, step], lens))
        cache.lengths.copy_(lens)
        cache.note_advanced(1)
    return found


@pytest.mark.parametrize('name', list(MODEL_CASES))
@pytest.mark.parametrize('bits,zeros,group', [(16, False, 128), (16, True, 32), (8, False, 64), (8, True, 128)])
def test_logits_match_the_plain_operators(name, bits, zeros, group, monkeypatch):
    model = model_of(name, torch.float32, weight_bits=4, group_size=group, zeros=zeros, activation_bits=bits)
    found = logits_of(model, name)
    plain_operators(monkeypatch)
    expected = logits_of(model, name)
    for got, want in zip(found, expected):
        bound = (2.0 ** -8 if bits == 8 else 2.0 ** -12) * float(want.abs().max())
        assert float((got - want).abs().max()) <= bound


@pytest.mark.parametrize('name', list(MODEL_CASES))
def test_a_prompt_is_multiplied_by_codes_or_by_the_written_out_weights(name, monkeypatch):
    """Both ways of prefill, against F.linear on the weights of the formula."""
    from micro_vllm_b200 import runtime
    from micro_vllm_b200.w4_linear import w4_dequantize
    model = model_of(name, torch.float32, weight_bits=4, group_size=64)
    prompts = torch.from_numpy(make_prompts(name)).cuda()
    found = []
    for rows in (0, 1 << 30):
        monkeypatch.setattr(runtime, 'CODES_ROWS', rows)
        cache = model.allocate_cache(prompts.shape[0], prompts.shape[1])
        found.append(model.prefill(prompts, cache))
    for w in model.layers:
        for key in ('qkv', 'self_attn.o_proj.weight', 'gate_up', 'mlp.down_proj.weight'):
            w[key] = w4_dequantize(w[key], torch.float32)
    model.weight_bits = 16
    cache = model.allocate_cache(prompts.shape[0], prompts.shape[1])
    expected = model.prefill(prompts, cache)
    for got in found:
        assert float((got - expected).abs().max()) <= 2.0 ** -12 * float(expected.abs().max())


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('batch', [2, 19])
def test_graph_replayed_steps_equal_eager_steps(bits, batch):
    from micro_vllm_b200.generate import GreedyDecoder
    name = 'tiny_qwen2_tied'
    model = model_of(name, torch.bfloat16, weight_bits=4, activation_bits=bits)
    prompts = torch.from_numpy(make_prompts(name)).cuda().repeat(batch, 1)[:batch]
    tokens = GreedyDecoder(model, batch, prompts.shape[1] + 12).run(prompts, 12)
    eager = GreedyDecoder(model, batch, prompts.shape[1] + 12, use_graph=False).run(prompts, 12)
    assert torch.equal(tokens, eager) and tokens.shape == (batch, 12)
    assert int(tokens.min()) >= 0 and int(tokens.max()) < model.vocab


def test_bits_are_checked_and_sixteen_bits_change_nothing():
    from micro_vllm_b200.runtime import PreparedModel
    name = 'tiny_qwen2_fp32'
    for kw in (dict(weight_bits=8), dict(activation_bits=8), dict(weight_bits=4, activation_bits=4)):
        with pytest.raises(ValueError, match='bits'):
            model_of(name, torch.float32, **kw)
    model = model_of(name, torch.bfloat16)
    assert isinstance(model, PreparedModel) and isinstance(model.layers[0]['qkv'], torch.Tensor)
    w = model.layers[0]
    x = torch.randn((3, 256), device='cuda').to(torch.bfloat16)
    assert torch.equal(model._project(x, w, 'gate_up'), F.linear(x, w['gate_up']))
