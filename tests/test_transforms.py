"""Function transforms, forward-mode differentiation and tracing: the 4-bit and 8-bit operators refuse them."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from micro_vllm_b200 import row_ops, w4_linear
from micro_vllm_b200._tensors import refuse_transforms


def test_what_is_refused_and_what_is_not():
    t = torch.ones(3)
    refuse_transforms(t, 't')
    with forward_ad.dual_level():
        refuse_transforms(t, 't')
        dual = forward_ad.make_dual(t, t)
        with pytest.raises(RuntimeError, match='forward-mode'):
            refuse_transforms(dual, 't')
        with torch.inference_mode():  # where torch leaves tangents out too
            refuse_transforms(dual, 't')

    def check(x):
        with pytest.raises(RuntimeError, match='traced'):
            refuse_transforms(x, 'x')
        return x + 1

    make_fx(check)(t)
    make_fx(check, tracing_mode='fake')(t)
    torch.vmap(check)(t)
    torch.func.functionalize(check)(t)
    torch.func.jvp(check, (t,), (t,))
    torch.func.grad(lambda x: check(x).sum())(t)
    with FakeTensorMode():
        check(torch.ones(3))

    class Counting(TorchDispatchMode):  # a mode of the user's own, over real tensors
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Counting():
        refuse_transforms(t, 't')


def test_fake_cuda_tensors_are_refused_without_a_gpu():
    with FakeTensorMode():
        x, w = torch.ones((2, 128), device='cuda'), torch.ones(128, device='cuda')
        for call in (lambda: row_ops.add_rms_norm(x, x, w, 1e-6), lambda: row_ops.add_rms_norm_quant(x, None, w, 1e-6),
                     lambda: row_ops.silu_mul_quant(x)):
            with pytest.raises(RuntimeError, match='traced'):
                call()


def calls(x, weight):
    w = torch.ones(128, device='cuda')
    residual = torch.ones_like(x)
    return [lambda t: w4_linear.w4_linear(t, weight), lambda t: w4_linear.w4_linear(x, weight, t[0, :64]),
            lambda t: row_ops.add_rms_norm(t, residual, w, 1e-6)[0], lambda t: row_ops.add_rms_norm(x, t, w, 1e-6)[0],
            lambda t: row_ops.add_rms_norm(x, residual, t[0], 1e-6)[0],
            lambda t: row_ops.add_rms_norm_quant(t, None, w, 1e-6)[1], lambda t: row_ops.silu_mul_quant(t)[1]]


@pytest.mark.gpu
def test_the_operators_refuse_transforms_and_run_beside_them():
    x = torch.randn((2, 128), device='cuda')
    weight = w4_linear.quantize_w4(torch.randn((64, 128), device='cuda'))
    for call in calls(x, weight):
        expected = call(x)
        with forward_ad.dual_level():
            assert torch.equal(call(x), expected)
            with pytest.raises(RuntimeError, match='forward-mode'):
                call(forward_ad.make_dual(x, x))
            with torch.inference_mode():
                assert torch.equal(call(forward_ad.make_dual(x, x)), expected)
        with pytest.raises(RuntimeError, match='traced'):
            make_fx(call)(x)
        with pytest.raises(RuntimeError, match='traced'):
            make_fx(call, tracing_mode='fake')(x)
        with pytest.raises(RuntimeError, match='traced'):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError, match='traced'):
            torch.vmap(call)(x[None])

        class Seen(TorchDispatchMode):
            def __torch_dispatch__(self, func, types, args=(), kwargs=None):
                seen.append(func)
                return func(*args, **(kwargs or {}))

        seen = []
        with Seen():
            assert torch.equal(call(x), expected)
        assert seen  # the outputs' allocation at least
    with pytest.raises(RuntimeError, match='traced'):
        make_fx(lambda t: w4_linear.w4_dequantize(weight, torch.float32) + t)(x[0])
