"""GPU: the 4-bit kernels' bounded wait gives up, sets the status bit and leaves the context usable.

``mvq_selftest_wait_timeout`` runs the tcgen05 kernel's own wait on a barrier that nothing completes, with a short limit.
"""
import ctypes
import time

import pytest
import torch

from tests.test_gpu_w4_linear import activations, assert_linear, make

pytestmark = pytest.mark.gpu


def _status(lib, device):
    from micro_vllm_b200 import _quant_native
    value = ctypes.c_uint32(7)
    _quant_native.check(lib.mvq_device_status(device, ctypes.byref(value)))
    return value.value


def test_a_wait_that_nothing_ends_gives_up_and_sets_the_status():
    from micro_vllm_b200 import _native, _quant_native
    from micro_vllm_b200.w4_linear import w4_linear
    lib, device = _quant_native.library(), torch.cuda.current_device()
    weight, w = make(200, 300, seed=1)
    x, _ = activations(16, 300, torch.bfloat16, seed=2)
    y = w4_linear(x.cuda(), weight)
    _quant_native.check(lib.mvq_clear_device_status(device))
    assert _status(lib, device) == 0
    torch.cuda.synchronize()
    for limit_ns in (1, 5_000_000):
        start = time.perf_counter()
        _quant_native.check(lib.mvq_selftest_wait_timeout(limit_ns, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert limit_ns * 1e-9 <= time.perf_counter() - start < 5
        assert _status(lib, device) == _quant_native.DEVICE_STATUS_WAIT_TIMEOUT
        # The other library has a word of its own.
        value = ctypes.c_uint32(7)
        _native.check(_native.library().mv_device_status(device, ctypes.byref(value)))
        assert value.value & _native.DEVICE_STATUS_WAIT_TIMEOUT == 0
        again = w4_linear(x.cuda(), weight)
        assert torch.equal(again, y)
        assert_linear(again, x, None, w, group=128)
        assert _status(lib, device) == _quant_native.DEVICE_STATUS_WAIT_TIMEOUT  # kept until it is cleared
        _quant_native.check(lib.mvq_clear_device_status(device))
        assert _status(lib, device) == 0


def test_limits_outside_the_range_are_refused_without_a_launch():
    from micro_vllm_b200 import _quant_native
    lib, device = _quant_native.library(), torch.cuda.current_device()
    _quant_native.check(lib.mvq_clear_device_status(device))
    for limit in (0, 100_000_001):
        assert lib.mvq_selftest_wait_timeout(limit, None) == 1
        assert b'limit_ns' in lib.mvq_last_error()
    torch.cuda.synchronize()
    assert _status(lib, device) == 0
