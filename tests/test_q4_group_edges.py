"""4-bit group weights where they can go wrong: addresses, cancellation, activations that are not finite."""
import numpy as np
import pytest

import ratchet_b200 as rb
from ratchet_b200 import Device, DType, Linear, Tensor
from ratchet_b200 import _lib
from test_q4_group import BF16, F16, G32, G64, G128, GROUP, HALF_STEP, activations, error_bound, pack, values, weight


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [G32, G64, G128, DType.Q4_K, DType.Q8_0H])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_addresses_inside_an_element_are_refused(dt, rows, gpu):
    """A byte off: refused on the host, before a kernel would read half a scale or half an activation."""
    lib, m, k = _lib.load(), 64, 256
    w = Tensor((m, k), dt, gpu)
    lin = Linear(w, Tensor((m,), F16, gpu))
    plan = gpu.plan_for(lin.schedule(Tensor((1, rows, k), F16, gpu)).op.desc)
    store = rb.GpuBuffer(gpu, 1 << 18)
    lhs, rhs, bias, out = (store.ptr + i * 65536 for i in range(4))
    zero = np.zeros(1 << 18, np.uint8)
    _lib.check(lib.rt_upload(gpu._h, store._h, 0, zero.ctypes.data, zero.size, 1))
    launch = lambda *at: lib.rt_matmul_launch(plan, *at, None)  # noqa: E731
    assert launch(lhs, rhs, bias, out) == _lib.RT_OK
    for bad in range(4):
        at = [lhs, rhs, bias, out]
        at[bad] += 1
        assert launch(*at) == _lib.RT_ERR_ARG, bad
    deq = lambda src, dst: lib.rt_dequantize_device(gpu._h, int(dt), 1024, src, dst, None)  # noqa: E731
    assert deq(lhs, out) == _lib.RT_OK and deq(lhs + 1, out) == _lib.RT_ERR_ARG and deq(lhs, out + 1) == _lib.RT_ERR_ARG
    gpu.sync()
