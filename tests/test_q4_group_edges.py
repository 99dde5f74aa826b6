"""4-bit group weights where they can go wrong: addresses, cancellation, activations that are not finite."""
import ctypes

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


def apart_bound(act, dt, q, s, z, x, y):
    """How far the GEMV may be off: it sums q x and x apart and takes z times the second from the first, so that its f32 roundings go
    with (q + z) |x|.  Of a group: four warp MMAs one after the other for each half of its codes, each the sum of 16 products and what
    came before, a step of 2^-23 for each of the 17 at most; nine additions for the sum of x; one to join the halves.  Of a row: two
    roundings a step of 128 values, then the sums of at most 20 warps, 4 CTAs and 4 lanes.  Then the output's rounding."""
    mass = np.abs(x).astype(np.float64) @ ((q + np.repeat(z, GROUP[dt], 1)) * np.abs(np.repeat(s.astype(np.float64), GROUP[dt], 1))).T
    steps = 4 * 17 * 2 + 9 + 1 + 2 * (q.shape[1] / 128) + 28
    return steps * 2.0**-24 * mass * (1 + HALF_STEP[act]) + HALF_STEP[act] * np.abs(y) + 2.0**-25


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("dt", [G32, G64, G128])
@pytest.mark.parametrize("zero,near", [(8, 0), (8, 1), (15, 0), (15, 1), (31, 0)])
def test_codes_at_their_zero_point(zero, near, dt, act, gpu):
    """Weights that are differences of much larger numbers: every code equal to its zero point, or next to it, under activations that
    do not cancel of themselves."""
    for i, (m, k, rows) in enumerate([(50, 384, 1), (64, 2560, 2), (40, 10240, 5), (33, 2560, 7), (64, 5120, 16), (2000, 1280, 3)]):
        rng = np.random.default_rng(300 + i)
        q = np.clip(zero + rng.integers(-near, near + 1, (m, k)), 0, 15)
        s = (rng.uniform(0.2, 1.0, (m, k // GROUP[dt])) * rng.choice([-0.02, 0.02], (m, k // GROUP[dt]))).astype(np.float16)
        z = np.full(s.shape, zero)
        x = activations(act, (1, rows, k), 400 + i)
        x[0, ::2] = np.abs(x[0, ::2])
        y = x[0].astype(np.float64) @ values(dt, q, s, z).T
        out = Linear(Tensor.from_quantized(pack(dt, q, s, z), dt, (m, k)).to(gpu)).schedule(Tensor.from_data(x, gpu, act))
        assert "q4_group_gemv" in _lib.load().rt_plan_kernel(gpu.plan_for(out.op.desc)).decode()
        got = out.resolve().to(Device.CPU).to_f32()
        over = np.abs(got[0] - y) - apart_bound(act, dt, q, s, z, x[0], y)
        assert np.all(over <= 0), (m, k, rows, float(over.max()))


@pytest.mark.gpu
def test_scatter_destinations_inside_an_element_are_refused(gpu):
    lib, m, k, rows = _lib.load(), 256, 256, 64
    plan = gpu.plan_for(Linear(Tensor((m, k), G64, gpu)).schedule(Tensor((1, rows, k), F16, gpu)).op.desc)
    assert "umma" in lib.rt_plan_kernel(plan).decode()
    store = rb.GpuBuffer(gpu, 1 << 18)
    zero = np.zeros(1 << 18, np.uint8)
    _lib.check(lib.rt_upload(gpu._h, store._h, 0, zero.ctypes.data, zero.size, 1))
    opts = _lib.rt_launch_opts()
    opts.n_out, opts.out_ld, opts.out_col = 1, m, 0
    for off, want in ((0, _lib.RT_OK), (1, _lib.RT_ERR_ARG)):
        opts.outs[0] = store.ptr + (1 << 17) + off
        assert lib.rt_matmul_launch_ex(plan, store.ptr, store.ptr + 65536, None, None, None, ctypes.byref(opts)) == want
    gpu.sync()
