"""4-bit weights with group scales (Q4_G32 / G64 / G128): codec and rules on the CPU, products against 64-bit sums on the GPU."""
import ctypes

import numpy as np
import pytest

import ratchet_b200 as rb
from ratchet_b200 import Device, DType, Executable, InvariantError, Linear, MLP, Quantizer, RatchetError, ShapeError, Tensor
from ratchet_b200 import _lib
from util import round_to

GROUP = {DType.Q4_G32: 32, DType.Q4_G64: 64, DType.Q4_G128: 128}
G32, G64, G128 = GROUP
F16, BF16, F32 = DType.F16, DType.BF16, DType.F32
HALF_STEP = {F16: 2.0**-11, BF16: 2.0**-8}


def pack(dt, q, s, z):
    """Codes [M][K] 0..15, scales [M][K/g] f16 and zero points as the dtype's buffer."""
    out = np.zeros(dt.nbytes(q.size), np.uint8)
    flat = q.reshape(-1).astype(np.uint8)
    for (offset, _), part in zip(dt.segments(q.size), (flat[0::2] | flat[1::2] << 4, s.astype(np.float16).view(np.uint8), z.astype(np.uint8))):
        out[offset:offset + part.size] = part.reshape(-1)
    return out


def values(dt, q, s, z):
    g = GROUP[dt]
    lead = q.shape[:-1]
    steps = q.reshape(*lead, -1, g).astype(np.float64) - (z.astype(np.int64) & 31)[..., None]
    return (steps * s.astype(np.float16).astype(np.float64)[..., None]).reshape(q.shape)


def weight(dt, shape, seed, zmax=16, signed=True):
    """(tensor, its values in 64 bits): any codes, scales of either sign, zero points 0 .. zmax."""
    rng, g = np.random.default_rng(seed), GROUP[dt]
    q = rng.integers(0, 16, size=shape)
    s = (rng.uniform(0.2, 1.0, size=(*shape[:-1], shape[-1] // g)) * 0.02).astype(np.float16)
    if signed:
        s = s * rng.choice([-1, 1], size=s.shape).astype(np.float16)
    z = rng.integers(0, zmax + 1, size=s.shape)
    return Tensor.from_quantized(pack(dt, q, s, z), dt, shape), values(dt, q, s, z)


# ------------------------------------------------------------------------------------------------ CPU

@pytest.mark.parametrize("dt", list(GROUP))
def test_segments_codes_scales_zero_points(dt):
    g = GROUP[dt]
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    for groups in (1, 3, 8, 301):
        n = groups * g
        assert dt.segments(n) == [(0, up(n // 2)), (up(n // 2), up(groups * 2)), (up(n // 2) + up(groups * 2), up(groups))]
        assert dt.nbytes(n) == up(n // 2) + up(groups * 2) + up(groups)
    assert dt.is_quantized() and dt.activation_dt() == F16 and dt.size_of() == 0
    with pytest.raises(ShapeError):
        dt.segments(g + g // 2)
    # two entries are too few for this format's three segments
    segs, n = (_lib.rt_segment * 2)(), ctypes.c_int32(2)
    assert _lib.load().rt_dtype_segments(int(dt), g, segs, ctypes.byref(n)) == _lib.RT_ERR_ARG


@pytest.mark.parametrize("dt", list(GROUP))
def test_decode_is_the_definition(dt):
    t, want = weight(dt, (5, 3 * GROUP[dt]), seed=int(dt), zmax=31)
    got = Quantizer.dequantize_bytes(t.storage, dt, want.size).reshape(want.shape)
    assert np.array_equal(got.astype(np.float64), want)
    # only the low five bits of a zero point count
    raw = t.storage.copy()
    off, _ = dt.segments(want.size)[2]
    raw[off:off + want.size // GROUP[dt]] |= 0xE0
    assert np.array_equal(Quantizer.dequantize_bytes(raw, dt, want.size), got.reshape(-1))


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dt", list(GROUP))
def test_quantiser_stays_within_half_a_step(dt, symmetric):
    """Affine: 15 steps from min(v, 0) to max(v, 0); a value is off by half a step, the zero point's rounding can cost the
    far end another half, and s itself is half an f16 step off over at most 15 of them."""
    g = GROUP[dt]
    x = (np.random.default_rng(7).standard_normal((64, 2 * g)) * 0.02).astype(np.float32)
    x[0, :g], x[1, :g], x[2, :g] = 0, np.abs(x[1, :g]), -np.abs(x[2, :g])
    x[3, :g], x[3, 5] = 0, 1e-3
    t = Quantizer.q4_group_quantize(Tensor.from_data(x), dt, symmetric)
    got = Quantizer.dequantize_bytes(t.storage, dt, x.size).reshape(-1, g)
    v = x.reshape(-1, g).astype(np.float64)
    lo, hi = np.minimum(v.min(1), 0), np.maximum(v.max(1), 0)
    step = np.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15
    slack = step * (0.5 if symmetric else 1.0) * (1 + 2.0**-10) + 15 * step * 2.0**-11 + 2.0**-24 * 15
    assert np.all(np.abs(got - v) <= slack[:, None])
    assert np.all(got[0] == 0) and got.shape[0] == 128


def test_quantiser_takes_what_is_not_finite():
    x = np.zeros(64, np.float32)
    x[:4] = [np.nan, np.inf, -1.0, 1.0]
    x[32:36] = [1e30, -1e30, 3.0, 0.0]
    t = Quantizer.q4_group_quantize(Tensor.from_data(x), G32)
    got = Quantizer.dequantize_bytes(t.storage, G32, 64)
    assert np.all(np.isfinite(got)) and got[0] == 0 and got[1] > 0 and got[32] > 0 > got[33]


def test_quantiser_refusals():
    x = Tensor.from_data(np.zeros((2, 48), np.float32))
    with pytest.raises(ShapeError):
        Quantizer.q4_group_quantize(x, G128)
    with pytest.raises(InvariantError):
        Quantizer.q4_group_quantize(Tensor.from_data(np.zeros((2, 64), np.float16)), G64)
    lib, out = _lib.load(), np.zeros(4096, np.uint8)
    src = np.zeros(128, np.float32)
    for dt in (DType.Q4_K, DType.Q8_0F, DType.F16):
        assert lib.rt_quantize_q4_group(src.ctypes.data, 128, int(dt), 0, out.ctypes.data) == _lib.RT_ERR_ARG
        assert lib.rt_dequantize_q4_group(out.ctypes.data, 128, int(dt), src.ctypes.data) == _lib.RT_ERR_ARG


def test_matmul_rules():
    w, _ = weight(G64, (16, 192), 1)
    lin = Linear(w)
    for dt in (F16, BF16):
        y = lin.schedule(Tensor.from_data(np.zeros((1, 3, 192), np.float32), dt=dt))
        assert y.shape == [1, 3, 16] and y.dt == dt
    for dt in (F32, DType.I32):
        with pytest.raises(InvariantError, match="Failed to validate DTypes"):
            lin.schedule(Tensor.from_data(np.zeros((1, 3, 192)), dt=dt))
    with pytest.raises(InvariantError, match="Transposed quantized"):
        w.gemm(Tensor.from_data(np.zeros((16, 2), np.float16)), None, True, False, False)
    with pytest.raises(ShapeError, match="multiple of 128"):
        Linear(Tensor.from_quantized(np.zeros(G128.nbytes(4 * 192), np.uint8), G128, (4, 192))).schedule(
            Tensor.from_data(np.zeros((1, 192), np.float16)))


@pytest.mark.parametrize("dt", list(GROUP))
def test_a_shard_is_the_rows_of_the_whole(dt):
    t, want = weight(dt, (37, 3 * GROUP[dt]), 5)
    for r0, r1 in ((0, 37), (0, 1), (11, 30), (36, 37), (4, 4)):
        part = rb.shard_rows(t, r0, r1)
        got = Quantizer.dequantize_bytes(part.storage, dt, part.numel()) if part.numel() else np.zeros(0)
        assert part.shape == [r1 - r0, want.shape[1]] and np.array_equal(got, want[r0:r1].reshape(-1).astype(np.float32))


# ------------------------------------------------------------------------------------------------ GPU

def error_bound(dt, w, x, y, bias=None, rounded_weights=False):
    """How far a correct result may be from y = x w^T + bias: the output's rounding (f16 rounds the sum, then adds the bias and
    rounds again), the f32 sum's (each of its K additions half a step of a partial sum, which is at most sum |w x|; the
    products are exact: 5 + 11 or 8 bits, the group's scale 11 more), and, on the GEMM route, each weight's to f16."""
    mass = np.abs(x) @ np.abs(w).T
    u = HALF_STEP[dt]
    out = u * np.abs(y) + (u * np.abs(y - (0 if bias is None else bias)) if bias is not None else 0) + 2.0**-24
    return out * (1 + 2.0**-6) + mass * ((w.shape[1] + 8) * 2.0**-24 + (2.0**-11 if rounded_weights else 0))


def run(w, x, dt, gpu, bias=None, epilogue=rb.EPILOGUE_NONE):
    b = Tensor.from_data(bias, gpu, dt) if bias is not None else None
    out = Linear(w.to(gpu), b, epilogue).schedule(Tensor.from_data(x, gpu, dt))
    kernel = _lib.load().rt_plan_kernel(gpu.plan_for(out.op.desc)).decode()
    return out.resolve().to(Device.CPU).to_f32(), kernel


def activations(dt, shape, seed):
    return round_to(dt, np.random.default_rng(seed).standard_normal(shape).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(GROUP))
def test_device_decode_is_bit_exact(dt, gpu):
    t, want = weight(dt, (33, 5 * GROUP[dt]), 2, zmax=31)
    assert np.array_equal(t.to(gpu).dequantize_on_device().reshape(-1).astype(np.float64), want.reshape(-1))


SHAPES = [  # rows of W, groups per row: one group, odd numbers of both, rows around a tile's, long rows, many rows
    (1, 1), (7, 1), (16, 3), (17, 5), (31, 4), (33, 7), (200, 11), (515, 20), (130, 85), (2048, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("dt", list(GROUP))
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17, 40])
def test_linear_against_64_bit_sums(dt, act, rows, gpu):
    for i, (m, groups) in enumerate(SHAPES):
        k = groups * GROUP[dt]
        w, wv = weight(dt, (m, k), seed=100 + i)
        x = activations(act, (1, rows, k), seed=200 + i)
        y = x[0].astype(np.float64) @ wv.T
        got, kernel = run(w, x, act, gpu)
        over = np.abs(got[0] - y) - error_bound(act, wv, x[0].astype(np.float64), y, rounded_weights="umma" in kernel)
        assert got.shape == (1, rows, m) and np.all(over <= 0), (kernel, m, k, float(over.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 3, 16, 33])
def test_bias_gelu_and_the_gate_up_fold(act, rows, gpu):
    m, k = 258, 384
    w, wv = weight(G64, (m, k), 9)
    x = activations(act, (1, rows, k), 10)
    bias = round_to(act, np.random.default_rng(11).standard_normal(m).astype(np.float32))
    plain = x[0].astype(np.float64) @ wv.T + bias
    got, kernel = run(w, x, act, gpu, bias)
    e = error_bound(act, wv, x[0].astype(np.float64), plain, bias.astype(np.float64), "umma" in kernel)
    assert np.all(np.abs(got[0] - plain) <= e), kernel
    u = HALF_STEP[act]
    gelu = lambda v: v * 0.5 * (1 + np.tanh(v * (0.7978846 + 0.035677407 * v * v)))  # noqa: E731
    got, kernel = run(w, x, act, gpu, bias, rb.EPILOGUE_GELU_TANH)
    # gelu's slope is below 1.13; its f32 evaluation loses a few steps of 2^-24 of v
    assert np.all(np.abs(got[0] - gelu(plain)) <= 1.13 * e + u * np.abs(gelu(plain)) * (1 + 2.0**-6) + 2.0**-20 * np.abs(plain) + 2.0**-24), kernel
    got, kernel = run(w, x, act, gpu, bias, rb.EPILOGUE_SILU_MUL)
    gate, up, eg, eu = plain[:, :m // 2], plain[:, m // 2:], e[:, :m // 2], e[:, m // 2:]
    silu = gate / (1 + np.exp(-gate))
    want = silu * up
    es = 1.1 * eg + (u + 2.0**-20) * np.abs(silu) + 2.0**-24  # silu's slope is below 1.1
    assert np.all(np.abs(got[0] - want) <= es * (np.abs(up) + eu) + np.abs(silu) * eu + u * (np.abs(want) + es * np.abs(up)) * 1.02 + 2.0**-24), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 1), (16, 1), (3, 5), (40, 1), (2, 20)])
def test_batches_share_one_weight(shape, gpu):
    """[batch, rows, K] against one W: the same as its rows one after the other, whatever the split."""
    w, wv = weight(G128, (100, 640), 3)
    x = activations(F16, (*shape, 640), 4)
    y = x.astype(np.float64) @ wv.T
    got, kernel = run(w, x, F16, gpu)
    e = error_bound(F16, wv, x.reshape(-1, 640).astype(np.float64), y.reshape(-1, 100), rounded_weights="umma" in kernel)
    assert got.shape == (*shape, 100) and np.all(np.abs(got - y).reshape(-1, 100) <= e), kernel


@pytest.mark.gpu
def test_a_weight_per_batch_and_the_other_forms(gpu):
    """W of [batch, M, K]; outputs not transposed; a vector rhs; rhs stored [K][N]."""
    w, wv = weight(G32, (3, 50, 160), 6)
    x = activations(F16, (3, 2, 160), 7)
    y = np.einsum("bmk,bnk->bnm", wv, x.astype(np.float64))
    e = np.stack([error_bound(F16, wv[b], x[b].astype(np.float64), y[b]) for b in range(3)])
    wg, xg = w.to(gpu), Tensor.from_data(x, gpu, F16)
    assert np.all(np.abs(wg.gemm(xg, None, False, True, True).resolve().to(Device.CPU).to_f32() - y) <= e)
    got = wg.gemm(xg, None, False, True, False).resolve().to(Device.CPU).to_f32()
    assert np.all(np.abs(got.transpose(0, 2, 1) - y) <= e)
    xt = Tensor.from_data(np.ascontiguousarray(x.transpose(0, 2, 1)), gpu, F16)
    got = wg.gemm(xt, None, False, False, False).resolve().to(Device.CPU).to_f32()
    assert np.all(np.abs(got.transpose(0, 2, 1) - y) <= e)
    w1, v1 = weight(G32, (50, 160), 8)
    got = w1.to(gpu).gemm(Tensor.from_data(x[0, 0], gpu, F16), None, False, False, False).resolve().to(Device.CPU).to_f32()
    y1 = v1 @ x[0, 0].astype(np.float64)
    assert got.shape == (50,) and np.all(np.abs(got - y1) <= error_bound(F16, v1, x[0, :1].astype(np.float64), y1[None])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 2, 6, 16])
def test_infinities_and_nans_stay_in_their_rows(act, rows, gpu):
    """An infinite activation gives +-inf by the weight's sign and NaN against a zero weight; other rows keep their bits."""
    dt, m, k = G64, 96, 512
    w, wv = weight(dt, (m, k), 12)
    x = activations(act, (1, rows, k), 13)
    clean, kernel = run(w, x, act, gpu)
    for bad in (np.inf, -np.inf, np.nan):
        v = x.copy()
        v[0, rows - 1, 130] = bad
        got, _ = run(w, v, act, gpu)
        assert np.array_equal(got[0, :-1], clean[0, :-1]), kernel
        with np.errstate(invalid="ignore"):
            want = bad * wv[:, 130]
        assert np.array_equal(got[0, -1], want.astype(np.float32), equal_nan=True), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 16])
def test_operands_off_a_16_byte_boundary(rows, gpu):
    w, wv = weight(G32, (40, 96), 14)
    x = activations(F16, (1, rows, 96), 15)
    y = x[0].astype(np.float64) @ wv.T
    out = Linear(w.to(gpu)).schedule(Tensor.from_data(x, gpu, F16))
    plan, lib = gpu.plan_for(out.op.desc), _lib.load()
    store = rb.GpuBuffer(gpu, 1 << 16)
    raw = np.zeros(1 << 16, np.uint8)
    raw[8:8 + w.storage.size] = w.storage
    raw[32768 + 2:32768 + 2 + x.size * 2] = x.astype(np.float16).view(np.uint8).reshape(-1)
    rb._lib.check(lib.rt_upload(gpu._h, store._h, 0, raw.ctypes.data, raw.size, 1))
    rb._lib.check(lib.rt_matmul_launch(plan, store.ptr + 8, store.ptr + 32770, None, store.ptr + 49152 + 2, None))
    back = np.zeros(1 << 16, np.uint8)
    rb._lib.check(lib.rt_download(gpu._h, store._h, 0, back.ctypes.data, back.size, 1))
    got = back[49154:49154 + rows * 40 * 2].view(np.float16).reshape(rows, 40).astype(np.float64)
    assert np.all(np.abs(got - y) <= error_bound(F16, wv, x[0].astype(np.float64), y))
    assert np.array_equal(back[:49154], raw[:49154]) and not back[49154 + rows * 80:].any()  # nothing else was written


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 30])
def test_mlp_and_executable_run_the_lazy_graph_s_bits(rows, gpu):
    w1, _ = weight(G128, (512, 256), 16)
    w2, _ = weight(G32, (256, 256), 17)
    fc1, fc2 = Linear(w1.to(gpu)), Linear(w2.to(gpu))
    x = Tensor.from_data(activations(F16, (1, rows, 256), 18), gpu, F16)
    mlp = MLP(fc1, fc2, "silu_gate")
    got = mlp.schedule(x)
    gpu.sync()
    lazy = fc2.schedule(Linear(fc1.w, None, rb.EPILOGUE_SILU_MUL).schedule(x)).resolve()
    want = lazy.to(Device.CPU).to_f32()
    assert np.array_equal(got.to(Device.CPU).to_f32(), want)
    for graph in (True, False):
        exe = Executable(gpu, [lazy.op.rhs, lazy], use_graph=graph)
        for _ in range(3):
            exe.dispatch()
        gpu.sync()
        assert np.array_equal(lazy.to(Device.CPU).to_f32(), want)


@pytest.mark.gpu
def test_empty_products(gpu):
    w, _ = weight(G32, (8, 64), 19)
    y = Linear(w.to(gpu)).schedule(Tensor.from_data(np.zeros((1, 0, 64), np.float16), gpu)).resolve()
    assert y.shape == [1, 0, 8]


# What a product's kernel is called depends on the GPU's number of SMs in the last part only (how rows and K are shared out).

def product(w, wv, x, act, gpu, bias=None, epilogue=rb.EPILOGUE_NONE):
    """(result, 64-bit sums, how far off they may be, kernel)"""
    y = x[0].astype(np.float64) @ wv.T + (0 if bias is None else bias)
    got, kernel = run(w, x, act, gpu, bias, epilogue)
    return got[0], y, error_bound(act, wv, x[0].astype(np.float64), y, bias, "umma" in kernel), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("m,k,rows,ranks", [(16, 5120, 8, 2), (50, 5120, 7, 2), (16, 3200, 16, 4), (130, 3232, 13, 1), (200, 6432, 15, 4), (25, 10272, 16, 4), (16, 25600, 1, None), (40, 20480, 3, None)])
def test_k_shared_by_warps_and_by_a_cluster(m, k, rows, ranks, act, gpu):
    """Few rows of great length, the last step partial or a whole CTA's share shorter; infinities there as well."""
    w, wv = weight(G32, (m, k), 31)
    x = activations(act, (1, rows, k), 32)
    got, y, e, kernel = product(w, wv, x, act, gpu)
    assert kernel.startswith(f"q4_group_gemv_g32_nv{rows}_") and (ranks is None or f"x{ranks}_" in kernel), kernel
    assert np.all(np.abs(got - y) <= e), kernel
    x[0, rows - 1, k - 1] = np.inf
    bad, _ = run(w, x, act, gpu)
    with np.errstate(invalid="ignore"):
        assert np.array_equal(bad[0, :-1], got[:-1]) and np.array_equal(bad[0, -1], (np.inf * wv[:, k - 1]).astype(np.float32), equal_nan=True), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 4, 8, 12, 16])
def test_k_that_is_no_multiple_of_a_step(rows, gpu):
    for dt, k in ((G32, 32), (G32, 96), (G32, 160), (G32, 2592), (G64, 64), (G64, 192), (G64, 2624)):
        w, wv = weight(dt, (37, k), k)
        for act in (F16, BF16):
            got, y, e, kernel = product(w, wv, activations(act, (1, rows, k), 33), act, gpu)
            assert np.all(np.abs(got - y) <= e), (kernel, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,m", [(12, 16), (16, 16), (9, 300), (12, 2)])
def test_rows_too_long_for_the_gemv(rows, m, gpu):
    """25600 values of 9 and more vectors do not fit its shared memory: the general routes take them, with the fold as well."""
    w, wv = weight(G128, (m, 25600), 34)
    x = activations(F16, (1, rows, 25600), 35)
    got, y, e, kernel = product(w, wv, x, F16, gpu)
    assert "q4_group_gemv" not in kernel and np.all(np.abs(got - y) <= e), kernel
    fold, kernel = run(w, x, F16, gpu, None, rb.EPILOGUE_SILU_MUL)
    gate, up, eg, eu = y[:, :m // 2], y[:, m // 2:], e[:, :m // 2], e[:, m // 2:]
    silu = gate / (1 + np.exp(-gate))
    es = 1.1 * eg + (2.0**-11 + 2.0**-20) * np.abs(silu) + 2.0**-24
    bound = es * (np.abs(up) + eu) + np.abs(silu) * eu + 2.0**-11 * (np.abs(silu * up) + es * np.abs(up)) * 1.02 + 2.0**-24
    assert np.all(np.abs(fold[0] - silu * up) <= bound), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 5, 20])
def test_the_cuda_core_kernel_s_bits_are_within_the_same_bounds(rows, act, gpu, monkeypatch):
    monkeypatch.setenv("RT_FORCE_KERNEL", "simt")
    for dt in GROUP:
        w, wv = weight(dt, (70, 3 * GROUP[dt]), 36)
        x = activations(act, (1, rows, 3 * GROUP[dt]), 37)
        bias = round_to(act, np.random.default_rng(38).standard_normal(70).astype(np.float32)).astype(np.float64)
        got, y, e, kernel = product(w, wv, x, act, gpu, bias)
        assert "simt" in kernel and np.all(np.abs(got - y) <= e), kernel
        fold, kernel = run(w, x, act, gpu, bias, rb.EPILOGUE_SILU_MUL)
        gate, up = y[:, :35], y[:, 35:]
        silu, u = gate / (1 + np.exp(-gate)), HALF_STEP[act]
        es = 1.1 * e[:, :35] + (u + 2.0**-20) * np.abs(silu) + 2.0**-24
        bound = es * (np.abs(up) + e[:, 35:]) + np.abs(silu) * e[:, 35:] + u * (np.abs(silu * up) + es * np.abs(up)) * 1.02 + 2.0**-24
        assert "simt" in kernel and np.all(np.abs(fold[0] - silu * up) <= bound), kernel


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 8, 16])
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-8, 1e8, 1e30, 1e36])
def test_bf16_activations_of_every_size(scale, rows, gpu):
    """Every step of a vector has a power of two of its own: sizes that f16 does not have, and steps that differ by 2^40."""
    for dt in GROUP:
        k = 640
        w, wv = weight(dt, (48, k), 39)
        x = np.random.default_rng(40).standard_normal((1, rows, k)) * scale
        if scale < 1:
            x[..., 128:256] *= 2.0**-20
            x[..., 256:384] *= 2.0**20
        x = round_to(BF16, x.astype(np.float32))
        v = x[0].astype(np.float64)
        y = v @ wv.T
        got, kernel = run(w, x, BF16, gpu)
        # a value that leaves f16's range below loses 2^-24 of its step's largest or less: 2^-25 of a step's largest magnitude for each of its weights
        steps = np.abs(v).reshape(rows, -1, 128).max(-1)
        lost = np.einsum("ns,ms->nm", steps, np.abs(wv).reshape(48, -1, 128).sum(-1)) * 2.0**-24
        e = HALF_STEP[BF16] * np.abs(y) * (1 + 2.0**-6) + (np.abs(v) @ np.abs(wv).T) * ((k + 8) * 2.0**-24) + lost + 2.0**-133
        assert np.all(np.abs(got[0] - y) <= e), (kernel, float((np.abs(got[0] - y) - e).max()))


@pytest.mark.gpu
def test_the_gemv_on_two_streams_and_in_a_replayed_graph(gpu):
    import torch
    lib = _lib.load()
    w, wv = weight(G32, (130, 3232), 41)
    w2, wv2 = weight(G64, (200, 640), 42)
    cases = []
    for wt, vals, rows in ((w, wv, 13), (w2, wv2, 1)):
        k = vals.shape[1]
        x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).half().cuda()
        dev = Linear(wt.to(gpu))
        plan = gpu.plan_for(dev.schedule(Tensor.from_data(np.zeros((1, rows, k), np.float32), gpu, F16)).op.desc)
        cases.append((dev, plan, x, torch.zeros(rows, vals.shape[0], dtype=torch.half, device="cuda"), vals))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def launch(case, stream):
        dev, plan, x, out, _ = case
        _lib.check(lib.rt_matmul_launch(plan, dev.w.ptr, x.data_ptr(), None, out.data_ptr(), stream.cuda_stream))

    def right(case):
        _, _, x, out, vals = case
        v = x.double().cpu().numpy()
        y = v @ vals.T
        assert np.all(np.abs(out.double().cpu().numpy() - y) <= error_bound(F16, vals, v, y))

    for _ in range(20):
        for case, stream in zip(cases, streams):
            launch(case, stream)
    torch.cuda.synchronize()
    for case in cases:
        right(case)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for case in cases:
            launch(case, torch.cuda.current_stream())
    for _ in range(3):
        for case in cases:
            case[2].normal_()
        graph.replay()
        torch.cuda.synchronize()
        for case in cases:
            right(case)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 12, 40, 130])
def test_a_weight_per_batch_with_any_number_of_rows(rows, gpu):
    w, wv = weight(G64, (3, 130, 320), 51)
    x = activations(F16, (3, rows, 320), 52)
    y = np.einsum("bmk,bnk->bnm", wv, x.astype(np.float64))
    e = np.stack([error_bound(F16, wv[b], x[b].astype(np.float64), y[b], rounded_weights=True) for b in range(3)])
    got = w.to(gpu).gemm(Tensor.from_data(x, gpu, F16), None, False, True, True).resolve().to(Device.CPU).to_f32()
    assert np.all(np.abs(got - y) <= e)


@pytest.mark.gpu
def test_a_weight_whose_offsets_pass_32_bits(gpu):
    """1.7 million rows of 2560: 4.4 thousand million values; rows from all over it."""
    import torch
    m, k = 1_700_003, 2560
    lib, parts = _lib.load(), G128.segments(m * k)
    buf = torch.zeros(G128.nbytes(m * k), dtype=torch.uint8, device="cuda")
    codes, scales, zeros = (buf[at:at + n] for (at, _), n in zip(parts, (m * k // 2, m * k // 64, m * k // 128)))
    gen = torch.Generator(device="cuda").manual_seed(53)
    codes.random_(0, 256, generator=gen), zeros.random_(0, 16, generator=gen)
    scales.view(torch.half).uniform_(0.005, 0.02, generator=gen)
    pick = np.unique(np.concatenate([np.arange(20), np.arange(m - 20, m), np.random.default_rng(54).integers(0, m, 200), [m * 5 // 8 + i for i in range(20)]]))
    at = torch.from_numpy(pick).cuda()
    q = codes.view(m, k // 2)[at].cpu().numpy()
    wv = values(G128, np.stack([q & 15, q >> 4], -1).reshape(len(pick), k), scales.view(torch.half).view(m, k // 128)[at].cpu().numpy(), zeros.view(m, k // 128)[at].cpu().numpy())
    for rows in (1, 4):
        x = activations(F16, (1, rows, k), 55)
        xg = torch.from_numpy(x).half().cuda()
        out = torch.zeros(rows, m, dtype=torch.half, device="cuda")
        plan = gpu.plan_for(Linear(Tensor((m, k), G128, gpu)).schedule(Tensor((1, rows, k), F16, gpu)).op.desc)
        torch.cuda.synchronize()
        _lib.check(lib.rt_matmul_launch(plan, buf.data_ptr(), xg.data_ptr(), None, out.data_ptr(), None))
        gpu.sync()
        y = x[0].astype(np.float64) @ wv.T
        kernel = lib.rt_plan_kernel(plan).decode()
        assert "q4_group_gemv" in kernel and np.all(np.abs(out[:, at].double().cpu().numpy() - y) <= error_bound(F16, wv, x[0].astype(np.float64), y)), kernel
