"""What stands around the Linears of a decode step: residual norms and log probabilities, against 64-bit arithmetic."""
import ctypes

import numpy as np
import pytest

import ratchet_b200 as rb
from ratchet_b200 import Device, DType, Executable, LayerNorm, Linear, MLP, Quantizer, RatchetError, ResidualNorm, RMSNorm, ShapeError, Tensor
from ratchet_b200 import _lib
from util import round_to

F16, BF16, F32, I32, U32 = DType.F16, DType.BF16, DType.F32, DType.I32, DType.U32
HALF_STEP = {F16: 2.0**-11, BF16: 2.0**-8, F32: 2.0**-24}
TINY = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}  # half the smallest subnormal
E24 = 2.0**-24
KINDS = {None: _lib.RT_NORM_NONE, "rms": _lib.RT_NORM_RMS, "layer": _lib.RT_NORM_LAYER}

# ------------------------------------------------------------------------------------------------ CPU: layouts and refusals


def test_structs_have_the_layout_the_ctypes_mirror_assumes():
    buf = (ctypes.c_uint64 * 64)()
    n = _lib.load().rt_abi_layout_steps(buf, 64)
    S, L = ctypes.sizeof, _lib
    off = lambda t, *names: [getattr(t, f).offset for f in names]  # noqa: E731
    want = [S(L.rt_norm), *off(L.rt_norm, "weight"), S(L.rt_residual_norm), *off(L.rt_residual_norm, "rows", "gate", "post", "h", "x_ld"),
            S(L.rt_log_probs), *off(L.rt_log_probs, "rows", "logits", "top_log_prob"), S(L.rt_step), *off(L.rt_step, "matmul", "norm", "log_probs")]
    assert [int(buf[i]) for i in range(n)] == want


BASE = 1 << 20  # addresses for descriptions that are only checked


def norm_op(**kw):
    p = _lib.rt_residual_norm()
    p.dt, p.residual_scale, p.block_scale, p.rows, p.d = _lib.RT_F16, 1, 1, 4, 64
    p.residual, p.block, p.h, p.x = BASE, 2 * BASE, 3 * BASE, 4 * BASE
    p.residual_ld = p.block_ld = p.h_ld = p.x_ld = 64
    p.gate_rows = 1
    p.pre.kind, p.pre.dt, p.pre.eps, p.pre.weight = _lib.RT_NORM_RMS, _lib.RT_F16, 1e-5, 5 * BASE
    for k, v in kw.items():
        at, name = (getattr(p, k.split("__")[0]), k.split("__")[1]) if "__" in k else (p, k)
        setattr(at, name, v)
    return p


def check_norm(**kw):
    return _lib.load().rt_residual_norm_check(ctypes.byref(norm_op(**kw)))


def test_residual_norm_refusals():
    ok, arg, shape, dtype, invariant = _lib.RT_OK, _lib.RT_ERR_ARG, _lib.RT_ERR_SHAPE, _lib.RT_ERR_DTYPE, _lib.RT_ERR_INVARIANT
    assert check_norm() == ok and check_norm(rows=0) == ok
    assert check_norm(dt=99) == arg and check_norm(dt=_lib.RT_I32) == dtype and check_norm(dt=_lib.RT_Q8_0H) == dtype
    assert check_norm(rows=-1) == shape and check_norm(d=0) == shape and check_norm(rows=1 << 31) == shape
    assert check_norm(d=32769, residual_ld=32769, block_ld=32769, h_ld=32769, x_ld=32769) == _lib.RT_ERR_UNSUPPORTED
    assert check_norm(residual=None) == ok and check_norm(block=None) == ok and check_norm(residual=None, block=None) == arg
    assert check_norm(block=None, gate=6 * BASE) == arg and check_norm(block=None, post__kind=_lib.RT_NORM_RMS) == arg
    assert check_norm(h=None) == ok and check_norm(x=None) == arg and check_norm(pre__kind=_lib.RT_NORM_NONE) == arg
    assert check_norm(x=None, pre__kind=_lib.RT_NORM_NONE) == ok and check_norm(x=None, h=None, pre__kind=_lib.RT_NORM_NONE) == arg
    assert check_norm(pre__kind=7) == arg and check_norm(pre__eps=-1.0) == arg and check_norm(pre__eps=float("nan")) == arg
    assert check_norm(pre__eps=float("inf")) == arg and check_norm(pre__eps=0.0) == ok
    assert check_norm(pre__dt=_lib.RT_F32) == ok and check_norm(pre__dt=_lib.RT_BF16) == dtype and check_norm(pre__dt=55) == dtype
    assert check_norm(pre__weight=None, pre__dt=55) == ok  # nothing to read
    assert check_norm(pre__bias=6 * BASE) == arg and check_norm(pre__bias=6 * BASE, pre__kind=_lib.RT_NORM_LAYER) == ok
    for ld in ("residual_ld", "block_ld", "h_ld", "x_ld"):
        assert check_norm(**{ld: 63}) == shape and check_norm(**{ld: 65}) == ok
    for name in ("residual", "block", "h", "x", "gate"):
        assert check_norm(**{name: 6 * BASE + 1}) == arg
    assert check_norm(pre__weight=6 * BASE + 1) == arg
    assert check_norm(gate=6 * BASE, gate_rows=2) == ok and check_norm(gate=6 * BASE, gate_rows=3) == shape
    assert check_norm(gate=6 * BASE, gate_rows=0) == shape
    # in place is allowed, any other overlap is not
    assert check_norm(h=BASE) == ok and check_norm(h=2 * BASE, x=BASE) == ok
    assert check_norm(h=BASE, h_ld=65) == invariant and check_norm(h=BASE + 2) == invariant and check_norm(h=3 * BASE, x=3 * BASE) == invariant
    assert check_norm(x=5 * BASE) == invariant and check_norm(gate=6 * BASE, h=6 * BASE) == invariant
    # two windows of one wider matrix interleave without touching, one value closer they touch
    wide = dict(residual_ld=130, block_ld=130, h_ld=130, x_ld=130)
    assert check_norm(residual=BASE, block=BASE + 128, h=3 * BASE, x=3 * BASE + 130, **wide) == ok
    assert check_norm(h=3 * BASE, x=3 * BASE + 126, **wide) == invariant
    assert check_norm(h=3 * BASE, x=3 * BASE + 134, **wide) == invariant


def lp_op(**kw):
    p = _lib.rt_log_probs()
    p.dt, p.top, p.rows, p.vocab, p.ld = _lib.RT_F16, 5, 4, 1000, 1000
    p.logits, p.tokens, p.log_prob, p.entropy, p.top_ids, p.top_log_prob = (BASE * i for i in range(1, 7))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_log_probs_refusals():
    check = lambda **kw: _lib.load().rt_log_probs_check(ctypes.byref(lp_op(**kw)))  # noqa: E731
    ok, arg, shape, invariant = _lib.RT_OK, _lib.RT_ERR_ARG, _lib.RT_ERR_SHAPE, _lib.RT_ERR_INVARIANT
    assert check() == ok and check(rows=0) == ok
    assert check(dt=99) == arg and check(dt=_lib.RT_U32) == _lib.RT_ERR_DTYPE
    assert check(rows=-1) == shape and check(vocab=0) == shape and check(ld=999) == shape and check(ld=1001) == ok
    assert check(top=-1) == shape and check(vocab=4) == shape and check(top=33) == _lib.RT_ERR_UNSUPPORTED and check(top=32) == ok
    assert check(logits=None) == arg and check(tokens=None) == arg and check(log_prob=None) == arg
    assert check(tokens=None, log_prob=None) == ok and check(entropy=None) == ok and check(top_ids=None) == arg and check(top=0) == arg
    none = dict(top=0, top_ids=None, top_log_prob=None)
    assert check(**none) == ok and check(entropy=None, tokens=None, log_prob=None, **none) == arg
    assert check(logits=BASE + 1) == arg and check(entropy=9 * BASE + 2) == arg and check(tokens=9 * BASE + 2) == arg
    assert check(entropy=BASE + 4) == invariant and check(entropy=3 * BASE) == invariant and check(top_ids=6 * BASE) == invariant
    assert check(log_prob=2 * BASE) == invariant


def test_graph_nodes_check_their_operands():
    t = lambda *shape, dt=F16: Tensor.from_data(np.zeros(shape), dt=dt)  # noqa: E731
    norm = RMSNorm(t(64))
    x = norm.schedule(t(2, 3, 64))
    assert x.shape == [2, 3, 64] and x.dt == F16 and not x.resolved()
    h, x = ResidualNorm(norm, LayerNorm(t(64), t(64)), 0.5, 2.0).schedule(t(2, 3, 64), t(2, 3, 64), t(2, 1, 64))
    assert h.shape == x.shape == [2, 3, 64] and h.op is x.op
    assert ResidualNorm(None).schedule(t(4, 64), t(4, 64))[1] is None
    for bad in (t(3, 1, 64), t(2, 3, 1), t(1, 3, 64), t(2, 64), t(32)):
        with pytest.raises(ShapeError):
            ResidualNorm(norm).schedule(t(2, 3, 64), t(2, 3, 64), bad)
    for gate in (t(64), t(1, 1, 64), t(2, 1, 64), t(2, 3, 64)):
        ResidualNorm(norm).schedule(t(2, 3, 64), t(2, 3, 64), gate)
    with pytest.raises(ShapeError):
        norm.schedule(t(2, 32))
    with pytest.raises(ShapeError):
        ResidualNorm(norm).schedule(t(2, 64), t(3, 64))
    with pytest.raises(RatchetError):
        ResidualNorm(norm).schedule(t(2, 64), t(2, 64, dt=F32))
    with pytest.raises(RatchetError):
        norm.schedule(t(2, 64, dt=I32))
    with pytest.raises(RatchetError):
        LayerNorm(t(64), t(64, dt=F32))
    lp = t(2, 3, 100).log_probs(t(2, 3, dt=I32), top=7)
    assert [v.shape for v in lp] == [[2, 3], [2, 3], [2, 3, 7], [2, 3, 7]] and [v.dt for v in lp] == [F32, F32, I32, F32]
    assert t(5, 100).log_probs().log_prob is None and t(5, 100).log_probs().top_ids is None
    for bad in (dict(top=-1), dict(top=101), dict(tokens=t(4, dt=I32))):
        with pytest.raises(ShapeError):
            t(5, 100).log_probs(**bad)
    for bad in (dict(top=33), dict(tokens=t(5, dt=F32))):
        with pytest.raises(RatchetError):
            t(5, 100).log_probs(**bad)
    with pytest.raises(RatchetError):  # host operands: refused before anything is launched
        norm.schedule(t(2, 64)).resolve()


# ------------------------------------------------------------------------------------------------ GPU: norms

#: what an f32 sum over a row may lose of the sum of its magnitudes: a thread adds at most 32 values, then trees of 5 and 5
SUM = 48 * E24


def normed(v, e, kind, w, b, eps):
    """N(v) in 64 bits, and how far f32 arithmetic may be off when v itself is off by at most e."""
    if kind is None:
        return v, e
    if kind == "layer":
        mean = v.mean(-1, keepdims=True)
        c = v - mean
        e = e + e.mean(-1, keepdims=True) + SUM * np.abs(v).mean(-1, keepdims=True) + E24 * (np.abs(v) + np.abs(mean))
    else:
        c = v
    var = (c * c).mean(-1, keepdims=True) + eps
    off = SUM + 4 * E24 + (2 * (np.abs(c) * e).mean(-1, keepdims=True) + (e * e).mean(-1, keepdims=True)) / var  # of var, relative
    y = c / np.sqrt(var)
    ey = e / np.sqrt(var) + np.abs(y) * (0.6 * off + 4 * E24)
    y, ey = y * w, ey * np.abs(w) + E24 * np.abs(y * w)
    return y + b, ey + E24 * np.abs(y + b)


def norm_truth(r, y, gate, post, pre, a, bs):
    v = np.zeros_like(r if y is None else y)
    e = 0 * v
    if y is not None:
        v, e = normed(y, e, *post)
        g = 1.0 if gate is None else gate
        v, e = bs * g * v, np.abs(bs * g) * e + 3 * E24 * np.abs(bs * g * v)
    if r is not None:
        v, e = a * r + v, e + E24 * (np.abs(a * r) + np.abs(a * r + v)) + E24 * np.abs(v)
    return (v, e), normed(v, e, *pre)


def close(got, truth, dt):
    want, e = truth
    return np.abs(got - want) <= e + HALF_STEP[dt] * (np.abs(want) + e) * (1 + 2.0**-20) + TINY[dt]


def norm_weights(kind, d, dt, rng):
    if kind is None:
        return None, (None, 1.0, 0.0, 0.0)
    w = round_to(dt, (1 + 0.3 * rng.standard_normal(d)).astype(np.float32))
    b = round_to(dt, (0.3 * rng.standard_normal(d)).astype(np.float32)) if kind == "layer" else None
    eps = 1e-5
    return (w, b, eps), (kind, w.astype(np.float64), 0.0 if b is None else b.astype(np.float64), np.float64(np.float32(eps)))


def norm_module(kind, p, gpu, dt):
    if kind is None:
        return None
    t = lambda v: Tensor.from_data(v, gpu, dt)  # noqa: E731
    return RMSNorm(t(p[0]), p[2]) if kind == "rms" else LayerNorm(t(p[0]), t(p[1]), p[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("post,pre", [(None, "rms"), (None, "layer"), ("rms", "rms"), ("layer", "layer"), ("rms", None)])
def test_residual_norm_over_widths(dt, post, pre, gpu):
    """One value, odd widths, both sides of a warp's, of every thread count's and of the two access widths' limits."""
    for i, d in enumerate([1, 2, 7, 8, 31, 64, 127, 256, 257, 384, 511, 512, 513, 520, 1000, 1024, 2047, 2048, 2056, 2560, 2561, 4095, 4096, 4104, 8192, 8200,
                           8193, 16384, 16392, 32760, 32768, 32767]):
        rows = [1, 3, 9][i % 3]
        rng = np.random.default_rng(1000 + d)
        r, y = (round_to(dt, (s * rng.standard_normal((rows, d))).astype(np.float32)) for s in (3.0, 1.0))
        gate = round_to(dt, rng.uniform(-1, 1, d).astype(np.float32)) if i % 2 else None
        pp, post_t = norm_weights(post, d, dt, rng)
        qq, pre_t = norm_weights(pre, d, F32 if i % 4 == 3 else dt, rng)
        a, b = (1.0, 0.5) if i % 2 else (0.75, -1.25)
        mod = ResidualNorm(norm_module(pre, qq, gpu, F32 if i % 4 == 3 else dt), norm_module(post, pp, gpu, dt), a, b)
        h, x = mod.schedule(Tensor.from_data(r, gpu, dt), Tensor.from_data(y, gpu, dt), None if gate is None else Tensor.from_data(gate, gpu, dt))
        f64 = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
        th, tx = norm_truth(f64(r), f64(y), f64(gate), post_t, pre_t, a, b)
        assert np.all(close(h.resolve().to(Device.CPU).to_f32(), th, dt)), (d, "h")
        if x is not None:
            assert np.all(close(x.resolve().to(Device.CPU).to_f32(), tx, dt)), (d, "x")
        if post is None and pre is not None:  # the norm alone
            alone = mod.pre.schedule(Tensor.from_data(r, gpu, dt)).resolve().to(Device.CPU).to_f32()
            assert np.all(close(alone, normed(f64(r), 0 * f64(r), *pre_t), dt)), (d, "alone")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("gate_shape", [(1, 1), (3, 1), (3, 5)])
def test_gates_per_sequence_and_per_row(dt, gate_shape, gpu):
    rng, d = np.random.default_rng(5), 96
    r, y = (round_to(dt, rng.standard_normal((3, 5, d)).astype(np.float32)) for _ in range(2))
    gate = round_to(dt, rng.standard_normal((*gate_shape, d)).astype(np.float32))
    p, pre = norm_weights("rms", d, dt, rng)
    h, x = ResidualNorm(norm_module("rms", p, gpu, dt)).schedule(*(Tensor.from_data(v, gpu, dt) for v in (r, y, gate)))
    th, tx = norm_truth(*(v.astype(np.float64) for v in (r, y, gate)), (None, 1.0, 0.0, 0.0), pre, 1.0, 1.0)
    assert np.all(close(h.resolve().to(Device.CPU).to_f32(), th, dt)) and np.all(close(x.resolve().to(Device.CPU).to_f32(), tx, dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_rows_a_long_way_from_zero_constant_rows_and_zeros(dt, gpu):
    """Cancellation: a spread of 1 around 1000; a constant row (nothing but eps under the root); a row of zeros."""
    rng, d = np.random.default_rng(6), 768
    v = np.zeros((4, d), np.float32)
    v[0], v[1], v[3] = 1000 + rng.standard_normal(d), 17.0, 1e-3 * rng.standard_normal(d)
    v = round_to(dt, v)
    for kind in ("rms", "layer"):
        p, t = norm_weights(kind, d, dt, rng)
        got = norm_module(kind, p, gpu, dt).schedule(Tensor.from_data(v, gpu, dt)).resolve().to(Device.CPU).to_f32()
        assert np.all(close(got, normed(v.astype(np.float64), 0 * v.astype(np.float64), *t), dt)), kind


@pytest.mark.gpu
def test_norms_keep_what_is_not_finite_in_its_row(gpu):
    rng, d = np.random.default_rng(7), 300
    r, y = rng.standard_normal((2, 6, d)).astype(np.float32)
    w = Tensor.from_data(np.ones(d, np.float32), gpu)
    mod = ResidualNorm(LayerNorm(w), RMSNorm(w))
    run = lambda: [t.resolve().to(Device.CPU).to_f32() for t in mod.schedule(Tensor.from_data(r, gpu), Tensor.from_data(y, gpu))]  # noqa: E731
    clean = run()
    r[1, 7], y[4, 299] = np.inf, np.nan
    bad = run()
    for c, b in zip(clean, bad):
        assert np.array_equal(c[[0, 2, 3, 5]], b[[0, 2, 3, 5]])
    assert bad[0][1, 7] == np.inf and np.isnan(bad[0][4]).all() and np.isnan(bad[1][[1, 4]]).all()


def device_array(gpu, a):
    buf = rb.GpuBuffer(gpu, a.nbytes)
    _lib.check(_lib.load().rt_upload(gpu._h, buf._h, 0, a.ctypes.data, a.nbytes, 1))
    return buf


def read_back(gpu, buf, like):
    out = np.empty_like(like)
    _lib.check(_lib.load().rt_download(gpu._h, buf._h, 0, out.ctypes.data, out.nbytes, 1))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("d,ld,shift", [(64, 72, 0), (64, 67, 0), (40, 67, 3), (384, 1160, 8)])
def test_strided_rows_in_place_and_windows_of_one_matrix(d, ld, shift, gpu):
    """Rows ld apart, off a 16-byte boundary; h over the residual, x over the block; nothing between the rows is touched."""
    rng, rows = np.random.default_rng(8), 11
    mats = [rng.standard_normal(rows * ld + shift).astype(np.float32) for _ in range(2)]
    bufs = [device_array(gpu, m) for m in mats]
    w = device_array(gpu, np.ones(d, np.float32))
    p = _lib.rt_residual_norm()
    p.dt, p.residual_scale, p.block_scale, p.rows, p.d = _lib.RT_F32, 0.5, 2.0, rows, d
    p.residual, p.block = bufs[0].ptr + 4 * shift, bufs[1].ptr + 4 * shift
    p.h, p.x = p.residual, p.block
    p.residual_ld = p.block_ld = p.h_ld = p.x_ld = ld
    p.pre.kind, p.pre.dt, p.pre.eps, p.pre.weight = _lib.RT_NORM_RMS, _lib.RT_F32, 0.0, w.ptr
    _lib.check(_lib.load().rt_residual_norm_launch(gpu._h, ctypes.byref(p), None))
    got = [read_back(gpu, b, m) for b, m in zip(bufs, mats)]
    at = (shift + np.arange(rows)[:, None] * ld + np.arange(d)[None, :]).reshape(-1)
    r, y = (m[at].reshape(rows, d).astype(np.float64) for m in mats)
    truths = norm_truth(r, y, None, (None, 1.0, 0.0, 0.0), ("rms", np.ones(d), 0.0, 0.0), 0.5, 2.0)
    for g, m, t in zip(got, mats, truths):
        assert np.all(close(g[at].reshape(rows, d), t, F32))
        rest = np.ones(m.size, bool)
        rest[at] = False
        assert np.array_equal(g[rest], m[rest])


@pytest.mark.gpu
def test_norms_of_no_rows_and_of_many(gpu):
    w = Tensor.from_data(np.ones(24, np.float32), gpu)
    assert RMSNorm(w).schedule(Tensor.from_data(np.zeros((0, 24), np.float32), gpu)).resolve().shape == [0, 24]
    v = np.random.default_rng(9).standard_normal((70001, 24)).astype(np.float32)
    got = RMSNorm(w, 1e-6).schedule(Tensor.from_data(v, gpu)).resolve().to(Device.CPU).to_f32()
    assert np.all(close(got, normed(v.astype(np.float64), 0 * v.astype(np.float64), "rms", 1.0, 0.0, np.float64(np.float32(1e-6))), F32))


#: (d, sequences, rows of one): more rows than are on the GPU at once, both sides of a warp's, of a team's and of the teams' largest width
MANY_ROWS = [(7, 2, 1500), (8, 3, 1700), (9, 1, 5000), (100, 4, 1000), (383, 3, 1001), (384, 2, 1500), (512, 5, 500), (513, 1, 2000), (520, 4, 400), (1000, 3, 301),
             (2560, 7, 100), (2561, 2, 351), (4104, 1, 333), (5001, 3, 67), (8191, 2, 75), (8192, 1, 151), (8193, 1, 77), (9001, 2, 40), (10240, 3, 33), (10248, 1, 50)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("post,pre", [("rms", "rms"), ("layer", "layer"), (None, "layer"), ("rms", None)])
def test_residual_norm_of_many_rows(dt, post, pre, gpu):
    f64 = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    for i, (d, sequences, rows) in enumerate(MANY_ROWS):
        rng = np.random.default_rng(2000 + d)
        r, y = (round_to(dt, (s * rng.standard_normal((sequences, rows, d), dtype=np.float32))) for s in (3.0, 1.0))
        gate = round_to(dt, rng.uniform(-1, 1, [(sequences, 1, d), (d,)][i % 2]).astype(np.float32)) if i % 3 else None
        pp, post_t = norm_weights(post, d, F32 if i % 4 == 3 else dt, rng)
        qq, pre_t = norm_weights(pre, d, dt, rng)
        mod = ResidualNorm(norm_module(pre, qq, gpu, dt), norm_module(post, pp, gpu, F32 if i % 4 == 3 else dt), 0.75, -1.25)
        h, x = mod.schedule(*(None if v is None else Tensor.from_data(v, gpu, dt) for v in (r, y, gate)))
        th, tx = norm_truth(f64(r), f64(y), f64(gate), post_t, pre_t, 0.75, -1.25)
        assert np.all(close(h.resolve().to(Device.CPU).to_f32(), th, dt)), (d, "h")
        if x is not None:
            assert np.all(close(x.resolve().to(Device.CPU).to_f32(), tx, dt)), (d, "x")
        if post is None:
            alone = mod.pre.schedule(Tensor.from_data(r, gpu, dt)).resolve().to(Device.CPU).to_f32()
            assert np.all(close(alone, normed(f64(r), 0 * f64(r), *pre_t), dt)), (d, "alone")


@pytest.mark.gpu
@pytest.mark.parametrize("d,ld,shift,rows", [(64, 72, 0, 4001), (64, 67, 1, 4001), (9, 9, 3, 6000), (9, 16, 0, 6000), (384, 1160, 8, 2500), (1001, 1001, 0, 900), (1001, 1003, 5, 900),
                                             (1000, 1003, 0, 900), (2560, 2560, 0, 400)])
def test_many_strided_rows_in_place(d, ld, shift, rows, gpu):
    """h over the block, x over the residual, while later rows are on their way; nothing between, before or behind the rows is touched."""
    rng = np.random.default_rng(18)
    for kind in (_lib.RT_NORM_RMS, _lib.RT_NORM_LAYER):
        mats = [round_to(F16, rng.standard_normal(rows * ld + shift + 11).astype(np.float32)).astype(np.float16) for _ in range(2)]
        bufs = [device_array(gpu, m) for m in mats]
        w = device_array(gpu, np.ones(d, np.float16))
        p = _lib.rt_residual_norm()
        p.dt, p.residual_scale, p.block_scale, p.rows, p.d = _lib.RT_F16, 0.5, 2.0, rows, d
        p.residual, p.block = bufs[0].ptr + 2 * shift, bufs[1].ptr + 2 * shift
        p.h, p.x = p.block, p.residual
        p.residual_ld = p.block_ld = p.h_ld = p.x_ld = ld
        p.pre.kind, p.pre.dt, p.pre.eps, p.pre.weight = kind, _lib.RT_F16, 1e-5, w.ptr
        _lib.check(_lib.load().rt_residual_norm_launch(gpu._h, ctypes.byref(p), None))
        x, h = [read_back(gpu, b, m) for b, m in zip(bufs, mats)]
        at = (shift + np.arange(rows)[:, None] * ld + np.arange(d)[None, :]).reshape(-1)
        r, y = (m[at].reshape(rows, d).astype(np.float64) for m in mats)
        truths = norm_truth(r, y, None, (None, 1.0, 0.0, 0.0), ("rms" if kind == _lib.RT_NORM_RMS else "layer", np.ones(d), 0.0, np.float64(np.float32(1e-5))), 0.5, 2.0)
        for g, m, t in zip((h, x), (mats[1], mats[0]), truths):
            assert np.all(close(g[at].reshape(rows, d).astype(np.float32), t, F16)), kind
            rest = np.ones(m.size, bool)
            rest[at] = False
            assert np.array_equal(g[rest], m[rest])


@pytest.mark.gpu
def test_what_is_not_finite_stays_in_its_row_of_many(gpu):
    rng = np.random.default_rng(19)
    for d in (300, 304, 1203):
        r, y = rng.standard_normal((2, 3000, d)).astype(np.float32)
        w = Tensor.from_data(np.ones(d, np.float32), gpu)
        for mod in (ResidualNorm(LayerNorm(w), RMSNorm(w)), ResidualNorm(RMSNorm(w))):
            run = lambda a, b: [t.resolve().to(Device.CPU).to_f32() for t in mod.schedule(Tensor.from_data(a, gpu), Tensor.from_data(b, gpu))]  # noqa: E731
            clean = run(r, y)
            r2, y2 = r.copy(), y.copy()
            bad = np.array([0, 7, 8, 1501, 2999])
            r2[bad[:3], d - 1], y2[bad[3:], 2] = np.inf, np.nan
            rest = np.delete(np.arange(3000), bad)
            for c, b in zip(clean, run(r2, y2)):
                assert np.array_equal(c[rest], b[rest]) and not np.isfinite(b[bad]).all(-1).any()


# ------------------------------------------------------------------------------------------------ GPU: log probabilities

def lp_truth(v):
    """log p, entropy (64 bits) and the order of each row; what f32 sums may lose of ln S and of the entropy."""
    v = v.astype(np.float64)
    m = v.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = v - m
        e = np.exp(d)
        s = e.sum(-1, keepdims=True)
        logp = d - np.log(s)
        p = e / s
        ent = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(-1)
        nothing = np.isneginf(m[..., 0])
    logp[nothing], ent[nothing] = -np.inf, 0.0
    order = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), -v), axis=-1)
    dd = np.where(p > 0, d, 0)
    # a term is off by the rounding of its exponent (|d| steps) and of the exponential (4); a thread adds at most a few hundred
    # terms before the trees
    steps = (v.shape[1] / 256 + 64) * E24
    loss = steps * (1 + (p * np.abs(dd)).sum(-1))
    ent_loss = steps * (2 + 2 * (p * np.abs(dd)).sum(-1) + (p * dd * dd).sum(-1)) + 4 * E24 * np.abs(np.log(s[..., 0]))
    return logp, ent, order, np.nan_to_num(loss), np.nan_to_num(ent_loss)


def lp_check(v, tokens, top, gpu, dt):
    lp = Tensor.from_data(v, gpu, dt).log_probs(None if tokens is None else Tensor.from_data(np.asarray(tokens, np.int32), gpu), top)
    lp.entropy.resolve()
    got = [None if t is None else t.resolve().to(Device.CPU).to_numpy() for t in lp]
    logp, ent, order, loss, ent_loss = lp_truth(v)
    near = lambda g, w, e: (g == w) | (np.abs(g - w) <= e + 4 * E24 * np.abs(w) + 1e-37)  # noqa: E731
    rows = np.arange(len(v))
    with np.errstate(invalid="ignore"):
        if tokens is not None:
            want = logp[rows, tokens]
            assert np.all(near(got[0], want, loss)), ("log_prob", got[0] - want)
        assert np.all(near(got[1], ent, ent_loss)), ("entropy", got[1] - ent)
        if top:
            assert np.array_equal(got[2], order[:, :top])
            assert np.all(near(got[3], np.take_along_axis(logp, order[:, :top], 1), loss[:, None]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 100, 511, 1000, 4096, 5003, 51865, 131072, 200003])
def test_log_probs_over_vocabularies(dt, vocab, gpu):
    """Rows of ordinary logits (16-bit ones repeat values: ties), from one token to more than any model has."""
    for rows, top in ((1, 5), (3, 20), (2, 32), (4, 1), (2, 0)):
        rng = np.random.default_rng(vocab + rows)
        v = round_to(dt, (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32))
        tokens = rng.integers(0, vocab, rows)
        lp_check(v, tokens if rows != 4 else None, min(top, vocab), gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 17, 64, 150, 400, 1500])
def test_log_probs_over_row_counts(rows, gpu):
    rng = np.random.default_rng(rows)
    v = round_to(BF16, (3 * rng.standard_normal((rows, 3001))).astype(np.float32))
    lp_check(v, rng.integers(0, 3001, rows), 7, gpu, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_log_probs_of_masked_rows(dt, gpu):
    """-inf and the type's lowest value as masks, one token left, none left, all equal, one far ahead, both zeros."""
    rng, vocab = np.random.default_rng(11), 3000
    lowest = {F16: -65504.0, BF16: -3.3895313892515355e38, F32: -3.4028234663852886e38}[dt]
    v = round_to(dt, rng.standard_normal((10, vocab)).astype(np.float32))
    v[0, rng.random(vocab) < 0.9] = -np.inf
    v[1, rng.random(vocab) < 0.9] = lowest
    v[2], v[2, 1234] = -np.inf, -7.0
    v[3] = -np.inf
    v[4], v[4, 2999] = lowest, lowest
    v[5] = 0.0
    v[6], v[6, ::3] = 0.0, -0.0
    v[7, 17] = 1000.0
    v[8], v[8, 5] = -np.inf, lowest
    v[9] = np.sort(v[9])[::-1]
    lp_check(v, rng.integers(0, vocab, 10), 20, gpu, dt)
    lp_check(v, [17, 0, 1234, 5, 2999, 1, 0, 17, 5, 2999], 32, gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, F32])
def test_orders_that_pile_the_likeliest_tokens_together(dt, gpu):
    """Everything near the top in one stretch, in one thread's stride, at the end, rising, falling, and few distinct values."""
    rng, vocab = np.random.default_rng(12), 40000
    v = round_to(dt, rng.standard_normal((9, vocab)).astype(np.float32))
    v[0, 100:164] += 20
    v[1, 3::4096] += 20
    v[2, -40:] += 20
    v[3], v[4] = np.sort(v[3]), np.sort(v[4])[::-1]
    v[5] = rng.integers(0, 3, vocab)
    v[6, 8::512] += 20
    v[7, :] = 1.0
    v[8, 0::2048], v[8, 1::2048] = 30.0, 30.0
    lp_check(round_to(dt, v), rng.integers(0, vocab, 9), 32, gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_nan_and_plus_infinity_stay_in_their_rows(dt, gpu):
    rng, vocab = np.random.default_rng(13), 2000
    v = round_to(dt, rng.standard_normal((5, vocab)).astype(np.float32))
    tokens = Tensor.from_data(rng.integers(0, vocab, 5).astype(np.int32), gpu)
    run = lambda: [t.resolve().to(Device.CPU).to_numpy() for t in Tensor.from_data(v, gpu, dt).log_probs(tokens, 4)]  # noqa: E731
    clean = run()
    v[1, 77], v[1, 1500], v[3, 1999], v[3, 5] = np.nan, np.inf, np.inf, np.inf
    bad = run()
    for c, b in zip(clean, bad):
        assert np.array_equal(c[[0, 2, 4]], b[[0, 2, 4]])
    for k in (0, 1, 3):
        assert np.isnan(bad[k][[1, 3]]).all()
    assert list(bad[2][1, :2]) == [77, 1500] and list(bad[2][3, :2]) == [5, 1999]


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary_and_u32_tokens(gpu):
    v = np.random.default_rng(14).standard_normal((5, 100)).astype(np.float32)
    logp = lp_truth(v)[0]
    got = Tensor.from_data(v, gpu).log_probs(Tensor.from_data(np.array([-1, 99, 100, 2**31 - 1, 0], np.int32), gpu)).log_prob
    got = got.resolve().to(Device.CPU).to_numpy()
    assert np.isnan(got[[0, 2, 3]]).all() and np.allclose(got[[1, 4]], logp[[1, 4], [99, 0]], atol=1e-6)
    got = Tensor.from_data(v, gpu).log_probs(Tensor.from_data(np.array([2**32 - 1, 99, 2**31, 3, 0], np.uint32), gpu)).log_prob
    got = got.resolve().to(Device.CPU).to_numpy()
    assert np.isnan(got[[0, 2]]).all() and np.allclose(got[[1, 3, 4]], logp[[1, 3, 4], [99, 3, 0]], atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("ld,shift", [(1003, 0), (1008, 0), (1003, 1), (2000, 5)])
@pytest.mark.parametrize("dt", [F16, F32])
def test_log_probs_of_strided_rows(dt, ld, shift, gpu):
    """Rows ld apart and off a 16-byte boundary; what lies behind a row is larger than anything in it."""
    rng, rows, vocab = np.random.default_rng(15), 6, 1003
    v = round_to(dt, rng.standard_normal((rows, vocab)).astype(np.float32))
    flat = np.full(shift + rows * ld, 100.0, np.float32)
    for r in range(rows):
        flat[shift + r * ld: shift + r * ld + vocab] = v[r]
    store = device_array(gpu, flat.astype(np.float16) if dt == F16 else flat)
    outs = [device_array(gpu, np.full((rows + 1, n), -1, t)) for n, t in ((1, np.float32), (1, np.float32), (9, np.int32), (9, np.float32))]
    p = _lib.rt_log_probs()
    p.dt, p.top, p.rows, p.vocab, p.ld = int(dt), 9, rows, vocab, ld
    tokens = device_array(gpu, np.arange(rows, dtype=np.int32))
    p.logits, p.tokens = store.ptr + shift * dt.size_of(), tokens.ptr
    p.log_prob, p.entropy, p.top_ids, p.top_log_prob = (b.ptr for b in outs)
    _lib.check(_lib.load().rt_log_probs_launch(gpu._h, ctypes.byref(p), None))
    got = [read_back(gpu, b, np.empty((rows + 1, n), t)) for b, (n, t) in zip(outs, ((1, np.float32), (1, np.float32), (9, np.int32), (9, np.float32)))]
    logp, ent, order, loss, ent_loss = lp_truth(v)
    assert np.all(np.abs(got[0][:rows, 0] - logp[np.arange(rows), np.arange(rows)]) <= loss + 4 * E24 * 10)
    assert np.all(np.abs(got[1][:rows, 0] - ent) <= ent_loss + 4 * E24 * 10) and np.array_equal(got[2][:rows], order[:, :9])
    assert all(np.all(g[rows] == -1) for g in got)  # behind the last row: left as it was


# ------------------------------------------------------------------------------------------------ GPU: together

def decode_step(gpu, rows, seed):
    """One feed-forward layer and the answer: x = N(r), MLP in 4 bits, (h, x) = residual norm, logits, log probabilities."""
    rng, d, ff, vocab = np.random.default_rng(seed), 256, 512, 1003
    q = lambda n, k, dt: Quantizer.q4_group_quantize(Tensor.from_data((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)), dt)  # noqa: E731
    w1, w2, head = q(2 * ff, d, DType.Q4_G64), q(d, ff, DType.Q4_G128), q(vocab, d, DType.Q4_G32)
    n1, n2, n3 = ((1 + 0.1 * rng.standard_normal(d)).astype(np.float16) for _ in range(3))
    r = (2 * rng.standard_normal((1, rows, d))).astype(np.float16)
    tokens = rng.integers(0, vocab, (1, rows)).astype(np.int32)
    t = lambda v: Tensor.from_data(v, gpu)  # noqa: E731
    rt = t(r)
    x = RMSNorm(t(n1)).schedule(rt)
    gate_up = Linear(w1.to(gpu), None, rb.EPILOGUE_SILU_MUL).schedule(x)
    y = Linear(w2.to(gpu)).schedule(gate_up)
    h, x2 = ResidualNorm(RMSNorm(t(n3)), RMSNorm(t(n2))).schedule(rt, y)
    logits = Linear(head.to(gpu)).schedule(x2)
    lp = logits.log_probs(t(tokens), 5)
    deq = [Quantizer.dequantize_bytes(w.storage, w.dt, w.numel()).reshape(w.shape).astype(np.float64) for w in (w1, w2, head)]
    rms = lambda v, w: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-5) * w.astype(np.float64)  # noqa: E731
    v = rms(r[0].astype(np.float64), n1) @ deq[0].T
    v = (v[:, :ff] / (1 + np.exp(-v[:, :ff])) * v[:, ff:]) @ deq[1].T
    hv = r[0].astype(np.float64) + rms(v, n2)
    lv = rms(hv, n3) @ deq[2].T
    return rt, [x, gate_up, y, h, x2, logits, *lp], hv, lv, tokens[0]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 16, 40])
def test_a_decode_step_lazily_and_as_one_executable(rows, gpu):
    rt, nodes, hv, lv, tokens = decode_step(gpu, rows, 20 + rows)
    nodes[-1].resolve()
    for t in nodes:
        t.resolve()
    read = lambda: [t.to(Device.CPU).to_f32() if t.dt == F16 else t.to(Device.CPU).to_numpy() for t in nodes]  # noqa: E731
    first = read()
    # f16 roundings: one per tensor on the way, each spread over a whole row by the products behind it
    assert np.linalg.norm(first[3][0] - hv) <= 4 * 2.0**-11 * np.linalg.norm(hv)
    assert np.linalg.norm(first[5][0] - lv) <= 6 * 2.0**-11 * np.linalg.norm(lv)
    logp, ent, order, _, _ = lp_truth(first[5][0])  # of the logits as they are
    assert np.allclose(first[6][0], logp[np.arange(rows), tokens], atol=1e-5) and np.allclose(first[7][0], ent, atol=1e-5)
    assert np.array_equal(first[8][0], order[:, :5])
    for graph in (False, True):
        exe = Executable(gpu, nodes, use_graph=graph)
        assert exe.launches >= 6 and exe.kernel == ("graph" if graph else "nodes")
        for _ in range(3):
            exe.dispatch()
        gpu.sync()
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(read(), first))
    # new input through the same executable: what a fresh graph gives for it
    other = decode_step(gpu, rows, 20 + rows)
    fresh = np.random.default_rng(99).standard_normal((1, rows, 256)).astype(np.float16)
    rt.write(fresh)
    exe.dispatch()
    gpu.sync()
    got = read()
    other[0].write(fresh)
    for t in other[1]:
        t.resolve()
    want = [t.to(Device.CPU).to_f32() if t.dt == F16 else t.to(Device.CPU).to_numpy() for t in other[1]]
    assert all(np.array_equal(a, b) for a, b in zip(got, want)) and not np.array_equal(got[5], first[5])


@pytest.mark.gpu
def test_nodes_with_several_outputs_are_launched_once(gpu):
    rng = np.random.default_rng(30)
    r, y = (Tensor.from_data(rng.standard_normal((4, 64)).astype(np.float32), gpu) for _ in range(2))
    h, x = ResidualNorm(RMSNorm(None)).schedule(r, y)
    x.resolve()
    assert x.resolved() and not h.resolved()
    before = h.op._buffers
    h.resolve()
    assert h.op._buffers is before and h.storage is before[0] and x.storage is before[1]
    exe = Executable(gpu, [h, x], use_graph=False)
    assert exe.launches == 1
    with pytest.raises(RatchetError):
        Executable(gpu, [ResidualNorm(None).schedule(r, y)[0]])
    with pytest.raises(RatchetError, match="operand on"):
        RMSNorm(Tensor.from_data(np.ones(64, np.float32))).schedule(r).resolve()


@pytest.mark.gpu
def test_calls_on_other_streams_and_in_a_captured_graph(gpu):
    """The C entries on a caller's stream: two at once, and captured once and replayed on changed inputs."""
    import torch
    rng, lib = np.random.default_rng(31), _lib.load()
    cases = []
    for seed in range(2):
        v = torch.randn(8, 5000, generator=torch.Generator().manual_seed(seed)).cuda()
        r, y = torch.randn(2, 33, 520, generator=torch.Generator().manual_seed(9 + seed)).cuda()
        outs = torch.zeros(8, device="cuda"), torch.zeros(8, 6, dtype=torch.int32, device="cuda"), torch.zeros(8, 6, device="cuda")
        h, x, w = torch.zeros_like(r), torch.zeros_like(r), torch.ones(520, device="cuda")
        p = _lib.rt_log_probs()
        p.dt, p.top, p.rows, p.vocab, p.ld, p.logits = _lib.RT_F32, 6, 8, 5000, 5000, v.data_ptr()
        p.entropy, p.top_ids, p.top_log_prob = (o.data_ptr() for o in outs)
        n = _lib.rt_residual_norm()
        n.dt, n.residual_scale, n.block_scale, n.rows, n.d = _lib.RT_F32, 1, 1, 33, 520
        n.residual, n.block, n.h, n.x, n.gate_rows = r.data_ptr(), y.data_ptr(), h.data_ptr(), x.data_ptr(), 1
        n.residual_ld = n.block_ld = n.h_ld = n.x_ld = 520
        n.pre.kind, n.pre.dt, n.pre.eps, n.pre.weight = _lib.RT_NORM_LAYER, _lib.RT_F32, 1e-5, w.data_ptr()
        cases.append((v, r, y, outs, h, x, p, n, w))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def launch(case, stream):
        _lib.check(lib.rt_log_probs_launch(gpu._h, ctypes.byref(case[6]), stream.cuda_stream))
        _lib.check(lib.rt_residual_norm_launch(gpu._h, ctypes.byref(case[7]), stream.cuda_stream))

    def right(case):
        v, r, y, outs, h, x = case[:6]
        logp, ent, order, _, ent_loss = lp_truth(v.cpu().numpy())
        assert np.all(np.abs(outs[0].cpu().numpy() - ent) <= ent_loss + 4 * E24 * 10) and np.array_equal(outs[1].cpu().numpy(), order[:, :6])
        hv = (r.double() + y.double()).cpu().numpy()
        assert np.all(close(x.cpu().numpy(), normed(hv, E24 * np.abs(hv), "layer", 1.0, 0.0, np.float64(np.float32(1e-5))), F32))

    for _ in range(20):
        for case, stream in zip(cases, streams):
            launch(case, stream)
    torch.cuda.synchronize()
    for case in cases:
        right(case)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(cases[0], torch.cuda.current_stream())
    for k in range(3):
        cases[0][0].normal_(generator=None).mul_(k + 1)
        cases[0][1].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        right(cases[0])
    del graph


@pytest.mark.gpu
def test_many_rows_on_two_streams_and_in_a_replayed_graph(gpu):
    """Teams that walk rows, two launches at once on one device, and a captured one on changed inputs."""
    import torch
    lib, cases = _lib.load(), []
    for d, rows in ((520, 3000), (1001, 1200)):
        r, y = torch.randn(2, rows, d, generator=torch.Generator().manual_seed(d)).cuda()
        w, h, x = torch.ones(d, device="cuda"), torch.zeros_like(r), torch.zeros_like(r)
        n = _lib.rt_residual_norm()
        n.dt, n.residual_scale, n.block_scale, n.rows, n.d, n.gate_rows = _lib.RT_F32, 1, 1, rows, d, 1
        n.residual, n.block, n.h, n.x = r.data_ptr(), y.data_ptr(), h.data_ptr(), x.data_ptr()
        n.residual_ld = n.block_ld = n.h_ld = n.x_ld = d
        n.pre.kind, n.pre.dt, n.pre.eps, n.pre.weight = _lib.RT_NORM_RMS, _lib.RT_F32, 1e-5, w.data_ptr()
        cases.append((r, y, h, x, n, w))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    launch = lambda case, stream: _lib.check(lib.rt_residual_norm_launch(gpu._h, ctypes.byref(case[4]), stream.cuda_stream))  # noqa: E731

    def right(case):
        r, y, h, x = case[:4]
        hv = (r.double() + y.double()).cpu().numpy()
        assert np.all(close(h.cpu().numpy(), (hv, 0 * hv), F32))
        assert np.all(close(x.cpu().numpy(), normed(hv, E24 * np.abs(hv), "rms", 1.0, 0.0, np.float64(np.float32(1e-5))), F32))

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
            case[0].normal_()
            case[1].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        for case in cases:
            right(case)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("d", [96, 520, 1003])
def test_many_gates(d, dt, gpu):
    """A gate per row, per seven rows and per sequence of many rows: a team's rows cross from one to the next."""
    rng = np.random.default_rng(51)
    r, y = (round_to(dt, rng.standard_normal((70, 7, 9, d), dtype=np.float32)) for _ in range(2))
    pre, pre_t = norm_weights("layer", d, dt, rng)
    post, post_t = norm_weights("rms", d, dt, rng)
    mod = ResidualNorm(norm_module("layer", pre, gpu, dt), norm_module("rms", post, gpu, dt))
    for shape in ((70, 7, 9, d), (70, 7, 1, d), (70, 1, 1, d), (1, 1, 1, d)):
        gate = round_to(dt, rng.standard_normal(shape, dtype=np.float32))
        h, x = mod.schedule(*(Tensor.from_data(v, gpu, dt) for v in (r, y, gate)))
        th, tx = norm_truth(*(v.astype(np.float64) for v in (r, y, gate)), post_t, pre_t, 1.0, 1.0)
        assert np.all(close(h.resolve().to(Device.CPU).to_f32(), th, dt)) and np.all(close(x.resolve().to(Device.CPU).to_f32(), tx, dt)), shape


@pytest.mark.gpu
@pytest.mark.parametrize("dt,vocab", [(F32, 262143), (F32, 300001), (F32, 524289), (F16, 262145), (F16, 600011), (BF16, 1100003)])
def test_vocabularies_that_a_cluster_s_ctas_share(dt, vocab, gpu):
    """One to three rows of more tokens than a CTA takes alone: the likeliest at the ends of the CTAs' shares, and with nothing else."""
    for rows, top in ((1, 32), (3, 5), (2, 0)):
        rng = np.random.default_rng(vocab + rows)
        v = round_to(dt, (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32))
        at = [vocab * k // 8 + e for k in range(9) for e in (-1, 0, 1) if 0 <= vocab * k // 8 + e < vocab]
        v[0, at] = round_to(dt, (14 + 4 * rng.random(len(at))).astype(np.float32))
        if rows > 1:
            v[1] = -np.inf
            v[1, [0, vocab - 1]] = 1.0
        tokens = [0] * rows if rows != 2 else None
        lp_check(v, tokens, top, gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_many_rows_off_the_16_byte_boundary(dt, gpu):
    """Every way rows can lie: all operands shifted alike (each shift, constant or changing from row to row), and each differently."""
    rng, rows, lib = np.random.default_rng(61), 700, _lib.load()
    size = 4 if dt == F32 else 2
    store = {F16: lambda v: v.astype(np.float16), F32: lambda v: v,
             BF16: lambda v: (v.view(np.uint32) >> 16).astype(np.uint16)}[dt]
    back = {F16: lambda b: b.astype(np.float32), F32: lambda b: b,
            BF16: lambda b: (b.astype(np.uint32) << 16).view(np.float32)}[dt]
    for d, ld, shifts in ((1001, 1001, (0, 0, 0, 0)), (1002, 1002, (0, 0, 0, 0)), (1004, 1004, (1, 1, 1, 1)), (1000, 1000, (3, 3, 3, 3)), (1000, 1008, (7, 7, 7, 7)), (513, 520, (8, 0, 16, 24)),
                          (1001, 1001, (0, 1, 0, 0)), (1001, 1003, (0, 0, 5, 0)), (2047, 2047, (5, 5, 5, 5)), (1500, 1501, (2, 2, 2, 10))):
        mats = [round_to(dt, rng.standard_normal(rows * ld + 40, dtype=np.float32)) for _ in range(2)] + [np.zeros(rows * ld + 40, np.float32)] * 2
        bufs = [device_array(gpu, store(m)) for m in mats]
        for kind in (_lib.RT_NORM_RMS, _lib.RT_NORM_LAYER):
            w = [round_to(dt, (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2)]
            wb = [device_array(gpu, store(v)) for v in w]
            p = _lib.rt_residual_norm()
            p.dt, p.residual_scale, p.block_scale, p.rows, p.d = int(dt), 0.5, 2.0, rows, d
            p.residual, p.block, p.h, p.x = (b.ptr + size * s for b, s in zip(bufs, shifts))
            p.residual_ld = p.block_ld = p.h_ld = p.x_ld = ld
            for n, b in ((p.post, wb[0]), (p.pre, wb[1])):
                n.kind, n.dt, n.eps, n.weight = kind, int(dt), 1e-5, b.ptr
            _lib.check(lib.rt_residual_norm_launch(gpu._h, ctypes.byref(p), None))
            at = [(s + np.arange(rows)[:, None] * ld + np.arange(d)[None, :]).reshape(-1) for s in shifts]
            r, y = (m[a].reshape(rows, d).astype(np.float64) for m, a in zip(mats[:2], at))
            name, eps = "rms" if kind == _lib.RT_NORM_RMS else "layer", np.float64(np.float32(1e-5))
            truths = norm_truth(r, y, None, (name, w[0].astype(np.float64), 0.0, eps), (name, w[1].astype(np.float64), 0.0, eps), 0.5, 2.0)
            for b, a, t in zip(bufs[2:], at[2:], truths):
                got = read_back(gpu, b, store(mats[2]))
                rest = np.ones(got.size, bool)
                rest[a] = False
                assert not got[rest].any() and np.all(close(back(got[a]).reshape(rows, d), t, dt)), (d, ld, shifts, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("d,rows", [(520, 3), (1000, 900), (1001, 900), (40, 4000)])
def test_a_block_without_a_residual_and_x_without_h(d, rows, dt, gpu):
    rng, lib = np.random.default_rng(71), _lib.load()
    np_dt = np.float16 if dt == F16 else np.float32
    r, y = (round_to(dt, rng.standard_normal((rows, d), dtype=np.float32)) for _ in range(2))
    w, w_t = norm_weights("rms", d, dt, rng)
    rb_, yb, wb, hb, xb = (device_array(gpu, np.ascontiguousarray(v.astype(np_dt))) for v in (r, y, w[0], 0 * r, 0 * r))
    for residual in (True, False):
        p = _lib.rt_residual_norm()
        p.dt, p.residual_scale, p.block_scale, p.rows, p.d = int(dt), 1.5, -0.5, rows, d
        p.residual, p.block, p.h, p.x = rb_.ptr if residual else None, yb.ptr, None if residual else hb.ptr, xb.ptr
        p.residual_ld = p.block_ld = p.h_ld = p.x_ld = d
        for n in (p.post, p.pre):
            n.kind, n.dt, n.eps, n.weight = _lib.RT_NORM_RMS, int(dt), w[2], wb.ptr
        _lib.check(lib.rt_residual_norm_launch(gpu._h, ctypes.byref(p), None))
        th, tx = norm_truth(r.astype(np.float64) if residual else None, y.astype(np.float64), None, w_t, w_t, 1.5, -0.5)
        assert np.all(close(read_back(gpu, xb, r.astype(np_dt)).astype(np.float32), tx, dt)), residual
        if not residual:
            assert np.all(close(read_back(gpu, hb, r.astype(np_dt)).astype(np.float32), th, dt))


@pytest.mark.gpu
def test_rows_whose_offsets_pass_32_bits(gpu):
    """Windows of a matrix of 2.4 thousand million values: the first and the last rows."""
    import torch
    rows, ld, lib = 1200, 2_000_001, _lib.load()
    big = torch.zeros(rows * ld, dtype=torch.half, device="cuda")
    m, rng = big.view(rows, ld), np.random.default_rng(72)
    for d, at in ((1001, 5), (1000, 8)):
        r = round_to(F16, rng.standard_normal((rows, d), dtype=np.float32))
        m[:, at:at + d] = torch.from_numpy(r).half().cuda()
        w = torch.ones(d, dtype=torch.half, device="cuda")
        torch.cuda.synchronize()
        p = _lib.rt_residual_norm()
        p.dt, p.residual_scale, p.rows, p.d, p.residual_ld, p.x_ld = _lib.RT_F16, 1.0, rows, d, ld, ld
        p.residual, p.x = big.data_ptr() + 2 * at, big.data_ptr() + 2 * (at + 4096)
        p.pre.kind, p.pre.dt, p.pre.eps, p.pre.weight = _lib.RT_NORM_RMS, _lib.RT_F16, 1e-5, w.data_ptr()
        _lib.check(lib.rt_residual_norm_launch(gpu._h, ctypes.byref(p), None))
        gpu.sync()
        want = normed(r.astype(np.float64), 0 * r.astype(np.float64), "rms", 1.0, 0.0, np.float64(np.float32(1e-5)))
        assert np.all(close(m[:, at + 4096:at + 4096 + d].float().cpu().numpy(), want, F16))
    ent, ids, tops = torch.zeros(rows, device="cuda"), torch.zeros(rows, 3, dtype=torch.int32, device="cuda"), torch.zeros(rows, 3, device="cuda")
    q = _lib.rt_log_probs()
    q.dt, q.top, q.rows, q.vocab, q.ld, q.logits = _lib.RT_F16, 3, rows, 1000, ld, big.data_ptr() + 16
    q.entropy, q.top_ids, q.top_log_prob = ent.data_ptr(), ids.data_ptr(), tops.data_ptr()
    torch.cuda.synchronize()
    _lib.check(lib.rt_log_probs_launch(gpu._h, ctypes.byref(q), None))
    gpu.sync()
    logp, want, order, loss, ent_loss = lp_truth(r)
    assert np.array_equal(ids.cpu().numpy(), order[:, :3]) and np.all(np.abs(ent.cpu().numpy() - want) <= ent_loss + 4 * E24 * np.abs(want))
    assert np.all(np.abs(tops.cpu().numpy() - np.take_along_axis(logp, order[:, :3], 1)) <= loss[:, None] + 4 * E24 * 20)
