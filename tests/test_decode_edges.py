"""Log probabilities and residual norms where they can go wrong: what is not finite, masks, values far from zero, very long rows."""
import ctypes

import numpy as np
import pytest

from ratchet_b200 import Device, DeviceRequest, DType, Executable, GpuBuffer, LayerNorm, Linear, RatchetError, ResidualNorm, RMSNorm, Tensor
from ratchet_b200 import _lib
from test_decode_ops import E24, close, lp_check, lp_truth, norm_truth
from util import round_to

F16, BF16, F32 = DType.F16, DType.BF16, DType.F32
LOWEST = {F16: -65504.0, BF16: -3.3895313892515355e38, F32: -3.4028234663852886e38}
HALF = {F16: 2.0**-11, BF16: 2.0**-8, F32: 2.0**-24}


def run_log_probs(v, tokens, top, gpu, dt):
    lp = Tensor.from_data(v, gpu, dt).log_probs(Tensor.from_data(np.asarray(tokens, np.int32), gpu), top)
    lp.entropy.resolve()
    return [None if t is None else t.resolve().to(Device.CPU).to_numpy() for t in lp]


def order_with_nan(v):
    """Each row's ids, NaN above all, equal values (and NaNs) by lower id."""
    nan = np.isnan(v)
    ids = np.broadcast_to(np.arange(v.shape[1]), v.shape)
    return np.lexsort((ids, -np.where(nan, 0.0, v.astype(np.float64)), ~nan), axis=-1)


# ------------------------------------------------------------------------------------------------ NaN

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 51865), (16, 51865), (400, 20003), (1, 160000), (2, 300001)])
def test_a_nan_anywhere_makes_its_row_nan_and_comes_first(rows, vocab, dt, gpu):
    """A NaN in the first, a middle and the last value a thread takes, in the partial chunks at both ends, in every CTA's share of a
    long row, beside +inf, alone among -inf, and two and forty of them; rows without one keep their answers."""
    rng, top = np.random.default_rng(81), 20
    v = round_to(dt, rng.standard_normal((rows, vocab), dtype=np.float32))
    tokens = rng.integers(0, vocab, rows)
    places = [[0], [5], [vocab - 1], [vocab - 9], [vocab // 2], [4096], [vocab // 8 - 1], [vocab // 8 + 3], [vocab * 7 // 8], [17, 17 + 8192], [3, vocab - 2],
              [8 * 513], list(range(40, vocab, vocab // 40))[:40]]
    clean = run_log_probs(v, tokens, top, gpu, dt)
    for k in range(0, len(places) + 2, max(1, rows - 1)):
        bad, hit = v.copy(), []
        for r in range(0 if rows == 1 else 1, rows):  # with several rows, the first stays as it is
            case = k + r - (rows > 1)
            if case >= len(places) + 2:
                break
            if case < len(places):
                bad[r, places[case]] = np.nan
            elif case == len(places):
                bad[r, 700], bad[r, vocab - 700] = np.inf, np.nan
            else:
                bad[r], bad[r, vocab // 3] = -np.inf, np.nan
            hit.append(r)
        got = run_log_probs(bad, tokens, top, gpu, dt)
        rest = np.setdiff1d(np.arange(rows), hit)
        for c, g in zip(clean, got):
            assert np.array_equal(c[rest], g[rest])
        assert np.isnan(got[0][hit]).all() and np.isnan(got[1][hit]).all() and np.isnan(got[3][hit]).all(), (k, hit)
        assert np.array_equal(got[2][hit], order_with_nan(bad[hit])[:, :top]), k


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [600, 5003, 300001])
def test_rows_of_many_nans_give_the_lowest_ids(vocab, dt, gpu):
    """Nothing but NaN, NaN from id 0 on and then values, and every other id: more of them than are collected before they are ranked."""
    v = np.zeros((3, vocab), np.float32)
    v[0], v[1, :580], v[2, ::2] = np.nan, np.nan, np.nan
    v[1, 590] = 3.0
    for rows in (v, np.tile(v, (100, 1))) if vocab < 300001 else (v,):
        got = run_log_probs(rows, np.zeros(len(rows)), 32, gpu, dt)
        assert np.isnan(got[0]).all() and np.isnan(got[1]).all() and np.isnan(got[3]).all()
        assert np.array_equal(got[2], order_with_nan(rows)[:, :32])


# ------------------------------------------------------------------------------------------------ masks and values far from zero

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 9, 1003, 20001])
def test_minus_infinity_is_not_the_type_s_lowest_value(vocab, dt, gpu):
    """Rows whose largest value is the type's lowest or next to it, with and without -inf beside it; odd rows lie off the 16-byte
    boundary, so that their partial chunks are filled up."""
    low = np.float32(LOWEST[dt])
    near = round_to(dt, np.array([low * (1 - k * HALF[dt]) for k in range(1, 9)], np.float32))  # 1 .. 8 half steps or so above
    rng = np.random.default_rng(82)
    v = np.full((16, vocab), low, np.float32)
    v[1] = -np.inf
    v[1, vocab // 2] = low
    v[2, rng.random(vocab) < 0.5] = -np.inf
    v[2, vocab - 1] = low
    v[3] = -np.inf
    v[4, 0] = near[7]
    for r in range(5, 13):
        v[r] = np.where(rng.random(vocab) < 0.7, -np.inf, low)
        v[r, rng.integers(vocab)] = near[r - 5]
    v[13], v[14, 0], v[15] = near[3], -np.inf, near[rng.integers(0, 8, vocab)]
    for tokens in (np.zeros(16, int), v.argmax(1)):
        lp_check(v, tokens, min(vocab, 5), gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 51865), (12, 51865), (320, 12001), (1, 300001)])
def test_rows_masked_in_stretches(rows, vocab, dt, gpu):
    """-inf over a prefix, a suffix, all but a few in the middle, and at random: threads that see nothing else first, or at all."""
    rng = np.random.default_rng(83)
    v = round_to(dt, 3 * rng.standard_normal((rows, vocab), dtype=np.float32))
    for k in range(0, 6, rows if rows < 6 else 6):
        m = v.copy()
        for r in range(rows):
            how = (k + r) % 6
            if how == 0:
                m[r, :vocab * 9 // 10] = -np.inf
            elif how == 1:
                m[r, 40000 % vocab:] = -np.inf
            elif how == 2:
                m[r, :vocab // 2], m[r, vocab // 2 + 50:] = -np.inf, -np.inf
            elif how == 3:
                m[r, rng.random(vocab) < 0.9] = -np.inf
            elif how == 4:
                m[r, :vocab - 1] = -np.inf
            else:
                m[r, rng.random(vocab) < 0.33] = -np.inf
        lp_check(m, m.argmax(1), 32, gpu, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [8, 1003, 51865])
def test_logits_far_from_zero(vocab, dt, gpu):
    """Rows of one value of any size and sign (a finite mask over everything), alone or with a smaller one in between, and rows that
    span most of the type's range: log probabilities follow the differences, which are exact."""
    rng = np.random.default_rng(84)
    top = 4 if dt == F16 else 38
    sizes = (10.0 ** rng.uniform(3, top, 40)).astype(np.float32)
    sizes = sizes[sizes < -LOWEST[dt]]
    sizes = round_to(dt, np.concatenate([sizes, [1e4, 3e4] if dt == F16 else [1e9, 2e9, 1e10, 3e10, 1e12, 1e30, 1.4e38, 1.9e38, 2.3e38, 2.4e38, 3.3e38]]).astype(np.float32))
    n = len(sizes)
    v = np.concatenate([np.repeat(s * sizes[:, None], vocab, 1) for s in (1, -1)])
    v[:n:2, vocab // 3] = v[:n:2, 0] / 2
    v[n::2, vocab // 3] = np.maximum(v[n::2, 0].astype(np.float64) * 1.5, LOWEST[dt] / 1.25)
    v[n::2, vocab // 3] = np.minimum(v[n::2, vocab // 3], v[n::2, 0])
    v[n + 1::4, 0] = LOWEST[dt]
    v[3::4, -1] = -np.inf
    v = round_to(dt, v)
    assert np.isfinite(v).any(1).all()
    lp_check(v, v.argmax(1), 5, gpu, dt)
    lp_check(v, np.zeros(len(v), int), 0, gpu, dt)


# ------------------------------------------------------------------------------------------------ long rows

@pytest.mark.gpu
def test_the_longest_row_that_is_taken(gpu):
    """2^31 - 1 logits of the type's lowest value, whose differences are taken in a second pass, and two at the end that are larger."""
    import torch
    vocab, lib = 2**31 - 1, _lib.load()
    v = torch.full((vocab,), LOWEST[BF16], dtype=torch.bfloat16, device="cuda")
    ent, given, tops, ids = (torch.zeros(n, dtype=t, device="cuda") for n, t in ((1, torch.float32), (1, torch.float32), (2, torch.float32), (2, torch.int32)))
    tokens = torch.tensor([vocab - 1], dtype=torch.int32, device="cuda")
    p = _lib.rt_log_probs()
    p.dt, p.top, p.rows, p.vocab, p.ld, p.logits, p.tokens = _lib.RT_BF16, 2, 1, vocab, vocab, v.data_ptr(), tokens.data_ptr()
    p.log_prob, p.entropy, p.top_ids, p.top_log_prob = given.data_ptr(), ent.data_ptr(), ids.data_ptr(), tops.data_ptr()

    def run():
        torch.cuda.synchronize()
        _lib.check(lib.rt_log_probs_launch(gpu._h, ctypes.byref(p), None))
        gpu.sync()
        return given.item(), ent.item(), ids.tolist(), tops.tolist()

    # every power is 1, so the sums are exact but for the last ones: a few steps of their 2^31, and of log2's 31 and ln 2
    slack = (16 + 8 * 21.5) * E24
    one, h, first, tp = run()
    assert abs(one + np.log(vocab)) <= slack and abs(h - np.log(vocab)) <= slack and first == [0, 1] and np.abs(np.array(tp) + np.log(vocab)).max() <= slack
    v[-1] = v[-3] = -3.2e38
    one, h, first, tp = run()
    assert abs(one + np.log(2)) <= slack and abs(h - np.log(2)) <= slack and first == [vocab - 3, vocab - 1] and np.abs(np.array(tp) + np.log(2)).max() <= slack


#: of an f32 sum, relative to the sum of the terms: a thread adds 2048 terms at most before its sum joins the others, each addition off
#: by half a step; an exponential by two steps of 2^-23 and its exponent's rounding; the sums' sum and the trees by as much as 300 more
LONG = (2048 + 300 + 16) * E24


@pytest.mark.gpu
@pytest.mark.parametrize("dt,vocab,rows", [(F32, 2**27 + 3, 1), (F16, 2**28 + 5, 1), (BF16, 2**28, 2), (F16, 2**22 + 1, 300), (F16, 2**31 - 1, 1), (BF16, 2**31 - 9, 1)])
def test_rows_of_many_millions(dt, vocab, rows, gpu):
    """A thread's first values are larger than all that follow, which are equal: its sums take the same term over and over, whose
    roundings all fall to the same side.  The last two ids are the likeliest, then the first two."""
    import torch
    kind = {F32: torch.float32, F16: torch.half, BF16: torch.bfloat16}[dt]
    v = torch.full((rows, vocab), 1.0, dtype=kind, device="cuda")
    for k in range(8):
        v[:, max(0, vocab // 8 * k - 64):vocab // 8 * k + 16500] = 4.3125
    v[:, -2:] = 5.0
    ent, ids, tops, given = (torch.zeros(rows, n, dtype=t, device="cuda") for n, t in ((1, torch.float32), (4, torch.int32), (4, torch.float32), (1, torch.float32)))
    tokens = torch.full((rows,), vocab - 1, dtype=torch.int32, device="cuda")
    p = _lib.rt_log_probs()
    p.dt, p.top, p.rows, p.vocab, p.ld, p.logits, p.tokens = int(dt), 4, rows, vocab, vocab, v.data_ptr(), tokens.data_ptr()
    p.log_prob, p.entropy, p.top_ids, p.top_log_prob = given.data_ptr(), ent.data_ptr(), ids.data_ptr(), tops.data_ptr()
    torch.cuda.synchronize()
    _lib.check(_lib.load().rt_log_probs_launch(gpu._h, ctypes.byref(p), None))
    gpu.sync()
    kinds = np.array([5.0, 4.3125, 1.0])
    ahead = int((v[0] == 4.3125).sum())
    weights = np.array([2, ahead, vocab - 2 - ahead]) * np.exp(kinds)
    logp = kinds - np.log(weights.sum())
    assert np.array_equal(ids.cpu().numpy(), np.tile([vocab - 2, vocab - 1, 0, 1], (rows, 1)))
    slack = LONG + 4 * E24 * 25  # (log2 and the last sums are f32 numbers of at most 25)
    assert np.abs(tops.double().cpu().numpy() - logp[[0, 0, 1, 1]]).max() <= slack
    assert np.abs(given.double().cpu().numpy() - logp[0]).max() <= slack
    # entropy = ln S - sum e t / S: both lose LONG, the second times its terms' size, 5.8 powers of two at most
    assert np.abs(ent.double().cpu().numpy() + (weights * logp).sum() / weights.sum()).max() <= slack + 2 * 5.8 * LONG


# ------------------------------------------------------------------------------------------------ norms

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("post", [None, "rms", "layer", "layer+bias"])
@pytest.mark.parametrize("d", [40, 520, 1003, 2560])
def test_infinite_gates_do_the_same_to_few_rows_and_to_many(d, post, dt, gpu):
    """h = a r + b g post(block) where g is infinite: +-inf by the block's sign at that place, NaN where the block is 0; the rest as ever."""
    rng, rows = np.random.default_rng(91), 5003
    r, y = (round_to(dt, rng.standard_normal((rows, d), dtype=np.float32)) for _ in range(2))
    if post is None:
        y[7, 3] = 0.0
    w, b = round_to(dt, rng.uniform(0.5, 2.0, d).astype(np.float32)), round_to(dt, rng.uniform(-2.0, 2.0, d).astype(np.float32))
    gate = round_to(dt, rng.uniform(0.5, 1.5, d).astype(np.float32))
    gate[[3, 17, d - 1]] = np.inf, -np.inf, np.inf
    t = lambda a: Tensor.from_data(a, gpu, dt)  # noqa: E731
    block = {None: None, "rms": lambda: RMSNorm(t(w)), "layer": lambda: LayerNorm(t(w)), "layer+bias": lambda: LayerNorm(t(w), t(b))}[post]
    kind, bias = None if post is None else post.split("+")[0], b.astype(np.float64) if post == "layer+bias" else 0.0
    truth = (kind, w.astype(np.float64), bias, np.float64(np.float32(1e-5)))
    finite = np.isfinite(gate)
    with np.errstate(invalid="ignore"):
        (v, e), _ = norm_truth(r.astype(np.float64), y.astype(np.float64), np.where(finite, gate, 1.0).astype(np.float64), truth, (None, 1, 0, 0), 0.5, -2.0)
        u, eu = norm_truth(None, y.astype(np.float64), None, truth, (None, 1, 0, 0), 1.0, -2.0)[0]
        want = np.where(finite, v, gate.astype(np.float64) * u)
    sure = finite | (np.abs(u) > 2 * eu) | (u == 0)  # (whose sign f32 has)
    assert sure.mean() > 0.99
    for pre in (None, LayerNorm(t(w))):
        for n in (3, 100, rows):
            mod = ResidualNorm(pre, block() if block else None, 0.5, -2.0)
            h, x = mod.schedule(t(r[:n]), t(y[:n]), t(gate))
            got = h.resolve().to(Device.CPU).to_f32().astype(np.float64)
            same = (got == want[:n]) | (np.isnan(got) & np.isnan(want[:n])) | (finite & close(got, (want[:n], e[:n]), dt))
            assert np.all(same | ~sure[:n]), (n, pre, np.argwhere(~(same | ~sure[:n]))[:4])
            assert x is None or np.isnan(x.resolve().to(Device.CPU).to_f32()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("d", [96, 383, 520, 1003])
def test_infinite_gates_of_some_rows_only(d, dt, gpu):
    """A gate per row and per sequence, infinite at a few places of a few of them, behind a layer norm with a bias: teams cross from
    ordinary gates to those and back."""
    rng = np.random.default_rng(93)
    shape = (60, 7, 9, d)
    r, y = (round_to(dt, rng.standard_normal(shape, dtype=np.float32)) for _ in range(2))
    w, b = round_to(dt, rng.uniform(0.5, 2.0, d).astype(np.float32)), round_to(dt, rng.uniform(-2.0, 2.0, d).astype(np.float32))
    t = lambda a: Tensor.from_data(a, gpu, dt)  # noqa: E731
    mod = ResidualNorm(RMSNorm(t(w)), LayerNorm(t(w), t(b)))
    truth, pre = ("layer", w.astype(np.float64), b.astype(np.float64), np.float64(np.float32(1e-5))), ("rms", w.astype(np.float64), 0.0, np.float64(np.float32(1e-5)))
    for lead in ((60, 7, 9), (60, 1, 1)):
        gate = round_to(dt, rng.uniform(0.5, 1.5, (*lead, d)).astype(np.float32))
        rows = gate.reshape(-1, d)
        for i in rng.choice(len(rows), max(3, len(rows) // 20), replace=False):
            rows[i, rng.integers(d)] = rng.choice([np.inf, -np.inf])
        h, x = mod.schedule(t(r), t(y), t(gate))
        h, x = (v.resolve().to(Device.CPU).to_f32().astype(np.float64) for v in (h, x))
        finite = np.broadcast_to(np.isfinite(gate), shape)
        with np.errstate(invalid="ignore"):
            th, tx = norm_truth(r.astype(np.float64), y.astype(np.float64), np.where(np.isfinite(gate), gate, 1.0).astype(np.float64), truth, pre, 1.0, 1.0)
            u, eu = norm_truth(None, y.astype(np.float64), None, truth, (None, 1, 0, 0), 1.0, 1.0)[0]
            want = np.where(finite, 0.0, gate.astype(np.float64) * u)
            ok = np.where(finite, close(h, th, dt), (h == want) | (np.abs(u) <= 2 * eu))
            assert np.all(ok)
            whole = finite.all(-1)
            # an infinite value's row has a root mean square of inf: 0 for what is finite, NaN for inf / inf
            assert np.all(close(x, tx, dt)[whole]) and np.all(np.where(finite, x == 0, np.isnan(x))[~whole])


# ------------------------------------------------------------------------------------------------ CPU: executables

def test_an_executable_refuses_nodes_of_another_device():
    """Their memory belongs to the other GPU: a Matmul node, an operator with several outputs, and one of each."""
    here, there = (Device(DeviceRequest.GPU, k) for k in range(2))

    def on(device, *outs):
        for t in outs:
            t.storage = GpuBuffer.__new__(GpuBuffer)
            t.storage.device, t.storage._h, t.storage.ptr, t.storage.size = device, None, 1 << 20, 1 << 16
        return list(outs)

    t = lambda *shape: Tensor(shape, F16, there)  # noqa: E731
    product = on(there, Linear(t(8, 64)).schedule(t(1, 2, 64)))
    both = on(there, *ResidualNorm(RMSNorm(t(64))).schedule(t(2, 64), t(2, 64)))
    for nodes in (product, both, product + both, both + product):
        with pytest.raises(RatchetError, match="a node is on Device::GPU"):
            Executable(here, nodes)
