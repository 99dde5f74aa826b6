"""The operators a decode step needs around its quantised Linears, and the work their speed is judged by.

    w4        y = x W^T for 1..16 rows of x, W in 4-bit codes with an f16 scale and a zero point per group of 32, 64 or 128
              values of a row: w = (q - z) s
    norm      what stands between two blocks: h = a r + b g * N_post(y) and x = N_pre(h), with RMS or layer norms, a gate per
              channel or per sequence, and the two scalars
    logprobs  from logits: the log probability of each row's given token, the row's entropy, and its most likely tokens

`own` false computes them in elementary torch operations, `own` true makes the framework's calls.  Everything is made from the seed.
"""
import math
import types

import torch

own = False

TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
SIZE = {"F32": 4, "F16": 2, "BF16": 2}


def listed():
    return [
        # one attention projection of Phi-2 on one token: the smallest product of a decode step
        {"name": "w4_projection_1row", "kind": "w4", "group": 128, "dtype": "F16", "out": 2560, "d": 2560, "rows": 1},
        # fc1 of Phi-2's MLP on one token, in bf16 with finer groups
        {"name": "w4_fc1_1row_bf16", "kind": "w4", "group": 64, "dtype": "BF16", "out": 10240, "d": 2560, "rows": 1},
        # Whisper-tiny's logits on one token: very many short rows, an odd number of them
        {"name": "w4_whisper_logits", "kind": "w4", "group": 32, "dtype": "F16", "out": 51865, "d": 384, "rows": 1},
        # fc2 of Phi-2's MLP for five streams decoded together: few long rows, the finest groups
        {"name": "w4_fc2_5rows", "kind": "w4", "group": 32, "dtype": "F16", "out": 2560, "d": 10240, "rows": 5},
        # the logits of Phi-2 for sixteen streams: the largest product
        {"name": "w4_lm_head_16rows", "kind": "w4", "group": 128, "dtype": "F16", "out": 51200, "d": 2560, "rows": 16},
        # between two layers of Phi-2, one token: the smallest norm
        {"name": "norm_1row", "kind": "norm", "dtype": "F16", "sequences": 1, "rows": 1, "d": 2560, "post": "none", "pre": "layer", "gate": "none"},
        # between two layers of Whisper-tiny's encoder over 30 s of audio
        {"name": "norm_whisper_encoder", "kind": "norm", "dtype": "F16", "sequences": 1, "rows": 1500, "d": 384, "post": "none", "pre": "layer",
         "gate": "none"},
        # norms on both sides of a block with a gate per channel, a short prompt of ragged length and odd width in f32
        {"name": "norm_prompt77_f32", "kind": "norm", "dtype": "F32", "sequences": 1, "rows": 77, "d": 2561, "post": "rms", "pre": "rms",
         "gate": "channel"},
        # the same on a batch of long prompts in bf16, a gate per sequence: the largest norm
        {"name": "norm_prefill_bf16", "kind": "norm", "dtype": "BF16", "sequences": 4, "rows": 2048, "d": 2560, "post": "rms", "pre": "rms",
         "gate": "sequence"},
        # one sampled token of Whisper with a third of the vocabulary masked out, and the five likeliest
        {"name": "logprobs_1row", "kind": "logprobs", "dtype": "F16", "rows": 1, "vocab": 51865, "top": 5, "masked": 0.33},
        # sixteen streams, f32 logits of Phi-2, twenty alternatives
        {"name": "logprobs_16rows_f32", "kind": "logprobs", "dtype": "F32", "rows": 16, "vocab": 51200, "top": 20, "masked": 0.0},
        # scoring a long prompt in bf16: the largest
        {"name": "logprobs_prompt_bf16", "kind": "logprobs", "dtype": "BF16", "rows": 2048, "vocab": 51865, "top": 20, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "norm", "logprobs"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        d = group * max(1, _log(rng, 256, 10240) // group)
        return {"kind": "w4", "group": group, "dtype": rng.choice(["F16", "F16", "BF16"]), "out": _log(rng, 200, min(51865, 51200 * 2560 // d)), "d": d,
                "rows": rng.choice([1, 1, 1, _log(rng, 2, 16), rng.randint(2, 16)])}
    if kind == "norm":
        d, sequences = _log(rng, 200, 9000), rng.choice([1, 1, 2, 3, 4])
        return {"kind": "norm", "dtype": rng.choice(["F16", "BF16", "F32"]), "sequences": sequences,
                "rows": rng.choice([1, _log(rng, 1, max(1, 8192 * 2560 // (2 * d * sequences)))]), "d": d, "post": rng.choice(["none", "rms", "layer"]),
                "pre": rng.choice(["rms", "layer"]), "gate": rng.choice(["none", "channel", "sequence"])}
    vocab, dtype = _log(rng, 1001, 160000), rng.choice(["F16", "BF16", "F32"])
    return {"kind": "logprobs", "dtype": dtype, "rows": rng.choice([1, _log(rng, 2, 64), _log(rng, 64, max(65, 2048 * 51865 * 2 // (vocab * SIZE[dtype])))]),
            "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]), "masked": rng.choice([0.0, 0.0, 0.33, 0.9])}


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda")
    gen.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = types.SimpleNamespace(kind=c["kind"], case=dict(c))
    dt = TORCH[c["dtype"]]
    if s.kind == "w4":
        # min-max quantised N(0, 1/d) weights; activations of unit scale, as they are behind a norm
        w = (randn(c["out"], c["d"]) / math.sqrt(c["d"])).view(c["out"], -1, c["group"])
        lo, hi = w.amin(-1, keepdim=True).clamp_max(0), w.amax(-1, keepdim=True).clamp_min(0)
        s.scales = ((hi - lo) / 15).half()
        zeros = torch.round(-lo / s.scales.float()).clamp(0, 15)
        q = (torch.round(w / s.scales.float()) + zeros).clamp(0, 15).to(torch.uint8).view(c["out"], -1)
        s.codes = q[:, 0::2] | q[:, 1::2] << 4  # the even value of a pair in the low half of its byte
        s.scales, s.zeros = s.scales[..., 0].contiguous(), zeros[..., 0].to(torch.uint8)
        s.x = randn(1, c["rows"], c["d"]).to(dt)
    elif s.kind == "norm":
        # a residual stream a few times as large as what a block adds to it; weights around one
        shape = (c["sequences"], c["rows"], c["d"])
        s.r, s.y = (3 * randn(*shape)).to(dt), randn(*shape).to(dt)
        weight = lambda: (1 + 0.1 * randn(c["d"])).to(dt)  # noqa: E731
        s.post = None if c["post"] == "none" else (weight(), (0.1 * randn(c["d"])).to(dt) if c["post"] == "layer" else None)
        s.pre = weight(), (0.1 * randn(c["d"])).to(dt) if c["pre"] == "layer" else None
        s.gate = None if c["gate"] == "none" else (0.5 + 0.2 * randn(*((c["d"],) if c["gate"] == "channel" else (c["sequences"], 1, c["d"])))).to(dt)
        s.a, s.b, s.eps = 1.0, 1.0 if c["gate"] != "none" else 0.7, 1e-5
    else:
        # logits of spread 2.5 with one clear favourite in most rows; the given tokens are likely ones
        s.logits = 2.5 * randn(c["rows"], c["vocab"])
        s.tokens = torch.randint(c["vocab"], (c["rows"],), generator=gen, device="cuda")
        s.logits[torch.arange(c["rows"], device="cuda"), s.tokens] += 8 * torch.rand(c["rows"], generator=gen, device="cuda")
        if c["masked"]:
            hide = torch.rand(c["rows"], c["vocab"], generator=gen, device="cuda") < c["masked"]
            hide[torch.arange(c["rows"], device="cuda"), s.tokens] = False
            s.logits.masked_fill_(hide, -math.inf)
        s.logits, s.tokens = s.logits.to(dt), s.tokens.to(torch.int32)
    if own:
        _bind(s)
    torch.cuda.synchronize()
    return s


class _Memory:
    """A library tensor's memory as torch sees it; holds the tensor."""

    def __init__(self, tensor, nbytes):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (tensor.ptr, False), "version": 2}


def _bind(s):
    """What a user's program holds before the call: the inputs and weights in the library's tensors, and the nodes bound as an executable."""
    import ratchet_b200 as rb
    from ratchet_b200 import Device, DeviceRequest, DType, Executable, GpuBuffer, Tensor

    torch.cuda.synchronize()
    gpu, c = Device.request_device(DeviceRequest.GPU, 0), s.case

    def view(t):
        types_ = {**TORCH, "I32": torch.int32}
        return torch.as_tensor(_Memory(t, t.numel() * t.dt.size_of()), device="cuda").view(types_[t.dt.name]).view(t.shape)

    def tensor(v, dt=None, parts=None):
        dt = dt or DType[c["dtype"]]
        shape = [c["out"], c["d"]] if parts else list(v.shape)
        t = Tensor(shape, dt, gpu, GpuBuffer(gpu, dt.nbytes(math.prod(shape))))
        raw = torch.as_tensor(_Memory(t, dt.nbytes(math.prod(shape))), device="cuda")
        for (offset, _), part in zip(dt.segments(math.prod(shape)), parts or [v]):
            part = part.contiguous().view(-1).view(torch.uint8)
            raw[offset:offset + part.numel()].copy_(part)
        return t

    if s.kind == "w4":
        lin = rb.Linear(tensor(None, DType["Q4_G%d" % c["group"]], [s.codes, s.scales, s.zeros]))
        x = tensor(s.x)
        torch.cuda.synchronize()
        outs = [lin.schedule(x)]
    elif s.kind == "norm":
        def norm(kind, p):
            if kind == "none":
                return None
            return rb.RMSNorm(tensor(p[0]), s.eps) if kind == "rms" else rb.LayerNorm(tensor(p[0]), tensor(p[1]), s.eps)
        between = rb.ResidualNorm(norm(c["pre"], s.pre), norm(c["post"], s.post), residual_scale=s.a, block_scale=s.b)
        r, y, gate = tensor(s.r), tensor(s.y), None if s.gate is None else tensor(s.gate)
        torch.cuda.synchronize()
        outs = list(between.schedule(r, y, gate))
    else:
        logits, tokens = tensor(s.logits), tensor(s.tokens, DType.I32)
        torch.cuda.synchronize()
        lp = logits.log_probs(tokens, top=c["top"])
        outs = [lp.log_prob, lp.entropy] + ([lp.top_ids, lp.top_log_prob] if c["top"] else [])
    for t in outs:
        t.resolve()
    s.exe, s.out = Executable(gpu, outs, use_graph=False), [view(t) for t in outs]


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        s.exe.dispatch()
        return s.out
    return {"w4": _w4, "norm": _norm, "logprobs": _log_probs}[s.kind](s)


def _w4(s):
    codes = torch.stack([s.codes & 15, s.codes >> 4], -1).view(*s.scales.shape, -1)
    w = (codes.float() - s.zeros[..., None].float()) * s.scales[..., None].float()
    return [(s.x.float() @ w.view(s.case["out"], -1).t()).to(s.x.dtype)]


def _normed(v, kind, p, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * p[0].float()
    return v + p[1].float() if kind == "layer" else v


def _norm(s):
    y = _normed(s.y.float(), s.case["post"], s.post, s.eps) * s.b
    h = s.a * s.r.float() + (y if s.gate is None else y * s.gate.float())
    return [h.to(s.r.dtype), _normed(h, s.case["pre"], s.pre, s.eps).to(s.r.dtype)]


def _log_probs(s):
    v, top = s.logits.float() + 0.0, s.case["top"]
    m = v.amax(-1, keepdim=True)
    d = v - m
    e = torch.exp(d)
    total = e.sum(-1, dtype=torch.float64)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, 0).sum(-1, dtype=torch.float64)
    given = d.gather(-1, s.tokens.long()[:, None])[:, 0].double() - log_total
    out = [given.float(), (log_total - weighted / total).float()]
    if top:
        # values in order, equal ones by index: one whole number for both
        bits = v.view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2**32 - torch.arange(v.shape[-1], device=v.device)
        ids = -(torch.topk(order, top, -1).values % 2**32) % 2**32
        out += [ids.to(torch.int32), (d.gather(-1, ids).double() - log_total[:, None]).float()]
    return out


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits

def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["kind"] == "w4":
        n = c["out"] * c["d"]
        return {"bytes": n / 2 + n / c["group"] * 3 + c["rows"] * (c["d"] + c["out"]) * size, "flops": 2.0 * c["rows"] * n}
    if c["kind"] == "norm":
        n, d = c["sequences"] * c["rows"] * c["d"], c["d"]
        params = {"none": 0, "rms": d, "layer": 2 * d}
        gate = {"none": 0, "channel": d, "sequence": c["sequences"] * d}[c["gate"]]
        return {"bytes": (4 * n + params[c["post"]] + params[c["pre"]] + gate) * size, "flops": 12.0 * n}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * size + c["rows"] * (4 + 8 + 8 * c["top"]), "flops": 6.0 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "w4":
        low, high = torch.bitwise_and(s.codes, 15).double(), torch.div(s.codes, 16, rounding_mode="floor").double()
        y, half = 0, s.case["group"] // 2
        for codes, x in ((low, s.x[..., 0::2].double()), (high, s.x[..., 1::2].double())):
            steps = codes.unflatten(-1, (-1, half)) - s.zeros.double().unsqueeze(-1)
            y = y + x @ (steps * s.scales.double().unsqueeze(-1)).flatten(1).T
        return [y]
    if s.kind == "norm":
        def norm(v, kind, p):
            if kind == "none":
                return v
            centre = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
            spread = ((v - centre) ** 2).sum(-1, keepdim=True) / v.shape[-1]
            v = (v - centre) / (spread + s.eps).sqrt() * p[0].double()
            return v if p[1] is None else v + p[1].double()
        add = norm(s.y.double(), s.case["post"], s.post)
        h = s.r.double() * s.a + s.b * add * (1.0 if s.gate is None else s.gate.double())
        return [h, norm(h, s.case["pre"], s.pre)]
    v = s.logits.double()
    lse = torch.logsumexp(v, -1)
    logp = v - lse[:, None]
    p = logp.exp()
    out = [logp[torch.arange(v.shape[0], device="cuda"), s.tokens.long()], -(p * logp.masked_fill(p == 0, 0)).sum(-1)]
    if s.case["top"]:
        out += [None, logp.sort(-1, descending=True).values[:, :s.case["top"]]]
    return out
