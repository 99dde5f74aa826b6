"""What stands around the Linears of a decode step: norms with the residual stream, and what a step answers with.

    RMSNorm, LayerNorm    crates/ratchet-nn/src/norm.rs (the modules' `schedule`)
    ResidualNorm          a block's output into the residual stream and the next block's input, in one launch
    Tensor.log_probs      log probabilities of given tokens, entropy and top alternatives of logits

Lazy like `Linear.schedule`: they build a node and `Tensor.resolve` launches it, on the device's stream; an `Executable` takes
their resolved outputs among its nodes.  The arithmetic and the checks are the library's (rt_residual_norm, rt_log_probs).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

from . import _lib
from ._lib import RatchetError, ShapeError
from .tensor import DType, LazyOp, Tensor

_FLOATS = (DType.F32, DType.F16, DType.BF16)


def _refuse(status: int, name: str, message: str):
    raise (ShapeError if status == _lib.RT_ERR_SHAPE else RatchetError)(status, name, message)


def _shape(ok: bool, message: str) -> None:
    if not ok:
        _refuse(_lib.RT_ERR_SHAPE, "RT_ERR_SHAPE", message)


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.ptr


class _Norm:
    kind = _lib.RT_NORM_NONE

    def __init__(self, weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
        self.weight, self.bias, self.eps = weight, bias, float(eps)
        if weight is not None and bias is not None and weight.dt != bias.dt:
            _refuse(_lib.RT_ERR_DTYPE, "RT_ERR_DTYPE", f"norm weight is {weight.dt.name}, bias {bias.dt.name}")

    def _srcs(self):
        return [t for t in (self.weight, self.bias) if t is not None]

    def _check(self, d: int) -> None:
        for t in self._srcs():
            _shape(t.numel() == d, f"a norm of {t.numel()} weights over rows of {d} values")

    def _fill(self, n: "_lib.rt_norm") -> None:
        n.kind, n.eps, n.weight, n.bias = self.kind, self.eps, _ptr(self.weight), _ptr(self.bias)
        n.dt = int((self.weight or self.bias).dt) if self._srcs() else _lib.RT_F32

    def schedule(self, input: Tensor) -> Tensor:
        """Module::schedule: the norm alone, over the last dimension."""
        op = _ResidualNormOp(input, None, None, None, self, 1.0, 1.0, want_h=False)
        return op.outputs(input.device)[0]


class RMSNorm(_Norm):
    """v / sqrt(mean(v^2) + eps) * weight (crates/ratchet-nn/src/norm.rs)."""

    kind = _lib.RT_NORM_RMS

    def __init__(self, weight: Optional[Tensor], eps: float = 1e-5):
        super().__init__(weight, None, eps)


class LayerNorm(_Norm):
    """(v - mean) / sqrt(var + eps) * weight + bias (crates/ratchet-nn/src/norm.rs)."""

    kind = _lib.RT_NORM_LAYER

    def __init__(self, weight: Optional[Tensor], bias: Optional[Tensor] = None, eps: float = 1e-5):
        super().__init__(weight, bias, eps)


class _ResidualNormOp(LazyOp):
    def __init__(self, residual: Optional[Tensor], block: Optional[Tensor], gate: Optional[Tensor], post: Optional[_Norm], pre: Optional[_Norm],
                 residual_scale: float, block_scale: float, want_h: bool):
        first = residual if residual is not None else block
        if first is None or not first.shape:
            _refuse(_lib.RT_ERR_ARG, "RT_ERR_ARG", "a norm needs an input of at least one dimension")
        self.residual, self.block, self.gate, self.post, self.pre = residual, block, gate, post, pre
        self.residual_scale, self.block_scale, self.want_h = float(residual_scale), float(block_scale), want_h
        self.dt, self.shape = first.dt, list(first.shape)
        self.d, self.gate_rows = self.shape[-1], 1
        self.rows = math.prod(self.shape[:-1])
        if self.dt not in _FLOATS:
            _refuse(_lib.RT_ERR_DTYPE, "RT_ERR_DTYPE", f"no norm of {self.dt.name} rows")
        _shape(self.d >= 1, "a norm over rows of no values")
        for t in (block, gate):
            if t is not None and t.dt != self.dt:
                _refuse(_lib.RT_ERR_DTYPE, "RT_ERR_DTYPE", f"residual, block and gate are of one type: {self.dt.name}, {t.dt.name}")
        if residual is not None and block is not None:
            _shape(list(block.shape) == self.shape, f"residual {self.shape} and block {list(block.shape)} differ in shape")
        if gate is not None:
            # [d], or [a, .., 1, .., d]: the leading dimensions of the input, then ones
            g = list(gate.shape)
            lead = g[:-1] if len(g) == len(self.shape) else None if len(g) > 1 else []
            full = 0 if lead is None else next((i for i, n in enumerate(lead) if n == 1 and self.shape[i] != 1), len(lead))
            _shape(lead is not None and g[-1] == self.d and lead[:full] == self.shape[:full] and all(n == 1 for n in lead[full:]),
                   f"a gate of shape {g} does not run along rows of {self.shape}")
            self.gate_rows = math.prod(lead)
        for n in (post, pre):
            if n is not None:
                n._check(self.d)
        self.specs = [(self.shape, self.dt)] * (int(want_h) + int(pre is not None))

    def srcs(self):
        found = [t for t in (self.residual, self.block, self.gate) if t is not None]
        for n in (self.post, self.pre):
            found += n._srcs() if n is not None else []
        return found

    def bind(self, step: "_lib.rt_step") -> None:
        step.kind, n = _lib.RT_STEP_RESIDUAL_NORM, step.norm
        n.dt, n.residual_scale, n.block_scale, n.rows, n.d = int(self.dt), self.residual_scale, self.block_scale, self.rows, self.d
        n.residual, n.block, n.gate, n.gate_rows = _ptr(self.residual), _ptr(self.block), _ptr(self.gate), max(1, self.gate_rows)
        n.residual_ld = n.block_ld = n.h_ld = n.x_ld = self.d
        for norm, field in ((self.post, n.post), (self.pre, n.pre)):
            if norm is not None:
                norm._fill(field)
        buffers = [b.ptr for b in self._buffers]
        n.h = buffers[0] if self.want_h else None
        n.x = buffers[-1] if self.pre is not None else None


class ResidualNorm:
    """Between two blocks: h = residual_scale * residual + block_scale * gate * post(block), x = pre(h).

    `pre` is the next block's norm (None: only h is computed), `post` the norm of this block's output, if the model has one.
    `schedule` gives (h, x): the new residual stream and the next block's input.  A gate has the input's dtype and shape [d],
    or the input's shape with trailing row dimensions of 1 (a gate per sequence: [batch, 1, d])."""

    def __init__(self, pre: Optional[_Norm], post: Optional[_Norm] = None, residual_scale: float = 1.0, block_scale: float = 1.0):
        self.pre, self.post, self.residual_scale, self.block_scale = pre, post, residual_scale, block_scale

    def schedule(self, residual: Tensor, block: Tensor, gate: Optional[Tensor] = None):
        op = _ResidualNormOp(residual, block, gate, self.post, self.pre, self.residual_scale, self.block_scale, want_h=True)
        outs = op.outputs(residual.device)
        return (outs[0], outs[1]) if self.pre is not None else (outs[0], None)


class LogProbs(NamedTuple):
    """What `Tensor.log_probs` gives, for logits of shape [.., vocab]."""

    log_prob: Optional[Tensor]      # [..] F32: of the given tokens (None without them)
    entropy: Tensor                 # [..] F32
    top_ids: Optional[Tensor]       # [.., top] I32, the likeliest first, equal logits by lower id (None for top = 0)
    top_log_prob: Optional[Tensor]  # [.., top] F32


class _LogProbsOp(LazyOp):
    def __init__(self, logits: Tensor, tokens: Optional[Tensor], top: int):
        if not logits.shape:
            _refuse(_lib.RT_ERR_ARG, "RT_ERR_ARG", "log_probs needs logits of at least one dimension")
        self.logits, self.tokens, self.top = logits, tokens, int(top)
        lead, self.vocab = list(logits.shape[:-1]), logits.shape[-1]
        self.rows = math.prod(lead)
        if logits.dt not in _FLOATS:
            _refuse(_lib.RT_ERR_DTYPE, "RT_ERR_DTYPE", f"no log probabilities of {logits.dt.name} logits")
        _shape(0 <= self.top <= self.vocab and self.vocab >= 1, f"top {self.top} of a vocabulary of {self.vocab}")
        if self.top > 32:
            _refuse(_lib.RT_ERR_UNSUPPORTED, "RT_ERR_UNSUPPORTED", "more than 32 alternatives")
        if tokens is not None:
            if tokens.dt not in (DType.I32, DType.U32):
                _refuse(_lib.RT_ERR_DTYPE, "RT_ERR_DTYPE", f"tokens are I32 or U32, not {tokens.dt.name}")
            _shape(tokens.numel() == self.rows, f"{tokens.numel()} tokens for {self.rows} rows of logits")
        self.specs = ([(lead, DType.F32)] if tokens is not None else []) + [(lead, DType.F32)]
        if self.top:
            self.specs += [(lead + [self.top], DType.I32), (lead + [self.top], DType.F32)]

    def srcs(self):
        return [self.logits] + ([self.tokens] if self.tokens is not None else [])

    def bind(self, step: "_lib.rt_step") -> None:
        step.kind, p = _lib.RT_STEP_LOG_PROBS, step.log_probs
        p.dt, p.top, p.rows, p.vocab, p.ld = int(self.logits.dt), self.top, self.rows, self.vocab, self.vocab
        p.logits, p.tokens = self.logits.ptr, _ptr(self.tokens)
        ptrs = [b.ptr for b in self._buffers]
        if self.top:
            p.top_log_prob, p.top_ids = ptrs.pop(), ptrs.pop()
        p.entropy = ptrs.pop()
        p.log_prob = ptrs.pop() if self.tokens is not None else None


def log_probs(logits: Tensor, tokens: Optional[Tensor] = None, top: int = 0) -> LogProbs:
    """log p(token), entropy and the `top` (0 .. 32) likeliest tokens of each row of logits [.., vocab].

    tokens: I32 or U32, one per row; one outside the vocabulary has the log probability NaN.  A logit of -inf is a token that
    cannot be drawn; a row of nothing else has log probabilities of -inf and an entropy of 0."""
    op = _LogProbsOp(logits, tokens, top)
    outs = op.outputs(logits.device)
    given = outs.pop(0) if tokens is not None else None
    return LogProbs(given, outs[0], *(outs[1:] if top else (None, None)))
