"""Rotary positions for the queries and keys of attention: beside the time embedding of the UNets (`vamd_timeembed`), what a
sequence model over codebook indices has in place of it.

    rotary = Rotary(head_dim, rotary_dim, layout="half", base=10000.0, scaling={"type": "yarn", "factor": 4.0, "original": 8192})
    q, k = rotary(positions, q, k)                 # differentiable (backward, forward mode); one kernel for both, one for both gradients
    rotary.apply_(positions, q, k)                 # in place, without gradients

q, k: [..., heads, head_dim], float32 or bfloat16 on the GPU, any strides with adjacent features (heads may come before tokens
in memory); positions: int32 or int64, of shape q.shape[:-2] or broadcast to it.  Angles are exact fractions of a turn at any
position (csrc/rotary.hip).  There is no CPU path.
"""
import math
from fractions import Fraction

import torch
from torch import nn

from . import _lib
from ._lib import call_on, has_tangent, overlapping, overwritten, self_overlapping

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_PI = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """(radians per position of each pair as Python floats, amplitude).

    f_i = base^(-2i / rotary_dim).  Contexts longer than the trained one:
      {"type": "linear", "factor": s}                    f / s: positions are squeezed
      {"type": "ntk", "factor": s}                       base * s^(R / (R - 2)): the slowest pair is slowed by s, the fastest not
      {"type": "yarn", "factor": s, "original": L}       pairs that turn less than `alpha` (1) times over L positions are slowed by
                                                         s, those that turn more than `beta` (32) times are left alone, a linear
                                                         blend between; the turned features grow by `amplitude` (0.1 ln s + 1)
    """
    R, amplitude = rotary_dim, 1.0
    base = float(base)
    scaling = dict(scaling) if scaling else {"type": "none"}
    kind = scaling.pop("type", None)
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",), "yarn": ("factor", "original", "alpha", "beta", "amplitude")}
    if kind not in known:
        raise ValueError(f"scaling type {kind!r} (linear, ntk or yarn)")
    odd = set(scaling) - set(known[kind])
    if odd:
        raise ValueError(f"scaling {kind!r} has no {sorted(odd)}")
    factor = float(scaling["factor"]) if kind != "none" else 1.0
    if not factor >= 1.0 or math.isinf(factor):
        raise ValueError(f"a scaling's factor is 1 or more, not {factor}")
    if not 1.0 < base < math.inf:
        raise ValueError(f"base {base}: a number above 1")
    if kind == "ntk" and R > 2:
        base *= factor ** (R / (R - 2))
    f = [base ** (-i / R) for i in range(0, R, 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind == "yarn":
        alpha, beta = float(scaling.get("alpha", 1.0)), float(scaling.get("beta", 32.0))
        if not alpha < beta:
            raise ValueError(f"yarn needs alpha < beta, not {alpha} and {beta}")
        turns = [float(scaling["original"]) * x / (2 * math.pi) for x in f]
        keep = [min(1.0, max(0.0, (r - alpha) / (beta - alpha))) for r in turns]
        f = [x * g + x / factor * (1 - g) for x, g in zip(f, keep)]
        amplitude = float(scaling.get("amplitude", 0.1 * math.log(factor) + 1))
    return f, amplitude


def _layout(t, lead=None):
    """(batch, tokens, batch stride, token stride, head stride) of t [..., heads, dim] as a launch walks over it, with the given
    (batch, tokens) or as its strides allow; None if no such walk exists."""
    s, n = t.stride(), t.dim()
    if n == 3:
        return 1, t.shape[0], 0, s[0], s[1]
    if n == 4:
        return t.shape[0], t.shape[1], s[0], s[1], s[2]
    if n == 2:
        return 1, 1, 0, 0, s[0]
    heads = t.shape[-2:]
    for split in ((lead,) if lead else ((t.shape[0], t.shape[1:-2].numel()), (t.shape[:-3].numel(), t.shape[-3]))):
        try:
            s = t.view(*split, *heads).stride()
            return (*split, s[0], s[1], s[2])
        except RuntimeError:
            pass
    return None


def _args(t, o, lead):
    """What the entry point wants to know of one tensor and its result; (arguments, (batch, tokens))."""
    a = _layout(t, lead)
    if a is None:                                    # it cannot be walked over as the first one is
        if o is t:
            raise ValueError(f"a tensor with strides {t.stride()} cannot be turned in place together with the other one")
        t = t.contiguous()
        a = _layout(t, lead)
    batch, tokens, x0, x1, x2 = a
    y0, y1, y2 = (x0, x1, x2) if o is t or o.stride() == t.stride() else _layout(o, (batch, tokens))[2:]
    return (t.data_ptr(), o.data_ptr(), t.shape[-2], x0, x1, x2, y0, y1, y2), (batch, tokens), t


_NONE = (None, None, 0, 0, 0, 0, 0, 0, 0)


def _turn(positions, frequencies, amplitude, turned, interleaved, inverse, q, k, yq, yk):
    """One launch for up to two tensors of equal leading dimensions; q or k may be None."""
    ref, lead, aq, ak = q, None, _NONE, _NONE
    if q is not None:
        aq, lead, q = _args(q, yq, None)             # (a copy that had to be made lives until the launch)
    else:
        ref = k
    if k is not None:
        ak, lead, k = _args(k, yk, lead)
    if positions.dim() != ref.dim() - 2 or positions.shape != ref.shape[:-2]:
        positions = positions.expand(ref.shape[:-2])
    if not positions.is_contiguous():
        positions = positions.contiguous()
    call_on(ref.device, "vamd_rotary", positions.data_ptr(), positions.dtype == torch.int64, frequencies.data_ptr(), amplitude,
            lead[0], lead[1], ref.shape[-1], turned, interleaved, inverse, *aq, *ak, _TYPES[ref.dtype])


def _readable(t):
    if t is not None:
        if t.is_neg():
            t = t.resolve_neg()                      # a view whose sign torch keeps apart from the memory (tensor.conj().imag)
    return t if t is None or (t.stride(-1) == 1 and (t.dim() <= 4 or _layout(t) is not None)) else t.contiguous()


def _fresh(x):
    """Memory for a result: x's own layout where it is dense and has few leading dimensions, else contiguous."""
    if x is None:
        return None
    y = torch.empty_like(x) if x.dim() <= 4 else None
    return y if y is not None and y.stride(-1) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _turned(positions, frequencies, how, q, k):
    q, k = _readable(q), _readable(k)
    yq, yk = _fresh(q), _fresh(k)
    _turn(positions, frequencies, *how, q, k, yq, yk)
    return yq, yk


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, frequencies, how, q, k):
        ctx.save_for_backward(positions, frequencies)
        ctx.save_for_forward(positions, frequencies)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return _turned(positions, frequencies, how, q, k)

    @staticmethod
    def backward(ctx, gq, gk):
        if not ctx.needs_input_grad[3]:
            gq = None
        if not ctx.needs_input_grad[4]:
            gk = None
        if gq is None and gk is None:
            return None, None, None, None, None
        # the transpose of a turn is the turn back, with the same amplitude: the same function, differentiable in turn
        turn = _RotaryFn.apply if torch.is_grad_enabled() else _turned
        return (None, None, None) + tuple(turn(*ctx.saved_tensors, (*ctx.how[:3], 1 - ctx.how[3]), gq, gk))


    @staticmethod
    def jvp(ctx, _positions, _frequencies, _how, tq, tk):
        # linear: a tangent is turned as its tensor is (forward: q and k both have one, or there is no other)
        turn = _RotaryFn.apply if torch.is_grad_enabled() else _turned
        tq, tk = (t.clone() if t is not None and t._is_zerotensor() else t for t in (tq, tk))    # (zeros that torch keeps without memory)
        return turn(*ctx.saved_tensors, ctx.how, tq, tk)


class Rotary(nn.Module):
    def __init__(self, head_dim, rotary_dim=None, layout="half", base=10000.0, scaling=None, device=None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout {layout!r} (half or interleaved)")
        if rotary_dim % 2 or not 2 <= rotary_dim <= head_dim:
            raise ValueError(f"{rotary_dim} of {head_dim} features cannot be turned (an even number, 2 to the head's size)")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        f, self.amplitude = rotary_frequencies(rotary_dim, base, scaling)
        # radians -> 64-bit fractions of a turn, rounded once; whole turns per position would drop out (none has any)
        turns = [round(Fraction(x) / (2 * _PI) * 2 ** 64) % 2 ** 64 for x in f]
        bits = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
        self.register_buffer("frequencies", bits, persistent=False)
        self._how = (self.amplitude, rotary_dim, int(layout == "interleaved"), 0)

    def _check(self, positions, q, k):
        shape, dtype = q.shape, q.dtype
        if dtype not in _TYPES:
            raise TypeError(f"q is {dtype}: float32 or bfloat16")
        if len(shape) < 2 or shape[-1] != self.head_dim:
            raise ValueError(f"q has shape {tuple(shape)}, not [..., heads, {self.head_dim}]")
        lead, index = shape[:-2], q.get_device()
        if k is not None and (k.dtype != dtype or k.dim() != len(shape) or k.shape[-1] != self.head_dim or k.shape[:-2] != lead or
                              k.get_device() != index):
            raise ValueError(f"q and k differ: {dtype} {tuple(shape)} on {q.device}, {k.dtype} {tuple(k.shape)} on {k.device}")
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"positions are {positions.dtype}: int32 or int64")
        have = positions.shape
        if have != lead and (len(have) > len(lead) or any(n not in (1, m) for n, m in zip(reversed(have), reversed(lead)))):
            raise ValueError(f"positions have shape {tuple(have)}, not {tuple(lead)} or broadcast to it")
        if not q.is_cuda:
            raise RuntimeError("Rotary runs on the GPU only (libvision_amd.so has no CPU path)")
        frequencies = self._buffers["frequencies"]
        if positions.get_device() != index or frequencies.get_device() != index:
            raise ValueError(f"q is on {q.device}, positions on {positions.device}, the frequencies on {frequencies.device}")
        return frequencies

    def forward(self, positions, q, k=None):
        frequencies = self._check(positions, q, k)
        if q.numel() == 0 or (k is not None and k.numel() == 0):
            if k is None:
                return q.clone()
            if q.numel() == 0 and k.numel() == 0:
                return q.clone(), k.clone()
            return (self.forward(positions, q), k.clone()) if k.numel() == 0 else (q.clone(), self.forward(positions, k))
        turn, tangent = _turned, has_tangent(q)
        if k is not None and has_tangent(k) != tangent:      # torch takes no result without a tangent beside one that has it
            return self.forward(positions, q), self.forward(positions, k)
        if tangent or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
            turn = _RotaryFn.apply
        yq, yk = turn(positions, frequencies, self._how, q, k)
        return yq if k is None else (yq, yk)

    def apply_(self, positions, q, k=None):
        """Turns q and k in place and returns them; for inference (no gradient passes through it)."""
        frequencies = self._check(positions, q, k)
        for name, t in (("q", q), ("k", k)):
            if t is None:
                continue
            if torch.is_grad_enabled() and t.requires_grad:
                raise RuntimeError(f"{name} requires a gradient: apply_ is not differentiable, call the module instead")
            if has_tangent(t):
                raise RuntimeError(f"{name} carries a tangent: apply_ is not differentiable, call the module instead")
            if t.numel() and (t.stride(-1) != 1 or _layout(t) is None or self_overlapping(t) or t.is_neg()):
                raise ValueError(f"{name} with strides {t.stride()}{' and a lazy sign' if t.is_neg() else ''} cannot be turned in place")
        if k is not None and overlapping(q, k):
            raise ValueError("q and k are the same memory, or share some of it")
        overwritten(q, k)
        if q.numel() == 0 or (k is not None and k.numel() == 0):
            if k is not None and (q.numel() or k.numel()):
                self.apply_(positions, q if q.numel() else k)
            return q if k is None else (q, k)
        _turn(positions, frequencies, *self._how, q, k, q, k)
        return q if k is None else (q, k)
