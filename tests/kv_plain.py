"""Plain 64-bit forms of the rotary positions, the 8-bit cache and the attention over it, on the CPU, element by element in the
order of their definitions (used by the tests of those operators only)."""
import math

import torch

LARGEST = {"e4m3": 448.0, "int8": 127.0}


def rotary(x, positions, frequencies, amplitude, turned, layout, inverse=False):
    """x [..., H, D] -> float64; positions broadcast to x.shape[:-2]; frequencies in radians per position (floats)."""
    x = x.double().cpu()
    y = x.clone()
    angle = positions.double().cpu()[..., None] * torch.tensor(frequencies, dtype=torch.float64)
    angle = angle.expand(*x.shape[:-2], turned // 2)[..., None, :]
    c, s = amplitude * torch.cos(angle), amplitude * torch.sin(angle) * (-1 if inverse else 1)
    if layout == "half":
        i, j = slice(0, turned // 2), slice(turned // 2, turned)
    else:
        i, j = slice(0, turned, 2), slice(1, turned, 2)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def power_scale(top, format):
    """The smallest 2^e (e from -110 on) under which `top` needs no code above the largest; NaN for what is not finite."""
    if not math.isfinite(top):
        return math.nan
    e = -110
    while top > LARGEST[format] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def code(x, format):
    """x (float64) to the nearest code, ties to even."""
    if format == "int8":
        return torch.round(x)
    m, e = torch.frexp(x)                                   # x = m 2^e, 0.5 <= |m| < 1
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 4, min=-9))
    return torch.round(x / step) * step


class Cache:
    """One (sequence, head)'s keys or values after any number of writes: block by block, token by token."""

    def __init__(self, block, format):
        self.block, self.format, self.blocks = block, format, {}

    def append(self, rows, start):
        """rows [n, D] float64 at positions start ..."""
        if start < 0:
            return
        n, i = rows.shape[0], 0
        while i < n:
            b, lo = (start + i) // self.block, (start + i) % self.block
            part = rows[i:i + self.block - lo]
            codes, scale = self.blocks.get(b, (torch.zeros(self.block, rows.shape[1], dtype=torch.float64), 0.0))
            if lo == 0:
                scale = 0.0
            need = power_scale(float(part.abs().max()) if not torch.isnan(part).any() else math.nan, self.format)
            now = math.nan if math.isnan(need) or math.isnan(scale) else max(need, scale)
            if not math.isnan(now):
                if lo > 0 and now != scale:
                    codes = code(codes * (scale / now), self.format)
                codes = codes.clone()
                last = LARGEST[self.format]
                if now * last >= 2.0 ** 128:                # code * scale is read as a float: the last code that is one (e4m3
                    last = 240.0 if self.format == "e4m3" else 63.0   # 240 * 2^120, int8 63 * 2^122; the next ones are 2^128)
                codes[lo:lo + part.shape[0]] = code((part / now).clamp(-last, last), self.format)
            self.blocks[b] = (codes, now)
            i += part.shape[0]

    def read(self, first, count, D):
        out = torch.zeros(count, D, dtype=torch.float64)
        for i in range(count):
            b, t = (first + i) // self.block, (first + i) % self.block
            if b in self.blocks:
                codes, scale = self.blocks[b]
                out[i] = codes[t] * scale
        return out


def attend(q, k, v, length, scale, causal=True, window=0, sinks=0, holes=None):
    """q [n, Hq, D], k, v [>= length, H, D] of one sequence -> (out, sum p |v|, max sum |q k| scale), all float64.
    holes: truth value for each token that is not there."""
    n, Hq, D = q.shape
    H = k.shape[1]
    G = Hq // H
    q, k, v = q.double().cpu(), k[:length].double().cpu(), v[:length].double().cpu()
    j = torch.arange(length)
    p = (length - n + torch.arange(n))[:, None]
    seen = (j <= p) if causal else torch.ones(n, length, dtype=torch.bool)
    if window:
        seen = seen & ((j < sinks) | (p - j < window))
    if holes is not None:
        seen = seen & ~holes[:length]
    out, size, reach = (torch.zeros(n, Hq, D, dtype=torch.float64) for _ in range(3))
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        s = (scale * (q[:, h] @ kh.T)).masked_fill(~seen, -math.inf)
        e = torch.exp(s - torch.where(seen.any(1), s.amax(1) if length else torch.zeros(n), torch.zeros(n, dtype=torch.float64))[:, None])
        e = e.masked_fill(~seen, 0.0)
        total = e.sum(1, keepdim=True)
        w = e / torch.where(total == 0, 1.0, total)
        vs = torch.where(seen.any(0)[:, None], vh, 0.0)
        out[:, h] = w @ vs
        size[:, h] = w @ vs.abs()
        if length:
            reach[:, h] = (abs(scale) * (q[:, h].abs() @ kh.abs().T)).masked_fill(~seen, 0.0).amax(1)[:, None]
    return out, size, reach


def attend_bound(out, size, reach, length, D, dtype):
    """How far a result may be off, element by element.  Roundings: u = half a step relative to the value (2^-24 in 32 bits, 2^-8 in
    bf16).  A score is a sum of D products in fp32 in some order, times a scale: (D + 4) u32 of sum |q k|; it moves exp by as much,
    in the numerator and in the sum; the exponential itself and the steps of the running maximum (one factor each per 64 tokens)
    and the sums over `length` terms: (length + length / 32 + 16) u32 in each.  bf16: the probabilities are rounded once (2^-8) and
    the result is (2^-8)."""
    u = 2.0 ** -24
    rel = 2 * (D + 4) * u * reach + 2 * (length + length / 32 + 16) * u
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * (out.abs() + size) + (1 + 2.0 ** -7) * rel * size + 1e-30
    return u * out.abs() + rel * size + 1e-30
