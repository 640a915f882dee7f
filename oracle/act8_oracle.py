"""64-bit restatements of the 8-bit activation format and of layer norm, for the tests.

``ln_fwd`` and ``ln_bwd`` also return, per output element, how far an fp32
computation may be from the value before the output's own rounding.  With
u = 2^-24 an n-term fp32 sum in any order is within 4 sqrt(n) u sum|terms| of
the exact one (Higham's sqrt(n) rule with a 4-sigma margin); everything else
is a handful of roundings, each within u of its result.
"""

from __future__ import annotations

import math

import torch

F64 = torch.float64
U = 2.0 ** -24
GROUP = 32


def _groups(x: torch.Tensor) -> torch.Tensor:
    C = x.shape[-1]
    G = -(-C // GROUP)
    full = torch.zeros(*x.shape[:-1], G * GROUP, dtype=F64)
    full[..., :C] = x.to("cpu", F64)
    return full.view(*x.shape[:-1], G, GROUP)


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """codes (..., C) int8 and scales (..., ceil(C / 32)) uint8 of x, on the CPU."""
    C = x.shape[-1]
    v = _groups(x)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    e = torch.frexp(safe).exponent - 1  # 2^e <= top < 2^(e + 1)
    E = torch.where(top == 0, torch.full_like(e, 7), (e + 127).clamp(7, 254))
    E = torch.where(bad, torch.full_like(E, 255), E)
    unit = torch.ldexp(torch.ones_like(top), (E - 133).to(torch.int32))
    q = torch.round(torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0) / unit.unsqueeze(-1)).clamp(-127, 127)
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q)
    return q.flatten(-2)[..., :C].to(torch.int8), E.to(torch.uint8)


def unpack8(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values."""
    E = scales.to("cpu", torch.int32)
    unit = torch.ldexp(torch.ones(E.shape, dtype=F64), E - 133)
    unit = torch.where(E == 255, torch.full_like(unit, math.nan), unit)
    return codes.to("cpu", F64) * unit.repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]


def _ones(x, like):
    return torch.ones(like.shape[-1], dtype=F64) if x is None else x.to("cpu", F64)


def ln_stats(x, eps):
    """mean, rstd and how far fp32 may be off: absolutely for the mean, relatively for rstd."""
    C = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    var = d.square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    dm = (4 * math.sqrt(C) + 2) * U * x.abs().mean(-1, keepdim=True)
    # The variance around a mean that is off by dm is dm^2 too large; rounding of
    # each difference, square and of the sum; then rsqrt (2 ulp).
    dr = 0.5 * ((4 * math.sqrt(C) + 8) * U + dm.square() / (var + eps)) + 4 * U
    # A rounding of x - mean is relative to the difference itself.
    return mean, rstd, dm, dr


def _h(x, mean, rstd, dm, dr):
    h = (x - mean) * rstd
    return h, dm * rstd + h.abs() * (dr + 3 * U)


def ln_fwd(x, weight, bias, eps):
    """(y, error) of layer norm, with x as it is."""
    x = x.to("cpu", F64)
    w = _ones(weight, x)
    b = torch.zeros_like(w) if bias is None else bias.to("cpu", F64)
    h, dh = _h(x, *ln_stats(x, eps))
    return h * w + b, dh * w.abs() + 2 * U * ((h * w).abs() + b.abs())


def ln_bwd(gy, x, kept, weight, eps):
    """{"x", "w", "b": (gradient, error)}; kept: what the backward has of x."""
    gy, x, kept = (t.to("cpu", F64) for t in (gy, x, kept))
    gy, x, kept = (t.reshape(-1, t.shape[-1]) for t in (gy, x, kept))
    T, C = x.shape
    w = _ones(weight, x)
    mean, rstd, dm, dr = ln_stats(x, eps)
    h, dh = _h(kept, mean, rstd, dm, dr)
    g = gy * w
    c1 = g.mean(-1, keepdim=True)
    c2 = (g * h).mean(-1, keepdim=True)
    k = (4 * math.sqrt(C) + 4) * U
    d1 = k * g.abs().mean(-1, keepdim=True)
    d2 = k * (g * h).abs().mean(-1, keepdim=True) + (g.abs() * dh).mean(-1, keepdim=True)
    gx = rstd * (g - c1 - h * c2)
    ex = rstd * (4 * U * (g.abs() + c1.abs() + (h * c2).abs()) + d1 + h.abs() * d2 + dh * c2.abs()) + dr * gx.abs()
    kt = (4 * math.sqrt(T) + 4) * U
    gw, gb = (gy * h).sum(0), gy.sum(0)
    ew = kt * (gy * h).abs().sum(0) + (gy.abs() * dh).sum(0)
    return {"x": (gx, ex), "w": (gw, ew), "b": (gb, kt * gy.abs().sum(0))}


def check(name, out, value, error):
    """out against the 64-bit value: the fp32 error, and half a step of out's type
    (relative to the value; the smallest subnormal below)."""
    o = out.detach().to("cpu", F64).reshape(value.shape)
    info = torch.finfo(out.dtype)
    tol = error + (value.abs() + error) * (info.eps / 2) + info.smallest_normal * info.eps
    bad = ~((o - value).abs() <= tol)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} out of tolerance, worst {float(((o - value).abs() / tol).max()):.3f}")
