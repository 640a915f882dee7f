"""64-bit restatements of RMS norm and of products of rows in 8 bits, for the tests.

As in ``act8_oracle``, values come with how far an fp32 computation may be from them
before the output's own rounding: with u = 2^-24 an n-term fp32 sum in any order is
within 4 sqrt(n) u sum|terms| of the exact one (Higham's sqrt(n) rule with a 4-sigma
margin); everything else is a handful of roundings, each within u of its result.
"""

from __future__ import annotations

import math

import torch

F64 = torch.float64
U = 2.0 ** -24
LEAST = 2.0 ** -100


def _w(weight, x):
    return torch.ones(x.shape[-1], dtype=F64) if weight is None else weight.to("cpu", F64)


def add(x, residual):
    """x + residual as the norm keeps it: one fp32 addition, rounded to x's dtype."""
    return (x.cpu().float() + residual.cpu().float()).to(x.dtype)


def _stat(s, eps):
    """rstd and how far fp32 may be off, relatively: the sum of squares (no
    cancellation), its product with 1 / C, the addition of eps, and rsqrt (2 ulp)."""
    ms = s.square().mean(-1, keepdim=True)
    return (ms + eps).rsqrt(), 0.5 * (4 * math.sqrt(s.shape[-1]) + 6) * U + 4 * U


def rms_fwd(s, weight, eps):
    """(y, error) of the norm of s (x, or its sum with the residual)."""
    s = s.to("cpu", F64)
    rstd, dr = _stat(s, eps)
    y = s * rstd * _w(weight, s)
    return y, y.abs() * (dr + 3 * U)


def rms_bwd(gy, s, weight, eps, gs=None):
    """{"x", "w": (gradient, error)}; gs: the sum's other gradient."""
    gy, s = (t.to("cpu", F64).reshape(-1, t.shape[-1]) for t in (gy, s))
    T, C = s.shape
    rstd, dr = _stat(s, eps)
    h, g = s * rstd, gy * _w(weight, s)
    c = (g * h).mean(-1, keepdim=True)
    # h is off by dr + U, g by U, their sum by the rule, and the division by C.
    dc = ((4 * math.sqrt(C) + 4) * U + dr + 2 * U) * (g * h).abs().mean(-1, keepdim=True)
    gx = rstd * (g - h * c)
    ex = (rstd * g).abs() * (dr + 3 * U) + (rstd * h * c).abs() * (2 * dr + 6 * U) + rstd * h.abs() * dc
    if gs is not None:
        gs = gs.to("cpu", F64).reshape(-1, C)
        gx = gx + gs
        ex = ex + 2 * U * (gs.abs() + gx.abs())
    gw = (gy * h).sum(0)
    ew = ((4 * math.sqrt(T) + 4) * U + dr + 2 * U) * (gy * h).abs().sum(0)
    return {"x": (gx, ex), "w": (gw, ew)}


def pack_rows(x):
    """codes and scales of rows, in fp32 as the format says (IEEE operations: the bits)."""
    v = x.cpu().float()
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    top = top.clamp(min=LEAST)
    codes = torch.round(v * (torch.full_like(top, 127.0) / top).unsqueeze(-1))
    codes = torch.where(bad.unsqueeze(-1), torch.zeros_like(codes), codes)
    return codes.to(torch.int8), torch.where(bad, torch.full_like(top, math.nan), top / 127.0)


def check_rows(codes, scales, y, error):
    """codes and scales against the rows' 64-bit values y, which fp32 has within error:
    the scale is the largest magnitude's 127th, and a code is off by half a scale, plus
    what the value, 127 / top and the product are off by."""
    q, sc = codes.detach().to("cpu", F64), scales.detach().to("cpu", F64)
    top, i = y.abs().max(-1)
    dtop = torch.gather(error, -1, i.unsqueeze(-1)).squeeze(-1) + 2 * U * top
    assert bool(((sc * 127 - top.clamp(min=LEAST)).abs() <= dtop + 2 * U * top.clamp(min=LEAST)).all())
    assert int(q.abs().max()) <= 127
    off = (q * sc.unsqueeze(-1) - y).abs()
    tol = sc.unsqueeze(-1) * (0.5 + 127 * 4 * U) + error + y.abs() * (dtop / top.clamp(min=LEAST)).unsqueeze(-1)
    assert bool((off <= tol).all()), float((off / tol).max())


def linear8(codes, scales, weight_codes, weight_scales, bias=None, residual=None):
    """(out, error): the integers' sum is exact; its rounding to fp32, the two scales'
    products, bias and residual."""
    q, w = codes.cpu(), weight_codes.cpu()
    lead = q.shape[:-1]
    acc = (q.reshape(-1, q.shape[-1]).double() @ w.double().t()).reshape(*lead, w.shape[0])  # exact below 2^53
    out = acc * scales.cpu().double().unsqueeze(-1) * weight_scales.cpu().double()
    err = 3 * U * out.abs()
    for t in (bias, residual):
        if t is not None:
            out = out + t.cpu().double()
            err = err + U * (out.abs() + t.cpu().double().abs())
    return out, err
