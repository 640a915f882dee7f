"""Test-only CPU stand-ins for the launchers of RMS norm and of rows in 8 bits (see pack8_cpu_kernels):
formulas in 64 bits, rounded once."""

from __future__ import annotations

from contextlib import contextmanager

import torch

import flash_mhc
from flash_mhc import block, kernels, norm, ops, rows8
from oracle import rows8_oracle as R

F32 = torch.float32


def _sum(x, residual):
    return None if residual is None else R.add(x, residual)


def rms_norm_fwd(x, residual, weight, eps, stats=True):
    total = _sum(x, residual)
    s = (x if total is None else total).double()
    rstd = (s.square().mean(-1) + eps).rsqrt().to(F32)
    return R.rms_fwd(s, weight, eps)[0].to(x.dtype), total, rstd


def rms_norm_bwd(gy, x, rstd, weight, pdt, need_weight=True, grad_x_in=None):
    C = gy.shape[-1]
    h, g = x.double() * rstd.double().unsqueeze(-1), gy.double() * (1 if weight is None else weight.double())
    gx = rstd.double().unsqueeze(-1) * (g - h * (g * h).mean(-1, keepdim=True))
    if grad_x_in is not None:
        gx = gx + grad_x_in.double()
    return gx.to(gy.dtype), (gy.double() * h).reshape(-1, C).sum(0).to(pdt) if need_weight else None


def _at_pitch(codes):
    out, _scales = kernels.empty_rows(torch.empty(codes.shape))
    return out.copy_(codes)


def pack8_rows(x):
    codes, scales = R.pack_rows(x)
    return _at_pitch(codes), scales


def rms_norm_pack8_rows(x, residual, weight, eps):
    total = _sum(x, residual)
    codes, scales = R.pack_rows(R.rms_fwd(x if total is None else total, weight, eps)[0].float())
    return _at_pitch(codes), scales, total


def linear8(codes, scales, weight_codes, weight_scales, bias=None, residual=None, dtype=torch.bfloat16):
    return R.linear8(codes, scales, weight_codes, weight_scales, bias, residual)[0].to(dtype)


def _registered_bwd(gy, gi, x, rstd, weight, need_weight):
    pdt = F32 if weight is None else weight.dtype
    gx, gw = rms_norm_bwd(gy, x, rstd, weight, pdt, need_weight, gi)
    return gx, gy.new_empty((0,), dtype=pdt) if gw is None else gw


REGISTERED = {
    "rms_norm": lambda x, w, eps: rms_norm_fwd(x, None, w, eps)[::2],
    "add_rms_norm": rms_norm_fwd,
    "rms_norm_backward": _registered_bwd,
    "pack8_rows": pack8_rows,
    "rms_norm_pack8_rows": lambda x, w, eps: rms_norm_pack8_rows(x, None, w, eps)[:2],
    "add_rms_norm_pack8_rows": rms_norm_pack8_rows,
    "linear8": linear8,
}


def eager(monkeypatch):
    """The eager paths on CPU tensors."""
    for module in (block, norm):
        monkeypatch.setattr(module, "_plain_eager", lambda x: True)
    monkeypatch.setattr(norm.RMSNorm, "_on_kernels", lambda self, x: True)
    monkeypatch.setattr(rows8.Linear8, "on_kernels", lambda self, x: True)
    for name, fn in (("rms_norm_fwd", rms_norm_fwd), ("rms_norm_bwd", rms_norm_bwd), ("pack8_rows", pack8_rows),
                     ("rms_norm_pack8_rows", rms_norm_pack8_rows), ("linear8", linear8)):
        monkeypatch.setattr(kernels, name, fn)


@contextmanager
def registered():
    """The ops on CPU tensors."""
    lib = torch.library.Library("flash_mhc", "IMPL")
    try:
        for name, fn in REGISTERED.items():
            lib.impl(name, ops.backward_op(fn) if "backward" in name else ops.without_tangents(fn), "CPU")
        yield
    finally:
        lib._destroy()


def make_block(C, norm="rms", seed=0, layer=None, dtype=torch.bfloat16, **kw):
    torch.manual_seed(seed)
    layer = layer or flash_mhc.Linear8.from_linear(torch.nn.Linear(C, C))
    return flash_mhc.MHCLiteBlock(4, C, layer, pre_norm=norm, **kw).to(dtype)
