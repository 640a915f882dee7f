"""Test-only CPU stand-ins for the launchers of the 8-bit activation and layer norm operators.

They let the autograd around the kernels (Functions, registered formulas, what is
kept and checked between forward and backward) run without a GPU: formulas in
64 bits, rounded once.  ``eager`` puts them in place of the launchers that the
eager Functions call, ``registered`` behind the ops' CPU key."""

from __future__ import annotations

from contextlib import contextmanager

import torch

import flash_mhc
from flash_mhc import activation8, block, kernels, norm, ops
from oracle import act8_oracle as A
from oracle_cpu_ops import _k1_bwd, _k4, _k4_bwd, _pre_map, _pre_map_bwd

F32 = torch.float32


def _unpack(codes, scales, dtype):
    return A.unpack8(codes, scales).to(dtype)


def layer_norm_fwd(x, weight, bias, eps, stats=True, packed=False):
    mean, rstd, _dm, _dr = A.ln_stats(x.double(), eps)
    y = A.ln_fwd(x, weight, bias, eps)[0].to(x.dtype)
    return (y, mean.squeeze(-1).to(F32), rstd.squeeze(-1).to(F32), *(A.pack8(x) if packed else (None, None)))


def layer_norm_fwd_joint(x, weight, bias, eps, packed):
    y, mean, rstd, codes, scales = layer_norm_fwd(x, weight, bias, eps, packed=packed)
    return y, torch.cat([mean.flatten(), rstd.flatten()]), codes, scales, norm._param_dtype(weight, bias)


def _ln_bwd(gy, x, codes, scales, mean, rstd, weight, pdt, need_weight, need_bias, gi):
    C = gy.shape[-1]
    h = ((x.double() if x is not None else A.unpack8(codes, scales)) - mean.double()) * rstd.double()
    g = gy.double() * (1 if weight is None else weight.double())
    gx = rstd.double() * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    gx = gx.to(gy.dtype)
    if gi is not None:
        gx = gi + gx
    rows = lambda t: t.reshape(-1, C).sum(0).to(pdt)
    return gx, rows(gy.double() * h) if need_weight else None, rows(gy.double()) if need_bias else None


def layer_norm_bwd(gy, x, codes, scales, mean, rstd, weight, pdt, need_weight=True, need_bias=True, grad_x_in=None):
    return _ln_bwd(gy, x, codes, scales, mean.unsqueeze(-1), rstd.unsqueeze(-1), weight, pdt, need_weight, need_bias,
                   grad_x_in)


def layer_norm_bwd_joint(gy, x, codes, scales, stats, weight, pdt, need_weight, need_bias, grad_x_in=None):
    mean, rstd = (t.view(*gy.shape[:-1], 1) for t in stats.chunk(2))
    return _ln_bwd(gy, x, codes, scales, mean, rstd, weight, pdt, need_weight, need_bias, grad_x_in)


def k4_fwd_pack8(x, lo, H, hp, pack_x=True, residual=None):
    if residual is not None:
        lo = residual + lo
    return (_k4(x, lo, H, hp), *(A.pack8(x) if pack_x else (None, None)), *A.pack8(lo))


def k4_bwd_pack8(go, xq, xs, lq, ls, H, hp):
    return _k4_bwd(go, _unpack(xq, xs, go.dtype), _unpack(lq, ls, go.dtype), H, hp)


def pre_map_bwd_pack8(g_li, g_H, g_hp, g_hpre, g_proj, g_sink, xq, xs, W, ap, apo, ar, b, perm, h_pre, proj, inv):
    return _pre_map_bwd(g_li, g_H, g_hp, g_hpre, g_proj, g_sink, _unpack(xq, xs, proj.dtype), W, ap, apo, ar, b, perm,
                        h_pre, proj, inv)


def _project_bwd(go, xq, xs, W, proj, inv):
    gx, gW = _k1_bwd(go, _unpack(xq, xs, go.dtype).flatten(1), W, proj, inv)
    return gx.view(xq.shape), gW


def _registered_ln_bwd(gy, x, codes, scales, mean, rstd, weight, pdt, need_weight, need_bias):
    gx, gw, gb = layer_norm_bwd(gy, x, codes, scales, mean, rstd, weight, pdt, need_weight, need_bias)
    none = lambda t: gy.new_empty((0,), dtype=pdt) if t is None else t
    return gx, none(gw), none(gb)


def _registered_post_res(x, sink, xq, xs, lo, H, hp):
    out, _q, _s, lq, ls = k4_fwd_pack8(x, lo, H, hp, pack_x=False)
    return out, lq, ls


REGISTERED = {
    "pack8": lambda x: A.pack8(x),
    "layer_norm": lambda x, w, b, eps: layer_norm_fwd(x, w, b, eps)[:3],
    "layer_norm_pack8": lambda x, w, b, eps: layer_norm_fwd(x, w, b, eps, packed=True),
    "layer_norm_backward": _registered_ln_bwd,
    "fused_post_res_pack8_traced": k4_fwd_pack8,
    "fused_post_res_backward_pack8": k4_bwd_pack8,
    "fused_rmsnorm_project_bwd_pack8": _project_bwd,
    "mhc_pre_map_pack8": lambda x, *params: (*_pre_map(x, *params), *A.pack8(x)),
    "mhc_pre_map_backward_pack8": pre_map_bwd_pack8,
    "mhc_post_res_pack8": _registered_post_res,
}


def eager(monkeypatch):
    """The eager Functions on CPU tensors."""
    for module in (block, norm):
        monkeypatch.setattr(module, "_plain_eager", lambda x: True)
    monkeypatch.setattr(norm.LayerNorm, "_on_kernels", lambda self, x: True)
    monkeypatch.setattr(activation8, "_mhc_pre_map_cuda", _pre_map)
    monkeypatch.setattr(activation8, "_mhc_pre_map_backward_pack8_cuda", pre_map_bwd_pack8)
    for name, fn in (("layer_norm_fwd", layer_norm_fwd), ("layer_norm_fwd_joint", layer_norm_fwd_joint),
                     ("layer_norm_bwd_joint", layer_norm_bwd_joint), ("k4_fwd_pack8", k4_fwd_pack8),
                     ("k4_bwd_pack8_saved", k4_bwd_pack8)):
        monkeypatch.setattr(kernels, name, fn)


@contextmanager
def registered():
    """The ops on CPU tensors."""
    lib = torch.library.Library("flash_mhc", "IMPL")
    try:
        for name, fn in REGISTERED.items():
            if name != "pack8":
                fn = ops.backward_op(fn) if "backward" in name or "bwd" in name else ops.without_tangents(fn)
            lib.impl(name, fn, "CPU")
        yield
    finally:
        lib._destroy()


def make_block(C, seed=0, layer=None, dtype=torch.bfloat16, **kw):
    torch.manual_seed(seed)
    blk = flash_mhc.MHCLiteBlock(4, C, layer or torch.nn.Linear(C, C), activation_bits=8, **kw).to(dtype)
    with torch.no_grad():
        blk.alpha_pre.fill_(0.8)
        blk.alpha_post.fill_(1.2)
        blk.alpha_res.fill_(1.7)
    return blk
