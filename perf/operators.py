"""Operators for 8-bit activation checkpoints and layer norm, as cases that can be timed and checked.

A case is one pass through one operator of the package:

  pack      pack8 then unpack8: a tensor to block-scaled 8 bits and back (groups of 32 columns share a power of two)
  post_res  the post-residual mix whose backward keeps x and the layer output in 8 bits: output and every gradient
  project   the backward of the RMSNorm + projection from x kept in 8 bits: the gradients of x and W
  norm      layer norm; with ``train`` forward and backward, ``bits`` 8 keeps its input in 8 bits for the backward

With ``own`` false, ``run`` computes a case in elementary torch operations in 32 bits, rounded once at the end; with
``own`` true it calls the package.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "flash-mhc_amd"))

own = False

BF16 = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
N = 4
D = 32  # width of the projection, 2 n + n!
GROUP = 32  # columns that share a scale
LN_EPS = 1e-5
RMS_EPS = 1e-6
DEV = "cuda"
KINDS = ("pack", "post_res", "project", "norm")


def listed():
    return [
        # The streams of a handful of tokens: the latency of two launches.
        {"name": "pack_T4_C1024_bf16", "kind": "pack", "T": 4, "C": 1024, "dtype": "bf16"},
        # The streams of a training batch, kept by one block until its backward.
        {"name": "pack_T32768_C2048_bf16", "kind": "pack", "T": 32768, "C": 2048, "dtype": "bf16"},
        # Streams in single precision at an odd width and token count.
        {"name": "pack_T6007_C1001_fp32", "kind": "pack", "T": 6007, "C": 1001, "dtype": "fp32"},
        # The post-residual mix of a small training step.
        {"name": "post_res_T1024_C1024", "kind": "post_res", "T": 1024, "C": 1024},
        # The same at the microbenchmark's size.
        {"name": "post_res_T65536_C1024", "kind": "post_res", "T": 65536, "C": 1024},
        # A small model's width that is no multiple of the group, ragged batch.
        {"name": "post_res_T20011_C300", "kind": "post_res", "T": 20011, "C": 300},
        # The projection's backward at the training width.
        {"name": "project_T16384_C4096", "kind": "project", "T": 16384, "C": 4096},
        # The same, few tokens, odd width.
        {"name": "project_T2003_C1001", "kind": "project", "T": 2003, "C": 1001},
        # One decoded token through a norm: latency.
        {"name": "norm_T1_C4096_eval", "kind": "norm", "T": 1, "C": 4096, "dtype": "bf16", "params": "bf16",
         "train": False, "bits": 16},
        # A training step's norm.
        {"name": "norm_T65536_C2048", "kind": "norm", "T": 65536, "C": 2048, "dtype": "bf16", "params": "bf16",
         "train": True, "bits": 16},
        # The same with its input kept in 8 bits and parameters in single precision, at the reference benchmark's
        # default width, ragged batch.
        {"name": "norm_T30011_C2560_8bit", "kind": "norm", "T": 30011, "C": 2560, "dtype": "bf16", "params": "fp32",
         "train": True, "bits": 8},
        # Single precision, odd width, small batch.
        {"name": "norm_T1003_C777_fp32", "kind": "norm", "T": 1003, "C": 777, "dtype": "fp32", "params": "fp32",
         "train": True, "bits": 16},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(KINDS)
    # A third each: the configurations' widths, any multiple of eight, any width.
    pick = rng.randrange(3)
    if pick == 0:
        C = rng.choice([256, 512, 1024, 2048, 2560, 4096])
    elif pick == 1:
        C = 8 * _log_uniform(rng, 2, 512)
    else:
        C = _log_uniform(rng, 9, 4096)
    case = {"kind": kind, "T": 0, "C": C}
    most = 1 << (27 if kind == "norm" else 26)  # T times C
    if kind in ("pack", "norm"):
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most //= 2 if case["dtype"] == "fp32" else 1
    if kind == "norm":
        # Half precision trains with parameters in single precision.
        case["params"] = "bf16" if case["dtype"] == "bf16" and rng.random() < 0.5 else "fp32"
        case["train"] = rng.random() < 0.75
        case["bits"] = rng.choice([8, 16]) if case["train"] else 16
    case["T"] = max(1, min(_log_uniform(rng, 1, 131072), most // C))
    return case


# ---------------------------------------------------------------------------
# Inputs


class _Draws:
    """Seeded normal tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def __call__(self, *shape, scale=1.0, mean=0.0, dtype=BF16):
        t = torch.randn(shape, device=DEV, dtype=dtype if dtype is BF16 else F32, generator=self.g)
        if scale != 1.0:
            t *= scale
        if mean != 0.0:
            t += mean
        return t.to(dtype)


def _streams(rn, T, C, dtype=BF16):
    """x ~ N(m, 1), every feature with a mean m of its own; every 100th token
    scaled by 100, the outliers that residual streams have."""
    x = rn(T, N, C, dtype=dtype)
    x += rn(1, N, C, scale=0.5, dtype=dtype)
    x[::100] *= 100
    return x


def _inputs(case, seed):
    rn = _Draws(seed)
    kind, T, C = case["kind"], case["T"], case["C"]
    if kind == "pack":
        return {"x": _streams(rn, T, C, DTYPES[case["dtype"]])}
    if kind == "post_res":
        h_post = 2.0 * torch.sigmoid(rn(T, N, dtype=F32))
        H = torch.softmax(rn(T, N, N, dtype=F32), dim=-1) - h_post.unsqueeze(-1) * torch.sigmoid(rn(T, 1, N, dtype=F32))
        return {"x": _streams(rn, T, C), "lo": rn(T, C), "H": H, "h_post": h_post, "g": rn(T, N, C)}
    if kind == "project":
        x = _streams(rn, T, C)
        W = rn(D, N * C, scale=0.02)
        # What the forward has left: the projection, 1 / rms, and x in 8 bits.
        xf = x.view(T, N * C)
        inv = torch.cat([torch.rsqrt(p.float().square().mean(-1) + RMS_EPS) for p in xf.split(16384)])
        proj = (inv.unsqueeze(-1) * (xf @ W.t()).float()).to(BF16)
        codes, scales = _pack(x)
        return {"codes": codes, "scales": scales, "W": W, "proj": proj, "inv": inv, "g": rn(T, D)}
    dt = DTYPES[case["dtype"]]
    x = rn(T, C, dtype=dt)
    x += rn(1, C, scale=0.5, dtype=dt)
    x[::100] *= 100
    pt = DTYPES[case["params"]]
    return {"x": x, "w": rn(C, scale=0.1, mean=1.0, dtype=pt), "b": rn(C, scale=0.1, dtype=pt),
            "g": rn(T, C, dtype=dt) + rn(1, C, scale=0.5, dtype=dt)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"] = case["kind"]
    if case["kind"] == "post_res":
        s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "lo", "H", "h_post")]
    elif case["kind"] == "norm":
        s["train"], s["bits"] = case["train"], case["bits"]
        if case["train"]:
            s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "w", "b")]
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _pack(x):
    """codes (..., C) int8 and scales (..., ceil(C / 32)) uint8: the group's
    largest magnitude gives the exponent E, an element is code 2^(E - 133)."""
    C = x.shape[-1]
    groups = -(-C // GROUP)
    v = torch.nn.functional.pad(x.float(), (0, groups * GROUP - C)).unflatten(-1, (groups, GROUP))
    E = (v.abs().amax(-1).view(torch.int32) >> 23).clamp(7, 254)
    codes = (v / _unit(E).unsqueeze(-1)).round().clamp(-127, 127)
    return codes.flatten(-2)[..., :C].to(torch.int8).contiguous(), E.to(torch.uint8)


def _unit(E):
    # 2^(E - 133), whose exponent field is E - 6: pow and ldexp on the GPU are not exact.
    return ((E.to(torch.int32) - 6) << 23).view(F32)


def _unpack(codes, scales):
    unit = _unit(scales).repeat_interleave(GROUP, dim=-1)[..., :codes.shape[-1]]
    return codes.float() * unit


def _plain_post_res(x, lo, H, h_post, g):
    out = torch.matmul(H, x.float()) + h_post.unsqueeze(-1) * lo.float().unsqueeze(1)
    # The backward has x and lo as they were kept.
    xk, lk, g = _unpack(*_pack(x)), _unpack(*_pack(lo)), g.float()
    gx = torch.matmul(H.transpose(1, 2).contiguous(), g)
    glo = (h_post.unsqueeze(-1) * g).sum(1)
    gH = torch.matmul(g, xk.transpose(1, 2).contiguous())
    ghp = (g * lk.unsqueeze(1)).sum(-1)
    return out.to(BF16), gx.to(BF16), glo.to(BF16), gH, ghp


def _plain_project(codes, scales, W, proj, inv, g):
    x = _unpack(codes, scales).flatten(1)
    g, W, inv = g.float(), W.float(), inv.unsqueeze(-1)
    s = (g * proj.float()).sum(-1, keepdim=True) * inv.square() / x.shape[1]
    gx = inv * (g @ W) - s * x
    gW = (g * inv).t().contiguous() @ x
    return gx.to(BF16).view(codes.shape), gW.to(BF16)


def _plain_norm(x, w, b, g, train, bits):
    v = x.float()
    mean = v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + LN_EPS)
    y = ((v - mean) * rstd * w.float() + b.float()).to(x.dtype)
    if not train:
        return y
    h = ((_unpack(*_pack(x)) if bits == 8 else v) - mean) * rstd
    g = g.float()
    gw = g * w.float()
    gx = rstd * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    return y, gx.to(x.dtype), (g * h).sum(0).to(w.dtype), g.sum(0).to(b.dtype)


def _run_plain(s):
    kind = s["kind"]
    if kind == "pack":
        return _unpack(*_pack(s["x"])).to(s["x"].dtype)
    if kind == "post_res":
        return _plain_post_res(s["x"], s["lo"], s["H"], s["h_post"], s["g"])
    if kind == "project":
        return _plain_project(s["codes"], s["scales"], s["W"], s["proj"], s["inv"], s["g"])
    return _plain_norm(s["x"], s["w"], s["b"], s["g"], s["train"], s["bits"])


# ---------------------------------------------------------------------------
# The package's calls


def _run_own(s):
    import flash_mhc

    ops = torch.ops.flash_mhc
    kind = s["kind"]
    if kind == "pack":
        codes, scales = flash_mhc.pack8(s["x"])
        return flash_mhc.unpack8(codes, scales, s["x"].dtype)
    if kind == "post_res":
        out = ops.fused_post_res_pack8(s["x"], s["lo"], s["H"], s["h_post"])[0]
        return (out.detach(), *torch.autograd.grad(out, s["leaves"], s["g"]))
    if kind == "project":
        return ops.fused_rmsnorm_project_bwd_pack8(s["g"], s["codes"], s["scales"], s["W"], s["proj"], s["inv"])
    if not s["train"]:
        with torch.no_grad():
            return flash_mhc.layer_norm(s["x"], s["w"], s["b"], LN_EPS)
    y = flash_mhc.layer_norm(s["x"], s["w"], s["b"], LN_EPS, activation_bits=s["bits"])
    return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["g"]))


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    kind, T, C = case["kind"], case["T"], case["C"]
    x = T * N * C
    kept = T * N * (C + -(-C // GROUP))  # the streams in 8 bits
    row = T * C
    row_kept = T * (C + -(-C // GROUP))
    if kind == "pack":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * size * x + 2 * kept, "flops": 2 * x}
    if kind == "post_res":
        coef = 4 * T * (N + N * N)
        fwd = 2 * x + 2 * row + coef + 2 * x + kept + row_kept
        bwd = 2 * x + kept + row_kept + coef + 2 * x + 2 * row + coef
        return {"bytes": fwd + bwd, "flops": (2 + 4) * T * N * (N + 1) * C}
    if kind == "project":
        w = 2 * D * N * C
        return {"bytes": kept + 2 * x + 2 * w + T * (4 * D + 4), "flops": 4 * T * D * N * C}
    size = 4 if case["dtype"] == "fp32" else 2
    params = (4 if case["params"] == "fp32" else 2) * C
    fwd = 2 * size * row + 2 * params
    if not case["train"]:
        return {"bytes": fwd, "flops": 7 * row}
    kept_bytes = (row_kept, row_kept) if case["bits"] == 8 else (0, size * row)  # written, read
    stats = 2 * 8 * T
    return {"bytes": fwd + kept_bytes[0] + kept_bytes[1] + stats + 2 * size * row + 3 * params, "flops": 20 * row}


# ---------------------------------------------------------------------------
# The same in 64 bits


def _power_of_two(e):
    return ((e.to(torch.int64) + 1023) << 52).view(F64)


def _kept(x):
    """What a tensor of 64-bit values stands for after 8 bits."""
    C = x.shape[-1]
    full = x.new_zeros(*x.shape[:-1], -(-C // GROUP) * GROUP)
    full[..., :C] = x
    v = full.view(*x.shape[:-1], -1, GROUP)
    top = v.abs().max(dim=-1, keepdim=True).values
    # 2^e <= top < 2^(e + 1): frexp gives top = m 2^(e + 1), m in [1/2, 1).
    e = torch.where(top > 0, torch.frexp(top).exponent - 1, torch.full_like(top, -1000).int()).clamp(-120, 127)
    step = _power_of_two(e - 6)
    q = torch.minimum(torch.maximum(torch.round(v / step), torch.full_like(top, -127.0)), torch.full_like(top, 127.0))
    return (q * step).view(full.shape)[..., :C]


def exact(case, seed):
    kind, T, C = case["kind"], case["T"], case["C"]
    if T * C * (1 if kind == "norm" else N) > (1 << 28):
        return None
    s = _inputs(case, seed)
    d = {k: v.to(F64) for k, v in s.items()}
    if kind == "pack":
        return _kept(d["x"])
    if kind == "post_res":
        x, lo, H, hp, g = (d[k] for k in ("x", "lo", "H", "h_post", "g"))
        del d
        out = hp.unsqueeze(-1) * lo.unsqueeze(1)
        for j in range(N):
            out += H[:, :, j:j + 1] * x[:, j:j + 1]
        xk, lk = _kept(x), _kept(lo)
        gx, gH = torch.zeros_like(x), torch.empty_like(H)
        for i in range(N):
            gx += H[:, i].unsqueeze(-1) * g[:, i:i + 1]
            gH[:, i] = (g[:, i:i + 1] * xk).sum(-1)
        return out, gx, (hp.unsqueeze(-1) * g).sum(1), gH, (g * lk.unsqueeze(1)).sum(-1)
    if kind == "project":
        x = (d["codes"] * torch.repeat_interleave(_power_of_two(d["scales"] - 133), GROUP, dim=-1)[..., :C]).reshape(T, N * C)
        a = d["inv"].unsqueeze(-1) * d["g"]
        # d/dx of sum_d g_d proj_d with proj = (x W^T) / rms(x)
        gx = a @ d["W"] - x * ((a * d["proj"]).sum(-1) * d["inv"] / (N * C)).unsqueeze(-1)
        return gx.view(T, N, C), a.t() @ x
    x, w, b, g = (d[k] for k in ("x", "w", "b", "g"))
    mu = x.sum(-1, keepdim=True) / C
    sd = ((x - mu).pow(2).sum(-1, keepdim=True) / C + LN_EPS).sqrt()
    y = (x - mu) / sd * w + b
    if not case["train"]:
        return y
    h = ((_kept(x) if case["bits"] == 8 else x) - mu) / sd
    p = g * w
    gx = (p - (p.sum(-1, keepdim=True) + h * (p * h).sum(-1, keepdim=True)) / C) / sd
    return y, gx, torch.sum(g * h, dim=0), torch.sum(g, dim=0)
