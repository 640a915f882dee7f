"""Operators for layers in 8-bit integers and root-mean-square norm, as cases that can be timed and checked.

A case is one pass through one operator of the package, or through two as a layer calls them:

  norm     rms_norm over the last axis, with ``residual`` of x + residual (the sum is an output too);
           with ``train`` forward and backward
  product  linear8: codes with a scale for each token times codes with a scale for each output channel
  linear   pack8_rows, then linear8: a linear layer with 8-bit weights on a 16-bit input
  layer    rms_norm_pack8_rows, then linear8 with the residual: u + F(norm(u)), F in 8 bits

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
EPS = 1e-6
TOP = 127.0  # the largest code
LEAST = 2.0 ** -100  # a row's largest magnitude counts as at least this
PITCH = 16  # rows of codes begin at multiples of this many bytes
DEV = "cuda"
KINDS = ("norm", "product", "linear", "layer")


def listed():
    return [
        # One decoded token through a norm that also adds the residual: latency.
        {"name": "norm_T1_C4096_eval", "kind": "norm", "T": 1, "C": 4096, "dtype": "bf16", "params": "bf16",
         "train": False, "residual": True},
        # A training step's norm between two sublayers, which adds the first one's output to the residual.
        {"name": "norm_T65536_C2048", "kind": "norm", "T": 65536, "C": 2048, "dtype": "bf16", "params": "bf16",
         "train": True, "residual": True},
        # A norm alone, parameters in single precision, at the reference benchmark's default width, ragged batch.
        {"name": "norm_T30011_C2560", "kind": "norm", "T": 30011, "C": 2560, "dtype": "bf16", "params": "fp32",
         "train": True, "residual": False},
        # Single precision, odd width.
        {"name": "norm_T6007_C1001_fp32", "kind": "norm", "T": 6007, "C": 1001, "dtype": "fp32", "params": "fp32",
         "train": True, "residual": True},
        # One decoded token times a square weight: the weight's bytes.
        {"name": "product_T1_N4096_K4096", "kind": "product", "T": 1, "N": 4096, "K": 4096, "dtype": "bf16",
         "bias": False},
        # A training-sized batch at the widest configuration: the matrix cores.
        {"name": "product_T16384_N4096_K4096", "kind": "product", "T": 16384, "N": 4096, "K": 4096, "dtype": "bf16",
         "bias": False},
        # Odd sizes throughout, single-precision output.
        {"name": "product_T2003_N777_K1001_fp32", "kind": "product", "T": 2003, "N": 777, "K": 1001, "dtype": "fp32",
         "bias": True},
        # A batch of decoded tokens through a projection that narrows.
        {"name": "linear_T64_N1024_K4096", "kind": "linear", "T": 64, "N": 1024, "K": 4096, "dtype": "bf16",
         "bias": False},
        # A prompt batch in half precision.
        {"name": "linear_T8192_N2048_K2048_fp16", "kind": "linear", "T": 8192, "N": 2048, "K": 2048, "dtype": "fp16",
         "bias": True},
        # A block's layer for one decoded token.
        {"name": "layer_T1_C4096", "kind": "layer", "T": 1, "N": 4096, "K": 4096, "dtype": "bf16", "bias": False},
        # A ragged prompt.
        {"name": "layer_T257_C2560", "kind": "layer", "T": 257, "N": 2560, "K": 2560, "dtype": "bf16", "bias": True},
        # The microbenchmark's size.
        {"name": "layer_T65536_C1024", "kind": "layer", "T": 65536, "N": 1024, "K": 1024, "dtype": "bf16",
         "bias": False},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    # A third each: the configurations' widths, any multiple of eight, any width.
    pick = rng.randrange(3)
    if pick == 0:
        return rng.choice([256, 512, 1024, 2048, 2560, 4096])
    return 8 * _log_uniform(rng, 2, 512) if pick == 1 else _log_uniform(rng, 9, 4096)


def draw(rng):
    kind = rng.choice(KINDS)
    T = _log_uniform(rng, 1, 131072)
    # Half and single precision now and then; what is packed in the call has 16 bits.
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32" if kind in ("norm", "product") else "fp16"])
    if kind == "norm":
        C = _width(rng)
        # Half precision trains with parameters in single precision.
        params = "bf16" if dtype == "bf16" and rng.random() < 0.5 else "fp32"
        most = 1 << (26 if dtype == "fp32" else 27)  # T times C
        return {"kind": kind, "T": max(1, min(T, most // C)), "C": C, "dtype": dtype, "params": params,
                "train": rng.random() < 0.75, "residual": rng.random() < 0.6}
    N = _width(rng)
    K = N if kind == "layer" else _width(rng)
    T = max(1, min(T, (1 << 38) // (N * K), (1 << 26) // max(N, K)))
    return {"kind": kind, "T": T, "N": N, "K": K, "dtype": dtype, "bias": rng.random() < 0.4}


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


def _activations(rn, T, C, dtype):
    """N(m, 1), every feature with a mean m of its own; every 100th token scaled
    by 100, the outliers that residual streams have."""
    x = rn(T, C, dtype=dtype)
    x += rn(1, C, scale=0.5, dtype=dtype)
    x[::100] *= 100
    return x


def _in_hand(codes):
    """Codes as a program keeps them: rows at a multiple of 16 bytes."""
    rows, K = codes.shape
    kept = codes.new_zeros(rows, -(-K // PITCH) * PITCH)
    kept[:, :K] = codes
    return kept[:, :K]


def _inputs(case, seed):
    rn = _Draws(seed)
    kind, T = case["kind"], case["T"]
    dt = DTYPES[case["dtype"]]
    if kind == "norm":
        C = case["C"]
        s = {"x": _activations(rn, T, C, dt), "w": rn(C, scale=0.1, mean=1.0, dtype=DTYPES[case["params"]])}
        if case["residual"]:
            s["r"] = _activations(rn, T, C, dt)
        if case["train"]:
            s["g"] = rn(T, C, dtype=dt)
            if case["residual"]:
                s["gs"] = rn(T, C, dtype=dt)  # what the sum gets from the layers behind
        return s
    N, K = case["N"], case["K"]
    # A linear layer's weight as it is initialised, in 8 bits with a scale for each output channel.
    wq, ws = _pack_rows((torch.rand(N, K, device=DEV, generator=rn.g) * 2 - 1) / math.sqrt(K))
    s = {"wq": _in_hand(wq), "ws": ws}
    x = _activations(rn, T, K, F32 if kind == "product" else dt)
    if kind == "product":
        xq, s["xs"] = _pack_rows(x)
        s["xq"] = _in_hand(xq)
    else:
        s["x"] = x
    if kind == "layer":
        s["w"] = rn(K, scale=0.1, mean=1.0, dtype=dt)
    if case["bias"]:
        s["b"] = rn(N, scale=0.1, dtype=dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"], s["dtype"] = case["kind"], DTYPES[case["dtype"]]
    if case["kind"] == "norm" and case["train"]:
        s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "r", "w") if k in s]
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _pack_rows(v):
    """codes int8 and scales fp32 of rows v fp32: the largest magnitude is code 127."""
    top = v.abs().amax(-1).clamp(min=LEAST)
    return (v * (TOP / top).unsqueeze(-1)).round().to(torch.int8), top / TOP


def _plain_rms(v, w):
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * rstd * w.float(), rstd


def _plain_norm(s):
    x, w, r, g, gs = (s.get(k) for k in ("x", "w", "r", "g", "gs"))
    dt = x.dtype
    total = x if r is None else (x.float() + r.float()).to(dt)
    v = total.float()
    y, rstd = _plain_rms(v, w)
    out = [y.to(dt)] if r is None else [y.to(dt), total]
    if g is None:
        return out
    h, g = v * rstd, g.float()
    gw = g * w.float()
    gx = rstd * (gw - h * (gw * h).mean(-1, keepdim=True))
    if gs is not None:
        gx += gs.float()
    gx = gx.to(dt)
    return out + ([gx] if r is None else [gx, gx]) + [(g * h).sum(0).to(w.dtype)]


def _plain_linear(xq, xs, wq, ws, b, u, dt):
    out = (xq.float() @ wq.float().t()) * xs.unsqueeze(-1) * ws
    if b is not None:
        out += b.float()
    if u is not None:
        out += u.float()
    return out.to(dt)


def _run_plain(s):
    kind, u = s["kind"], None
    if kind == "norm":
        return _plain_norm(s)
    if kind == "product":
        xq, xs = s["xq"], s["xs"]
    elif kind == "linear":
        xq, xs = _pack_rows(s["x"].float())
    else:
        u = s["x"]
        xq, xs = _pack_rows(_plain_rms(u.float(), s["w"])[0])
    return _plain_linear(xq, xs, s["wq"], s["ws"], s.get("b"), u, s["dtype"])


# ---------------------------------------------------------------------------
# The package's calls


def _run_own(s):
    import flash_mhc

    kind = s["kind"]
    if kind == "norm":
        if "g" not in s:
            with torch.no_grad():
                out = flash_mhc.rms_norm(s["x"], s["w"], EPS, residual=s.get("r"))
            return [out] if "r" not in s else list(out)
        if "r" not in s:
            y = flash_mhc.rms_norm(s["x"], s["w"], EPS)
            return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["g"])]
        y, total = flash_mhc.rms_norm(s["x"], s["w"], EPS, residual=s["r"])
        return [y.detach(), total.detach(), *torch.autograd.grad([y, total], s["leaves"], [s["g"], s["gs"]])]
    if kind == "product":
        xq, xs = s["xq"], s["xs"]
    elif kind == "linear":
        xq, xs = flash_mhc.pack8_rows(s["x"])
    else:
        xq, xs = flash_mhc.rms_norm_pack8_rows(s["x"], s["w"], EPS)
    return flash_mhc.linear8(xq, xs, s["wq"], s["ws"], s.get("b"), residual=s["x"] if kind == "layer" else None,
                             dtype=s["dtype"])


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    kind, T = case["kind"], case["T"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "norm":
        row, params = T * case["C"], (4 if case["params"] == "fp32" else 2) * case["C"]
        more = 1 if case["residual"] else 0
        fwd = 2 * (1 + more) * size * row + params
        if not case["train"]:
            return {"bytes": fwd, "flops": (4 + more) * row}
        # The input (or sum) again, its statistic, the gradients in and out.
        return {"bytes": fwd + (3 + more) * size * row + 2 * 4 * T + 2 * params, "flops": (12 + 2 * more) * row}
    N, K = case["N"], case["K"]
    weight = N * K + 4 * N + (size * N if case["bias"] else 0)
    x = (K + 4 if kind == "product" else size * K) * T
    norm = size * K if kind == "layer" else 0
    return {"bytes": weight + x + norm + size * T * N, "flops": 2 * T * N * K}


# ---------------------------------------------------------------------------
# The same in 64 bits


def _kept_rows(v):
    """What rows of 64-bit values stand for after 8 bits."""
    step = torch.maximum(torch.max(v.abs(), dim=-1, keepdim=True).values, torch.full_like(v[:, :1], LEAST)) / 127
    return torch.round(v / step) * step


def exact(case, seed):
    kind, T = case["kind"], case["T"]
    s = _inputs(case, seed)
    dt = DTYPES[case["dtype"]]
    if kind == "norm":
        C = case["C"]
        if T * C > (1 << 28):
            return None
        v, w = s["x"].to(F64), s["w"].to(F64)
        if case["residual"]:
            v = (v + s["r"].to(F64)).to(dt).to(F64)
        rms = (torch.sum(v * v, dim=1, keepdim=True) / C + EPS).sqrt()
        out = [v / rms * w] + ([v] if case["residual"] else [])
        if not case["train"]:
            return out
        # d/dv_i of sum_c g_c w_c v_c / rms, where d rms / d v_i = v_i / (C rms)
        p = s["g"].to(F64) * w
        gx = p / rms - v * (torch.sum(p * v, dim=1, keepdim=True) / (C * rms.pow(3)))
        gw = torch.sum(s["g"].to(F64) * v / rms, dim=0)
        if case["residual"]:
            gx += s["gs"].to(F64)
            return [*out, gx, gx, gw]
        return [*out, gx, gw]
    N, K = case["N"], case["K"]
    if kind == "product":
        x = s["xq"].to(F64) * s["xs"].to(F64)[:, None]
    else:
        x = s["x"].to(F64)
        if kind == "layer":
            x = x * s["w"].to(F64) / (torch.sum(x * x, dim=1, keepdim=True) / K + EPS).sqrt()
        x = _kept_rows(x)
    out = torch.mm(x, (s["wq"].to(F64) * s["ws"].to(F64)[:, None]).t().contiguous())
    if case["bias"]:
        out += s["b"].to(F64)[None]
    return out + s["x"].to(F64) if kind == "layer" else out
