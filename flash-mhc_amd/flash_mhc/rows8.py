"""Layers in 8-bit integers: rows as codes with one scale each, and their product.

A row (a token's activations, an output channel's weights) is kept as int8 codes
with an fp32 scale, its largest magnitude being code 127 (the format is defined in
``include/flash_mhc_hip.h``).  A product of such rows is a sum of integers, exact,
times the two rows' scales:

  pack8_rows            a tensor (..., C) to codes and scales
  rms_norm_pack8_rows   the same of its RMS norm, in the norm's pass
  linear8               codes times an 8-bit weight, with bias and residual
  Linear8               the module, made from an ``nn.Linear``

They serve inference: the backward of each raises, on any device.  ``MHCLiteBlock(pre_norm="rms")``
around a ``Linear8`` runs rms_norm_pack8_rows and linear8 with the block's residual.

Codes of rows whose length is no multiple of 16 lie at the next multiple's pitch, so
they are not contiguous; linear8 takes any strides, and copies codes whose rows do
not begin at multiples of 16 bytes.

No counterpart in the reference.
"""

from __future__ import annotations

import torch
import torch.library
import torch.nn as nn
import torch.nn.functional as F

from . import block as _block  # which imports this module: its names are read at call time
from . import kernels as _k
from .ops import _forward_ad, refuse_tangents, without_tangents

_lib = torch.library.Library("flash_mhc", "FRAGMENT")

_lib.define("pack8_rows(Tensor x) -> (Tensor codes, Tensor scales)")
_lib.define("rms_norm_pack8_rows(Tensor x, Tensor? weight, float eps) -> (Tensor codes, Tensor scales)")
_lib.define(
    "add_rms_norm_pack8_rows(Tensor x, Tensor residual, Tensor? weight, float eps) -> (Tensor codes, Tensor scales, Tensor sum)"
)
_lib.define(
    "linear8(Tensor codes, Tensor scales, Tensor weight_codes, Tensor weight_scales, Tensor? bias, Tensor? residual, ScalarType dtype) -> Tensor"
)


@torch.library.register_fake("flash_mhc::pack8_rows")
def _pack8_rows_fake(x):
    return _k.empty_rows(x)


@torch.library.register_fake("flash_mhc::rms_norm_pack8_rows")
def _rms_norm_pack8_rows_fake(x, weight, eps):
    return _k.empty_rows(x)


@torch.library.register_fake("flash_mhc::add_rms_norm_pack8_rows")
def _add_rms_norm_pack8_rows_fake(x, residual, weight, eps):
    return (*_k.empty_rows(x), x.new_empty(x.shape))


@torch.library.register_fake("flash_mhc::linear8")
def _linear8_fake(codes, scales, weight_codes, weight_scales, bias, residual, dtype):
    return codes.new_empty((*codes.shape[:-1], weight_codes.shape[0]), dtype=dtype)


def _dense(t):
    return None if t is None else t.contiguous()


@torch.library.impl(_lib, "pack8_rows", "CUDA")
@without_tangents
def _pack8_rows_cuda(x):
    return _k.pack8_rows(x.contiguous())


@torch.library.impl(_lib, "rms_norm_pack8_rows", "CUDA")
@without_tangents
def _rms_norm_pack8_rows_cuda(x, weight, eps):
    return _k.rms_norm_pack8_rows(x.contiguous(), None, _dense(weight), eps)[:2]


@torch.library.impl(_lib, "add_rms_norm_pack8_rows", "CUDA")
@without_tangents
def _add_rms_norm_pack8_rows_cuda(x, residual, weight, eps):
    return _k.rms_norm_pack8_rows(x.contiguous(), residual.contiguous(), _dense(weight), eps)


@torch.library.impl(_lib, "linear8", "CUDA")
@without_tangents
def _linear8_cuda(codes, scales, weight_codes, weight_scales, bias, residual, dtype):
    return _k.linear8(codes, scales.contiguous(), weight_codes, weight_scales.contiguous(), _dense(bias),
                      _dense(residual), dtype)


def _no_gradient(name):
    def backward(ctx, *grads):
        raise RuntimeError(f"flash_mhc::{name} has no gradient: it serves inference (torch.no_grad())")

    return backward


for _op in ("pack8_rows", "rms_norm_pack8_rows", "add_rms_norm_pack8_rows", "linear8"):
    torch.library.register_autograd(f"flash_mhc::{_op}", _no_gradient(_op))


def _direct(x, *tensors) -> bool:
    """The kernels' launchers can be called without the ops: an ordinary tensor in eager mode, and
    no graph is recorded (the ops' backward raises)."""
    if not _block._plain_eager(x):
        return False
    graph = torch.is_grad_enabled()
    if graph and x.requires_grad:
        return False
    for t in tensors:
        if t is not None and ((type(t) is not torch.Tensor and type(t) is not nn.Parameter)
                              or (graph and t.requires_grad)):
            return False
    if _forward_ad._current_level >= 0:
        refuse_tangents(x, *tensors)
    return True


def _check_rows(x, what) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} expects x of shape (..., C) with C >= 1, got {tuple(x.shape)}")


def pack8_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes (..., C) int8, scales (...,) fp32) of the rows of x (..., C), bf16, fp16 or
    fp32, on the GPU: x is about codes * scales[..., None], off by at most half a scale.
    A row that holds an Inf or NaN has scale NaN.  No gradient."""
    if _direct(x):
        return _k.pack8_rows(x.contiguous())
    _check_rows(x, "pack8_rows")
    return torch.ops.flash_mhc.pack8_rows(x)


def rms_norm_pack8_rows(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6,
                        residual: torch.Tensor | None = None):
    """(codes, scales) of rms_norm(x, weight, eps), taken from its fp32 values; with a
    residual (codes, scales, sum) of rms_norm(x, weight, eps, residual).  No gradient.

    (A row has scale NaN where its product with weight overflows fp32, and counts as zero where
    all of it is below 2^-126.)"""
    if _direct(x, weight, residual):
        out = _k.rms_norm_pack8_rows(x.contiguous(), _dense(residual), _dense(weight), eps)
        return out[:2] if residual is None else out
    from .norm import check_rms

    check_rms(x, weight, residual)
    if residual is None:
        return torch.ops.flash_mhc.rms_norm_pack8_rows(x, weight, eps)
    return torch.ops.flash_mhc.add_rms_norm_pack8_rows(x, residual, weight, eps)


def linear8(codes: torch.Tensor, scales: torch.Tensor, weight_codes: torch.Tensor, weight_scales: torch.Tensor,
            bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
            dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of rows in 8 bits, on the GPU: (..., N) in dtype, rounded once, of

        (codes @ weight_codes^T) * scales[..., None] * weight_scales + bias + residual

    codes (..., K) and weight_codes (N, K) int8 with K < 2^17 and N < 2^22, scales (...,) and
    weight_scales (N,) fp32 (pack8_rows of a token's row and of a weight's), bias (N,)
    fp32 or of dtype, residual (..., N) of dtype.  The sum of integers is exact, and the
    product overflows only where it is itself past fp32's range.  No gradient."""
    if _direct(codes, scales, weight_codes, weight_scales, bias, residual):
        return _k.linear8(codes, scales.contiguous(), weight_codes, weight_scales.contiguous(), _dense(bias),
                          _dense(residual), dtype)
    return torch.ops.flash_mhc.linear8(codes, scales, weight_codes, weight_scales, bias, residual, dtype)


def _plain_rows(x):
    """pack8_rows in PyTorch operations: the same codes and scales."""
    v = x.float()
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    top = top.clamp(min=2.0 ** -100)
    # (Divisions of tensors: those by or of a Python number may be products with a rounded reciprocal, which
    # moves half a row's largest magnitude, 63.5, off its tie.)
    most = torch.full_like(top, 127.0)
    codes = (v * (most / top).unsqueeze(-1)).round()
    codes = torch.where(bad.unsqueeze(-1), torch.zeros_like(codes), codes)
    return codes.to(torch.int8), torch.where(bad, torch.full_like(top, float("nan")), top / most)


_LARGE = 2.0 ** 96  # times a sum of products, at most 2^31, within fp32's range


class _PlainLinear8(torch.autograd.Function):
    """Linear8's plain formula where a graph is recorded: its backward raises."""

    @staticmethod
    def forward(layer, x, weight_scales, bias):
        return layer._plain(x)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    backward = staticmethod(_no_gradient("linear8"))


class Linear8(nn.Module):
    """A linear layer with an 8-bit weight, for inference: x (..., in_features) to
    (..., out_features) in x's dtype (bf16, fp16 or fp32), with x packed by rows in the
    call.  Tensors that are not on a GPU go through the same formulas in PyTorch
    operations; neither form has a gradient.  The scales stay fp32 where the module is
    cast.

    Args:
        in_features, out_features: K and N.
        bias: give the layer a bias.

    The layer is zero until it is filled (``from_linear``, ``load_state_dict``).
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        if not 1 <= in_features <= _k.MOST_K or not 1 <= out_features <= _k.MOST_N:
            raise ValueError(f"Linear8 takes in_features from 1 to {_k.MOST_K} and out_features from 1 to {_k.MOST_N}, "
                             f"got {in_features} and {out_features}")
        self.in_features = in_features
        self.out_features = out_features
        # Rows at the kernels' pitch; the columns past in_features are zero.
        self.register_buffer("weight_codes", torch.zeros(out_features, _k.row_pitch(in_features), dtype=torch.int8,
                                                         device=device))
        self.register_buffer("weight_scales", torch.zeros(out_features, dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Linear8":
        """The 8-bit layer of an nn.Linear's weight and bias, on its device."""
        w = linear.weight.detach()
        out = cls(w.shape[1], w.shape[0], linear.bias is not None, device=w.device, dtype=w.dtype)
        with torch.no_grad():
            codes, scales = pack8_rows(w) if w.is_cuda and w.dtype in _k.DTYPES else _plain_rows(w)
            out.weight_codes[:, :out.in_features].copy_(codes)
            out.weight_scales.copy_(scales)
            if linear.bias is not None:
                out.bias.copy_(linear.bias)
        return out.train(linear.training)

    def _apply(self, fn, *args, **kwargs):
        kept = self.weight_scales
        super()._apply(fn, *args, **kwargs)
        if self.weight_scales.dtype is not torch.float32:  # cast with the module
            self.weight_scales = (torch.empty_like(self.weight_scales, dtype=torch.float32) if kept.is_meta
                                  else kept.to(self.weight_scales.device))
        return self

    def _weight(self) -> torch.Tensor:
        K = self.in_features
        return self.weight_codes if self.weight_codes.shape[1] == K else self.weight_codes[:, :K]

    def _bias(self, dtype: torch.dtype):
        # (Of another type, in fp32: 16 bits of one type may not hold what 16 of another do.)
        b = self.bias
        return b if b is None or b.dtype is dtype else b.float()

    def on_kernels(self, x: torch.Tensor) -> bool:
        return x.is_cuda and x.dtype in _k.DTYPES

    def product(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype,
                residual: torch.Tensor | None = None) -> torch.Tensor:
        """The layer of rows that are packed already, plus a residual, in dtype."""
        return linear8(codes, scales, self._weight(), self.weight_scales, self._bias(dtype), residual=residual,
                       dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"expected x of shape (..., {self.in_features}), got {tuple(x.shape)}")
        if not x.is_floating_point():
            raise TypeError(f"expected x of a floating-point type, got {x.dtype}")
        if self.on_kernels(x):
            return self.product(*pack8_rows(x), x.dtype)
        kept = x, self.weight_scales, self.bias
        refuse_tangents(*kept)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in kept):
            return _PlainLinear8.apply(self, *kept)
        return self._plain(x)

    def _plain(self, x: torch.Tensor) -> torch.Tensor:
        codes, scales = _plain_rows(x)
        # In 64 bits the products of codes and their sums are exact.
        out = F.linear(codes.double(), self._weight().double()).float()
        # (As the kernels: a token's large scale multiplies last, lest the product on the way pass fp32's range.)
        scales = scales.unsqueeze(-1)
        last = scales.abs() > _LARGE
        out = out * torch.where(last, self.weight_scales, scales) * torch.where(last, scales, self.weight_scales)
        return (out if self.bias is None else out + self.bias.float()).to(x.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
