"""Layer norm and RMS norm over the last axis on the HIP kernels, forward and backward.

Every layer that an mHC block wraps starts with a norm of its (T, C) input;
``MHCLiteBlock(pre_norm=True)`` uses the layer norm, ``pre_norm="rms"`` the RMS norm.
The layer norm's backward reads the input either as it is or, with
``activation_bits=8``, from 8-bit codes that the forward writes in its own pass
(``flash_mhc.activation8``).  The RMS norm takes a residual: inside a layer of several
parts each norm but the first is that of the part's output added to what went in.

No counterpart in the reference, which leaves the layer's norm to the layer.
"""

from __future__ import annotations

import torch
import torch.library
import torch.nn as nn
import torch.nn.functional as F

from . import kernels as _k
from .activation8 import _packed_like
from .block import _plain_eager
from .ops import _forward_ad, backward_op, differentiable_once, refuse_tangents, without_tangents

_lib = torch.library.Library("flash_mhc", "FRAGMENT")

# Whether hooks for all modules are registered (a private name: without it, modules
# count as hooked).
_any_global_hook = getattr(torch.nn.modules.module, "_has_any_global_hook", None)

_lib.define("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor y, Tensor mean, Tensor rstd)")
_lib.define(
    "layer_norm_pack8(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor y, Tensor mean, Tensor rstd, Tensor x_codes, Tensor x_scales)"
)
# From x, or (x None) from its codes and scales.  The parameters' gradients are
# in the dtype of `weight` (fp32 without one) and empty where not asked for.
_lib.define(
    "layer_norm_backward(Tensor grad_y, Tensor? x, Tensor? x_codes, Tensor? x_scales, Tensor mean, Tensor rstd, Tensor? weight, ScalarType param_dtype, bool need_weight, bool need_bias) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias)"
)


@torch.library.register_fake("flash_mhc::layer_norm")
def _layer_norm_fake(x, weight, bias, eps):
    stat = x.new_empty(x.shape[:-1], dtype=torch.float32)
    return x.new_empty(x.shape), stat, torch.empty_like(stat)


@torch.library.register_fake("flash_mhc::layer_norm_pack8")
def _layer_norm_pack8_fake(x, weight, bias, eps):
    return (*_layer_norm_fake(x, weight, bias, eps), *_packed_like(x))


@torch.library.register_fake("flash_mhc::layer_norm_backward")
def _layer_norm_backward_fake(grad_y, x, x_codes, x_scales, mean, rstd, weight, param_dtype, need_weight, need_bias):
    C = grad_y.shape[-1]
    return (grad_y.new_empty(grad_y.shape), grad_y.new_empty((C if need_weight else 0,), dtype=param_dtype),
            grad_y.new_empty((C if need_bias else 0,), dtype=param_dtype))


_ORDINARY = (type(None), nn.Parameter, torch.Tensor)  # no subclass: the kernels can read its memory


def _dense(t):
    return None if t is None else t.contiguous()


@torch.library.impl(_lib, "layer_norm", "CUDA")
@without_tangents
def _layer_norm_cuda(x, weight, bias, eps):
    return _k.layer_norm_fwd(x.contiguous(), _dense(weight), _dense(bias), eps)[:3]


@torch.library.impl(_lib, "layer_norm_pack8", "CUDA")
@without_tangents
def _layer_norm_pack8_cuda(x, weight, bias, eps):
    return _k.layer_norm_fwd(x.contiguous(), _dense(weight), _dense(bias), eps, packed=True)


@torch.library.impl(_lib, "layer_norm_backward", "CUDA")
@backward_op
def _layer_norm_backward_cuda(grad_y, x, x_codes, x_scales, mean, rstd, weight, param_dtype, need_weight, need_bias):
    gx, gw, gb = _k.layer_norm_bwd(grad_y.contiguous(), _dense(x), _dense(x_codes), _dense(x_scales),
                                   mean.contiguous(), rstd.contiguous(), _dense(weight), param_dtype, need_weight,
                                   need_bias)
    none = lambda: grad_y.new_empty((0,), dtype=param_dtype)
    return gx, none() if gw is None else gw, none() if gb is None else gb


def _param_dtype(weight, bias):
    return weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32


def _setup(ctx, inputs, output):
    x, weight, bias, _eps = inputs
    _y, mean, rstd, *packed = output
    ctx.packed = bool(packed)
    ctx.has = weight is not None, bias is not None
    ctx.param_dtype = _param_dtype(weight, bias)
    kept = packed if packed else [x]
    ctx.save_for_backward(mean, rstd, *kept, *([] if weight is None else [weight]))
    ctx.set_materialize_grads(False)


@differentiable_once
def _backward(ctx, grad_y, *_rest):
    # mean and rstd are not differentiable.
    if grad_y is None:
        return None, None, None, None
    mean, rstd, *kept = ctx.saved_tensors
    has_weight, has_bias = ctx.has
    weight = kept.pop() if has_weight else None
    x, codes, scales = (None, *kept) if ctx.packed else (*kept, None, None)
    need = has_weight and ctx.needs_input_grad[1], has_bias and ctx.needs_input_grad[2]
    gx, gw, gb = torch.ops.flash_mhc.layer_norm_backward(grad_y, x, codes, scales, mean, rstd, weight, ctx.param_dtype,
                                                         *need)
    return gx, gw if need[0] else None, gb if need[1] else None, None


torch.library.register_autograd("flash_mhc::layer_norm", _backward, setup_context=_setup)
torch.library.register_autograd("flash_mhc::layer_norm_pack8", _backward, setup_context=_setup)


# The two eager Functions' backward.


@differentiable_once
def _eager_gradients(ctx, grad_y, grad_x):
    x, codes, scales, stats, weight = ctx.saved_tensors
    _nx, need_weight, need_bias, _ne, _np = ctx.needs_input_grad
    gx, gw, gb = _k.layer_norm_bwd_joint(grad_y.contiguous(), x, codes, scales, stats, weight, ctx.param_dtype,
                                         need_weight, need_bias, _dense(grad_x))
    return gx, gw, gb, None, None


def _eager_backward(ctx, grad_y, grad_x=None):
    if grad_y is None:  # the norm's output was not used: x's gradient is the residual's
        return grad_x, None, None, None, None
    return _eager_gradients(ctx, grad_y, grad_x)


def _eager_forward(ctx, x, weight, bias, eps, packed):
    """(y,), or (y, stats) where ctx keeps something else than x or weight itself."""
    ctx.set_materialize_grads(False)
    xc, wc = x.contiguous(), _dense(weight)
    y, stats, codes, scales, ctx.param_dtype = _k.layer_norm_fwd_joint(xc, wc, _dense(bias), eps, packed)
    ctx.save_for_backward(None if packed else xc, codes, scales, stats, wc)
    return (y, stats) if packed or xc is not x or wc is not weight else (y,)


class _LayerNormEager(torch.autograd.Function):
    """layer_norm / layer_norm_pack8 with their registered autograd, without the
    ops' dispatch: y, and what _eager_forward adds."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, packed):
        return _eager_forward(ctx, x, weight, bias, eps, packed)

    @staticmethod
    def backward(ctx, grad_y, _stats=None):
        return _eager_backward(ctx, grad_y)


class _LayerNormResidualEager(torch.autograd.Function):
    """(x, layer_norm(x)): the gradient of the first, which the residual around a
    block's layer gives, is added in the norm's backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, packed):
        return (x.view_as(x), *_eager_forward(ctx, x, weight, bias, eps, packed))

    @staticmethod
    def backward(ctx, grad_x, grad_y, _stats=None):
        return _eager_backward(ctx, grad_y, grad_x)


def _check(x, weight, bias, activation_bits) -> None:
    if activation_bits not in (8, 16):
        raise ValueError(f"activation_bits must be 16 (keep the input as it is) or 8, got {activation_bits}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm expects x of shape (..., C) with C >= 1, got {tuple(x.shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(t.shape)}")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, activation_bits: int = 16) -> torch.Tensor:
    """Layer norm of x (..., C) over its last axis, on the GPU.

    x is bf16, fp16 or fp32; weight and bias (C,), either may be None, are fp32
    or of x's dtype.  Statistics and sums are fp32, y and every gradient are
    rounded once.  activation_bits: 16 keeps x for the backward, 8 its 8-bit
    codes (the backward's normalised input is then that of the codes, with the
    statistics of x).  Differentiable once, in reverse mode: a gradient of its
    gradients raises, and so does a dual tensor."""
    packed = activation_bits == 8
    if (packed or activation_bits == 16) and _plain_eager(x) and type(weight) in _ORDINARY and type(bias) in _ORDINARY:
        # (The kernels' launchers check the tensors.)
        if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                        or (bias is not None and bias.requires_grad)):
            return _LayerNormEager.apply(x, weight, bias, eps, packed)[0]
        if _forward_ad._current_level >= 0:
            refuse_tangents(x, weight, bias)
        return _k.layer_norm_fwd(x.contiguous(), _dense(weight), _dense(bias), eps, stats=False)[0]
    _check(x, weight, bias, activation_bits)
    refuse_tangents(x, weight, bias)
    op = torch.ops.flash_mhc.layer_norm_pack8 if packed else torch.ops.flash_mhc.layer_norm
    return op(x, weight, bias, eps)[0]


def hooked(module: nn.Module, base: type) -> bool:
    """A call of module does more than base.forward."""
    cls = type(module)
    return (_any_global_hook is None or _any_global_hook() or cls.forward is not base.forward
            or cls.__call__ is not nn.Module.__call__ or cls._call_impl is not nn.Module._call_impl
            or "forward" in module.__dict__ or "_call_impl" in module.__dict__
            or getattr(module, "_compiled_call_impl", None) is not None
            or bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                    or module._backward_pre_hooks))


class LayerNorm(nn.Module):
    """``nn.LayerNorm`` over the last axis on the HIP kernels, with the same
    parameters (``weight`` ones, ``bias`` zeros) and state_dict.  Tensors that
    the kernels do not take (not on a GPU, or other dtypes) go through PyTorch's
    layer norm, as MHCLiteBlock's do through its plain formulation.  Autocast
    does not change the kernels' types: the output has x's.

    Args:
        hidden_size: C.
        eps: added to the variance.
        elementwise_affine: give the norm a weight (and a bias).
        bias: with elementwise_affine, give it a bias too.
        activation_bits: 16 keeps the input for the backward, 8 its 8-bit codes.
    """

    def __init__(self, hidden_size: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 activation_bits: int = 16, device=None, dtype=None) -> None:
        super().__init__()
        if activation_bits not in (8, 16):
            raise ValueError(f"activation_bits must be 16 or 8, got {activation_bits}")
        self.hidden_size = hidden_size
        self.eps = eps
        self.activation_bits = activation_bits
        kw = {"device": device, "dtype": dtype}
        self.weight = nn.Parameter(torch.ones(hidden_size, **kw)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(hidden_size, **kw)) if elementwise_affine and bias else None

    def _on_kernels(self, x: torch.Tensor) -> bool:
        pdt = _param_dtype(self.weight, self.bias)
        return x.is_cuda and x.dtype in _k.DTYPES and (pdt is torch.float32 or pdt is x.dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self._on_kernels(x):
            if self.weight is None and x.shape[-1:] != (self.hidden_size,):  # (weight's shape is checked)
                raise ValueError(f"expected x of shape (..., {self.hidden_size}), got {tuple(x.shape)}")
            return layer_norm(x, self.weight, self.bias, self.eps, self.activation_bits)
        return F.layer_norm(x, (self.hidden_size,), self.weight, self.bias, self.eps)

    def _hooked(self) -> bool:
        """A call of this module does more than LayerNorm.forward."""
        return hooked(self, LayerNorm)

    def with_residual(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(norm(x), x) for ``x + layer(norm(x))``: the norm's backward adds the
        gradient that x gets from the residual (as a separate addition would)."""
        if (_plain_eager(x) and torch.is_grad_enabled() and x.requires_grad and not self._hooked()
                and self._on_kernels(x) and type(self.weight) in _ORDINARY and type(self.bias) in _ORDINARY
                and x.shape[-1:] == (self.hidden_size,)):
            r, y, *_ = _LayerNormResidualEager.apply(x, self.weight, self.bias, self.eps, self.activation_bits == 8)
            return y, r
        return self(x), x

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}, activation_bits={self.activation_bits}"


# ---------------------------------------------------------------------------
# RMS norm

_lib.define("rms_norm(Tensor x, Tensor? weight, float eps) -> (Tensor y, Tensor rstd)")
_lib.define(
    "add_rms_norm(Tensor x, Tensor residual, Tensor? weight, float eps) -> (Tensor y, Tensor sum, Tensor rstd)"
)
# x is the norm's input, or its sum with the residual.  The weight's gradient is empty
# where it is not asked for.
_lib.define(
    "rms_norm_backward(Tensor grad_y, Tensor? grad_x_in, Tensor x, Tensor rstd, Tensor? weight, bool need_weight) -> (Tensor grad_x, Tensor grad_weight)"
)


@torch.library.register_fake("flash_mhc::rms_norm")
def _rms_norm_fake(x, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.register_fake("flash_mhc::add_rms_norm")
def _add_rms_norm_fake(x, residual, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32)


def _no_weight_grad(grad_y, weight):
    return grad_y.new_empty((0,), dtype=_param_dtype(weight, None))


@torch.library.register_fake("flash_mhc::rms_norm_backward")
def _rms_norm_backward_fake(grad_y, grad_x_in, x, rstd, weight, need_weight):
    gw = weight.new_empty(weight.shape) if need_weight else _no_weight_grad(grad_y, weight)
    return grad_y.new_empty(grad_y.shape), gw


@torch.library.impl(_lib, "rms_norm", "CUDA")
@without_tangents
def _rms_norm_cuda(x, weight, eps):
    y, _sum, rstd = _k.rms_norm_fwd(x.contiguous(), None, _dense(weight), eps)
    return y, rstd


@torch.library.impl(_lib, "add_rms_norm", "CUDA")
@without_tangents
def _add_rms_norm_cuda(x, residual, weight, eps):
    return _k.rms_norm_fwd(x.contiguous(), residual.contiguous(), _dense(weight), eps)


@torch.library.impl(_lib, "rms_norm_backward", "CUDA")
@backward_op
def _rms_norm_backward_cuda(grad_y, grad_x_in, x, rstd, weight, need_weight):
    if need_weight and weight is None:
        raise ValueError("rms_norm_backward: there is no weight to give a gradient")
    gx, gw = _k.rms_norm_bwd(grad_y.contiguous(), x.contiguous(), rstd.contiguous(), _dense(weight),
                             _param_dtype(weight, None), need_weight, _dense(grad_x_in))
    return gx, _no_weight_grad(grad_y, weight) if gw is None else gw


def _rms_setup(ctx, inputs, output):
    # (x, weight, eps) -> (y, rstd), or (x, residual, weight, eps) -> (y, sum, rstd)
    ctx.added = len(inputs) == 4
    x, weight = output[1] if ctx.added else inputs[0], inputs[-2]
    ctx.save_for_backward(x, output[-1], *([] if weight is None else [weight]))
    ctx.set_materialize_grads(False)


@differentiable_once
def _rms_gradients(ctx, grad_y, grad_sum):
    x, rstd, *weight = ctx.saved_tensors
    weight = weight[0] if weight else None
    need = weight is not None and ctx.needs_input_grad[2 if ctx.added else 1]
    gx, gw = torch.ops.flash_mhc.rms_norm_backward(grad_y, grad_sum, x, rstd, weight, need)
    return gx, gw if need else None


def _rms_backward(ctx, grad_y, *rest):
    # rstd is not differentiable.
    grad_sum = rest[0] if ctx.added else None
    # (Where the norm's output was not used, x's gradient is the sum's.)
    gx, gw = (grad_sum, None) if grad_y is None else _rms_gradients(ctx, grad_y, grad_sum)
    return (gx, gx, gw, None) if ctx.added else (gx, gw, None)


torch.library.register_autograd("flash_mhc::rms_norm", _rms_backward, setup_context=_rms_setup)
torch.library.register_autograd("flash_mhc::add_rms_norm", _rms_backward, setup_context=_rms_setup)


@differentiable_once
def _rms_eager_gradients(ctx, grad_y, grad_x):
    x, rstd, weight = ctx.saved_tensors  # (hooks for saved tensors may have given them other strides)
    return _k.rms_norm_bwd(grad_y.contiguous(), x.contiguous(), rstd.contiguous(), _dense(weight),
                           _param_dtype(weight, None),
                           weight is not None and ctx.needs_input_grad[ctx.weight_at], _dense(grad_x))


def _rms_eager_backward(ctx, grad_y, grad_x):
    if grad_y is None:
        return grad_x, None
    return _rms_eager_gradients(ctx, grad_y, grad_x)


def _rms_eager_forward(ctx, x, residual, weight, eps):
    """(y, sum, rstd); rstd is an output too where the graph would not lead to x and weight through
    what ctx keeps."""
    ctx.set_materialize_grads(False)
    xc, wc = x.contiguous(), _dense(weight)
    y, total, rstd = _k.rms_norm_fwd(xc, _dense(residual), wc, eps)
    ctx.save_for_backward(xc if total is None else total, rstd, wc)
    return y, total, rstd if total is None and (xc is not x or wc is not weight) else None


class _RMSNormEager(torch.autograd.Function):
    """rms_norm with its registered autograd, without the ops' dispatch."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.weight_at = 1
        y, _total, rstd = _rms_eager_forward(ctx, x, None, weight, eps)
        return (y,) if rstd is None else (y, rstd)

    @staticmethod
    def backward(ctx, grad_y, _rstd=None):
        return (*_rms_eager_backward(ctx, grad_y, None), None)


class _AddRMSNormEager(torch.autograd.Function):
    """add_rms_norm, likewise: (y, sum)."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.weight_at = 2
        return _rms_eager_forward(ctx, x, residual, weight, eps)[:2]

    @staticmethod
    def backward(ctx, grad_y, grad_sum):
        gx, gw = _rms_eager_backward(ctx, grad_y, grad_sum)
        return gx, gx, gw, None


class _RMSNormResidualEager(torch.autograd.Function):
    """(x, rms_norm(x)): as _LayerNormResidualEager."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.weight_at = 1
        y, _total, rstd = _rms_eager_forward(ctx, x, None, weight, eps)
        return (x.view_as(x), y) if rstd is None else (x.view_as(x), y, rstd)

    @staticmethod
    def backward(ctx, grad_x, grad_y, _rstd=None):
        return (*_rms_eager_backward(ctx, grad_y, grad_x), None)


def check_rms(x, weight, residual) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"rms_norm expects x of shape (..., C) with C >= 1, got {tuple(x.shape)}")
    if weight is not None and tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"weight must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} and dtype {x.dtype}, got "
                         f"{tuple(residual.shape)} and {residual.dtype}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6,
             residual: torch.Tensor | None = None):
    """RMS norm of x (..., C) over its last axis, on the GPU: x rsqrt(mean(x^2) + eps) weight.

    With a residual (of x's shape and dtype) it is that of sum = x + residual, and
    (y, sum) is returned: the sum is rounded to x's dtype, and the norm is that of the
    rounded sum.

    x is bf16, fp16 or fp32; weight (C,), or None, is fp32 or of x's dtype.  The
    statistic and sums are fp32, y and every gradient are rounded once.  Differentiable
    once, in reverse mode: a gradient of its gradients raises, and so does a dual tensor."""
    if _plain_eager(x) and type(weight) in _ORDINARY and type(residual) in _ORDINARY:
        # (The kernels' launchers check the tensors.)
        if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                        or (residual is not None and residual.requires_grad)):
            if residual is None:
                return _RMSNormEager.apply(x, weight, eps)[0]
            return _AddRMSNormEager.apply(x, residual, weight, eps)
        if _forward_ad._current_level >= 0:
            refuse_tangents(x, weight, residual)
        y, total, _rstd = _k.rms_norm_fwd(x.contiguous(), _dense(residual), _dense(weight), eps, stats=False)
        return y if residual is None else (y, total)
    check_rms(x, weight, residual)
    refuse_tangents(x, weight, residual)
    if residual is None:
        return torch.ops.flash_mhc.rms_norm(x, weight, eps)[0]
    return torch.ops.flash_mhc.add_rms_norm(x, residual, weight, eps)[:2]


class RMSNorm(nn.Module):
    """``nn.RMSNorm`` over the last axis on the HIP kernels, with the same parameter
    (``weight``, ones) and state_dict.  Tensors that the kernels do not take (not on a
    GPU, or other dtypes) go through PyTorch's RMS norm, as LayerNorm's do through its
    layer norm; autocast does not change the kernels' types.

    Args:
        hidden_size: C.
        eps: added to the mean of squares.
        elementwise_affine: give the norm a weight.
    """

    def __init__(self, hidden_size: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None,
                 dtype=None) -> None:
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype)) if elementwise_affine else None

    def _on_kernels(self, x: torch.Tensor) -> bool:
        pdt = _param_dtype(self.weight, None)
        return x.is_cuda and x.dtype in _k.DTYPES and (pdt is torch.float32 or pdt is x.dtype)

    def _check_width(self, x: torch.Tensor) -> None:
        if self.weight is None and x.shape[-1:] != (self.hidden_size,):  # (weight's shape is checked)
            raise ValueError(f"expected x of shape (..., {self.hidden_size}), got {tuple(x.shape)}")

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """norm(x); with a residual (norm(x + residual), x + residual)."""
        if self._on_kernels(x):
            self._check_width(x)
            return rms_norm(x, self.weight, self.eps, residual)
        if residual is None:
            return F.rms_norm(x, (self.hidden_size,), self.weight, self.eps)
        check_rms(x, None, residual)
        total = x + residual
        return F.rms_norm(total, (self.hidden_size,), self.weight, self.eps), total

    def packed(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """rms_norm_pack8_rows of x on the GPU: (codes, scales), with a residual and the sum."""
        from .rows8 import rms_norm_pack8_rows

        self._check_width(x)
        return rms_norm_pack8_rows(x, self.weight, self.eps, residual)

    def _hooked(self) -> bool:
        """A call of this module does more than RMSNorm.forward."""
        return hooked(self, RMSNorm)

    def with_residual(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(norm(x), x) for ``x + layer(norm(x))``: the norm's backward adds the gradient
        that x gets from the residual (and rounds the sum once)."""
        if (_plain_eager(x) and torch.is_grad_enabled() and x.requires_grad and not self._hooked()
                and self._on_kernels(x) and type(self.weight) in _ORDINARY and x.shape[-1:] == (self.hidden_size,)):
            r, y, *_ = _RMSNormResidualEager.apply(x, self.weight, self.eps)
            return y, r
        return self(x), x

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}"
