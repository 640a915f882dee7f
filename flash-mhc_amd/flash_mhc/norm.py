"""Layer norm over the last axis on the HIP kernels, forward and backward.

Every layer that an mHC block wraps starts with a norm of its (T, C) input;
``MHCLiteBlock(pre_norm=True)`` uses this one.  The backward reads the input
either as it is or, with ``activation_bits=8``, from 8-bit codes that the
forward writes in its own pass (``flash_mhc.activation8``).

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
        cls = type(self)
        return (_any_global_hook is None or _any_global_hook() or cls.forward is not LayerNorm.forward
                or cls.__call__ is not nn.Module.__call__ or cls._call_impl is not nn.Module._call_impl
                or "forward" in self.__dict__ or "_call_impl" in self.__dict__
                or getattr(self, "_compiled_call_impl", None) is not None
                or bool(self._forward_hooks or self._forward_pre_hooks or self._backward_hooks
                        or self._backward_pre_hooks))

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
