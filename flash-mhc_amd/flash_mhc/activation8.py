"""Activations kept in 8 bits between the forward and the backward.

What a block of streams keeps for its backward is nearly all x (T, 4, C) and
the layer output (T, C).  Here they are kept as block-scaled 8-bit codes, 33/64
of their bf16 bytes: groups of 32 columns share a power of two, an element is a
signed code times it (the format is defined in ``include/flash_mhc_hip.h``), off
by at most a 128th of the group's power of two (a 64th at its top).  The forward
is computed from the exact tensors; the backward reads the codes and gives the
bits that the bf16 backward gives on the unpacked tensors (K1's backward by
itself up to the order of fp32 sums where C % 8 != 0).

  pack8, unpack8                    a tensor (..., C) to codes and scales and back
  fused_post_res_pack8              fused_post_res that keeps its inputs packed
  fused_rmsnorm_project_bwd_pack8   K1's backward from packed streams
  mhc_pre_map_pack8, mhc_post_res_pack8
                                    the block's two ops (MHCLiteBlock with
                                    ``activation_bits=8``): mhc_pre_map packs x,
                                    and mhc_post_res reads the same codes
  pre_map_eager, post_res_eager     the block in eager mode: post-res's forward,
                                    the block's last kernel, packs x and the
                                    layer output while it has them in registers

No counterpart in the reference, whose backward reads bf16 tensors.
"""

from __future__ import annotations

import weakref

import torch
import torch.library

from . import _abi
from . import block as _block  # which imports this module: its names are read at call time
from . import kernels as _k
from .ops import (
    _check_k2_shapes,
    _check_n4,
    _coeff,
    _mhc_pre_map_cuda,
    _mhc_pre_map_fake,
    _params,
    backward_op,
    differentiable_once,
    graph_link,
    without_tangents,
)

_lib = torch.library.Library("flash_mhc", "FRAGMENT")

_lib.define("pack8(Tensor x) -> (Tensor codes, Tensor scales)")
_lib.define("unpack8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor")
# fused_post_res_pack8 in eager mode is an autograd Function around the device
# implementation (_FusedPostResEager); where it is traced it becomes
# fused_post_res_pack8_traced, which has its fake and registered autograd.
_lib.define(
    "fused_post_res_pack8(Tensor x_streams, Tensor layer_output, Tensor H_merged, Tensor h_post) -> (Tensor out, Tensor x_codes, Tensor x_scales, Tensor lo_codes, Tensor lo_scales)"
)
_lib.define(
    "fused_post_res_pack8_traced(Tensor x_streams, Tensor layer_output, Tensor H_merged, Tensor h_post) -> (Tensor out, Tensor x_codes, Tensor x_scales, Tensor lo_codes, Tensor lo_scales)"
)
_lib.define(
    "fused_post_res_backward_pack8(Tensor grad_out, Tensor x_codes, Tensor x_scales, Tensor lo_codes, Tensor lo_scales, Tensor H_merged, Tensor h_post) -> (Tensor grad_x, Tensor grad_layer_output, Tensor grad_H_merged, Tensor grad_h_post)"
)
_lib.define(
    "fused_rmsnorm_project_bwd_pack8(Tensor grad_out, Tensor x_codes, Tensor x_scales, Tensor W, Tensor proj_out, Tensor inv_rms) -> (Tensor grad_x, Tensor grad_W)"
)
# mhc_pre_map that also packs x, and keeps the codes instead of x.
_lib.define(
    "mhc_pre_map_pack8(Tensor x_streams, Tensor W, Tensor alpha_pre, Tensor alpha_post, Tensor alpha_res, Tensor bias, Tensor perm_mat) -> (Tensor layer_input, Tensor H_merged, Tensor h_post, Tensor h_pre, Tensor proj, Tensor inv_rms, Tensor x_sink, Tensor x_codes, Tensor x_scales)"
)
_lib.define(
    "mhc_pre_map_backward_pack8(Tensor? grad_layer_input, Tensor? grad_H_merged, Tensor? grad_h_post, Tensor? grad_h_pre, Tensor? grad_proj, Tensor? grad_x_sink, Tensor x_codes, Tensor x_scales, Tensor W, Tensor alpha_pre, Tensor alpha_post, Tensor alpha_res, Tensor bias, Tensor perm_mat, Tensor h_pre, Tensor proj, Tensor inv_rms) -> (Tensor grad_x, Tensor grad_W, Tensor grad_alpha_pre, Tensor grad_alpha_post, Tensor grad_alpha_res, Tensor grad_bias)"
)
# mhc_post_res for streams packed by mhc_pre_map_pack8: packs the layer output,
# and keeps both codes instead of the tensors.
_lib.define(
    "mhc_post_res_pack8(Tensor x_streams, Tensor x_sink, Tensor x_codes, Tensor x_scales, Tensor layer_output, Tensor H_merged, Tensor h_post) -> (Tensor out, Tensor lo_codes, Tensor lo_scales)"
)


# ---------------------------------------------------------------------------
# Fakes


def _packed_like(x):
    return (x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty((*x.shape[:-1], (x.shape[-1] + 31) // 32), dtype=torch.uint8))


@torch.library.register_fake("flash_mhc::pack8")
def _pack8_fake(x):
    return _packed_like(x)


@torch.library.register_fake("flash_mhc::unpack8")
def _unpack8_fake(codes, scales, dtype):
    return codes.new_empty(codes.shape, dtype=dtype)


@torch.library.register_fake("flash_mhc::fused_post_res_pack8_traced")
@torch.library.register_fake("flash_mhc::fused_post_res_pack8")
def _fused_post_res_pack8_fake(x_streams, layer_output, H_merged, h_post):
    return (torch.empty_like(x_streams, memory_format=torch.contiguous_format), *_packed_like(x_streams),
            *_packed_like(layer_output))


@torch.library.register_fake("flash_mhc::fused_post_res_backward_pack8")
def _fused_post_res_backward_pack8_fake(grad_out, x_codes, x_scales, lo_codes, lo_scales, H_merged, h_post):
    f32 = torch.float32
    return (grad_out.new_empty(x_codes.shape), grad_out.new_empty(lo_codes.shape),
            H_merged.new_empty(H_merged.shape, dtype=f32), h_post.new_empty(h_post.shape, dtype=f32))


@torch.library.register_fake("flash_mhc::fused_rmsnorm_project_bwd_pack8")
def _fused_rmsnorm_project_bwd_pack8_fake(grad_out, x_codes, x_scales, W, proj_out, inv_rms):
    return grad_out.new_empty(x_codes.shape), grad_out.new_empty(W.shape)


@torch.library.register_fake("flash_mhc::mhc_pre_map_pack8")
def _mhc_pre_map_pack8_fake(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat):
    return (*_mhc_pre_map_fake(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat),
            *_packed_like(x_streams))


@torch.library.register_fake("flash_mhc::mhc_pre_map_backward_pack8")
def _mhc_pre_map_backward_pack8_fake(grad_layer_input, grad_H_merged, grad_h_post, grad_h_pre, grad_proj, grad_x_sink,
                                     x_codes, x_scales, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat, h_pre,
                                     proj, inv_rms):
    return (proj.new_empty(x_codes.shape), torch.empty_like(W), torch.empty_like(alpha_pre),
            torch.empty_like(alpha_post), torch.empty_like(alpha_res), torch.empty_like(bias))


@torch.library.register_fake("flash_mhc::mhc_post_res_pack8")
def _mhc_post_res_pack8_fake(x_streams, x_sink, x_codes, x_scales, layer_output, H_merged, h_post):
    return (torch.empty_like(x_streams, memory_format=torch.contiguous_format), *_packed_like(layer_output))


# ---------------------------------------------------------------------------
# Device implementations


@torch.library.impl(_lib, "pack8", "CUDA")
def _pack8_cuda(x):
    return _k.pack8(x.contiguous())


@torch.library.impl(_lib, "unpack8", "CUDA")
def _unpack8_cuda(codes, scales, dtype):
    return _k.unpack8(codes.contiguous(), scales.contiguous(), dtype)


def _fused_post_res_pack8_cuda(x_streams, layer_output, H_merged, h_post):
    _check_n4(x_streams, "flash_mhc::fused_post_res_pack8 supports n=4 only")
    return _k.k4_fwd_pack8(x_streams.contiguous(), layer_output.contiguous(), _coeff(H_merged), _coeff(h_post))


for _op in ("fused_post_res_pack8_traced", "fused_post_res_pack8"):
    torch.library.impl(_lib, _op, "CUDA")(without_tangents(_fused_post_res_pack8_cuda))


@torch.library.impl(_lib, "fused_post_res_backward_pack8", "CUDA")
@backward_op
def _fused_post_res_backward_pack8_cuda(grad_out, x_codes, x_scales, lo_codes, lo_scales, H_merged, h_post):
    _check_n4(x_codes, "flash_mhc::fused_post_res_backward_pack8 supports n=4 only")
    return _k.k4_bwd_pack8(grad_out.contiguous(), x_codes.contiguous(), x_scales.contiguous(), lo_codes.contiguous(),
                           lo_scales.contiguous(), _coeff(H_merged), _coeff(h_post))


@torch.library.impl(_lib, "fused_rmsnorm_project_bwd_pack8", "CUDA")
@backward_op
def _fused_rmsnorm_project_bwd_pack8_cuda(grad_out, x_codes, x_scales, W, proj_out, inv_rms):
    _check_n4(x_codes, "flash_mhc::fused_rmsnorm_project_bwd_pack8 supports n=4 only")
    return _k.k1_bwd_pack8(grad_out.contiguous(), x_codes.contiguous(), x_scales.contiguous(),
                           W.to(grad_out.dtype).contiguous(), proj_out.contiguous(), inv_rms.contiguous())


@torch.library.impl(_lib, "mhc_pre_map_pack8", "CUDA")
@without_tangents
def _mhc_pre_map_pack8_cuda(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat):
    _check_n4(x_streams, "flash_mhc::mhc_pre_map_pack8 supports n=4 only")
    x = x_streams.contiguous()
    # A launch of its own: inside K1's kernels, which have two waves per SIMD or
    # one and all registers in use, the packing took as long as on its own (T =
    # 65536, C = 1024 135 -> 269 us, alone 132).
    packed = _k.pack8(x)
    return (*_mhc_pre_map_cuda(x, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat), *packed)


@torch.library.impl(_lib, "mhc_pre_map_backward_pack8", "CUDA")
@backward_op
def _mhc_pre_map_backward_pack8_cuda(grad_layer_input, grad_H_merged, grad_h_post, grad_h_pre, grad_proj, grad_x_sink,
                                     x_codes, x_scales, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat, h_pre,
                                     proj, inv_rms):
    _check_n4(x_codes, "flash_mhc::mhc_pre_map_backward_pack8 supports n=4 only")
    _check_k2_shapes((0, W.shape[0]), perm_mat)
    xq, xs = x_codes.contiguous(), x_scales.contiguous()
    T, n, C = xq.shape
    dt = proj.dtype
    Wc = W.to(dt).contiguous()
    coeffs = _params(alpha_pre, alpha_post, alpha_res, bias, perm_mat)
    g_li = (torch.zeros((T, C), device=xq.device, dtype=dt) if grad_layer_input is None
            else grad_layer_input.to(dt).contiguous())
    g_hp = None if grad_h_post is None else _coeff(grad_h_post)
    g_H = None if grad_H_merged is None else _coeff(grad_H_merged)
    g_sink = None if grad_x_sink is None else grad_x_sink.to(dt).contiguous()
    if grad_h_pre is None and grad_proj is None:
        gx, gW, ga1, ga2, ga3, gb = _k.premap_bwd_pack8(xq, xs, Wc, *coeffs, h_pre.contiguous(), proj.contiguous(),
                                                        inv_rms.contiguous(), g_li, g_hp, g_H, g_sink)
    else:
        # Gradients also flow into the h_pre / proj outputs (not in a block):
        # compose the launches, K3's on the unpacked streams.
        gx3, gh = _k.k3_bwd(g_li, _k.unpack8(xq, xs, dt), h_pre.contiguous())
        if grad_h_pre is not None:
            gh = gh + grad_h_pre.float()
        gp, ga1, ga2, ga3, gb = _k.k2_bwd(proj.contiguous(), *coeffs, gh, g_hp, g_H)
        if grad_proj is not None:
            gp = (gp.float() + grad_proj.float()).to(gp.dtype)
        gx1, gW = _k.k1_bwd_pack8(gp, xq, xs, Wc, proj.contiguous(), inv_rms.contiguous())
        gx = gx3 + gx1
        if g_sink is not None:
            gx = g_sink + gx
    return (gx, gW.to(W.dtype), ga1.to(alpha_pre.dtype), ga2.to(alpha_post.dtype), ga3.to(alpha_res.dtype),
            gb.to(bias.dtype))


@torch.library.impl(_lib, "mhc_post_res_pack8", "CUDA")
@without_tangents
def _mhc_post_res_pack8_cuda(x_streams, x_sink, x_codes, x_scales, layer_output, H_merged, h_post):
    _check_n4(x_streams, "flash_mhc::mhc_post_res_pack8 supports n=4 only")
    out, _xq, _xs, lo_codes, lo_scales = _k.k4_fwd_pack8(x_streams.contiguous(), layer_output.contiguous(),
                                                         _coeff(H_merged), _coeff(h_post), pack_x=False)
    return out, lo_codes, lo_scales


# ---------------------------------------------------------------------------
# Autograd.  Codes and scales are whole numbers and carry no gradient; the ops
# keep them and the coefficients, never x or the layer output.


def _setup_post_res(ctx, inputs, output):
    x, lo, H_merged, h_post = inputs
    ctx.save_for_backward(*output[1:], H_merged, h_post, graph_link(x, lo))
    ctx.set_materialize_grads(False)


@differentiable_once
def _fused_post_res_pack8_backward(ctx, grad_out, *_codes):
    if grad_out is None:
        return None, None, None, None
    return torch.ops.flash_mhc.fused_post_res_backward_pack8(grad_out, *ctx.saved_tensors[:-1])


torch.library.register_autograd("flash_mhc::fused_post_res_pack8_traced", _fused_post_res_pack8_backward,
                                setup_context=_setup_post_res)


class _FusedPostResEager(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x_streams, layer_output, H_merged, h_post):
        outs = _fused_post_res_pack8_cuda(x_streams, layer_output, H_merged, h_post)
        link = h_post.detach()  # h_post as a last output, for differentiable_once
        ctx.save_for_backward(*outs[1:], H_merged, link)
        ctx.mark_non_differentiable(*outs[1:])
        ctx.set_materialize_grads(False)
        return (*outs, link)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_out, *_codes):
        if grad_out is None:
            return None, None, None, None
        *codes, H_merged, h_post = ctx.saved_tensors
        return _k.k4_bwd_pack8_saved(grad_out.contiguous(), *codes, _coeff(H_merged), _coeff(h_post))


@torch.library.impl(_lib, "fused_post_res_pack8", "AutogradCUDA")
def _fused_post_res_pack8_autograd(x_streams, layer_output, H_merged, h_post):
    if _block._plain_eager(x_streams):
        return _FusedPostResEager.apply(x_streams, layer_output, H_merged, h_post)[:-1]
    return torch.ops.flash_mhc.fused_post_res_pack8_traced(x_streams, layer_output, H_merged, h_post)


def _version(x):
    """Counts x's changes in place (inference tensors are not changed where gradients are recorded)."""
    return None if x.is_inference() else x._version


def _check_version(x, version) -> None:
    # autograd's own check is of tensors that are kept, and x is not.
    if _version(x) != version:
        raise RuntimeError("the streams were modified by an inplace operation between the block's pre-map and "
                           "post-res, which both need them")


def _setup_pre_map(ctx, inputs, output):
    x, *params = inputs
    _li, _H, _hq, h_pre, proj, inv_rms, _sink, codes, scales = output
    codes._streams = id(x), _version(x)  # for mhc_post_res_pack8, also while a graph is traced
    ctx.save_for_backward(codes, scales, *params, h_pre, proj, inv_rms)
    ctx.set_materialize_grads(False)


@differentiable_once
def _mhc_pre_map_pack8_backward(ctx, g_li, g_H, g_hq, g_hpre, g_proj, _g_inv, g_sink, _gc, _gs):
    grads = torch.ops.flash_mhc.mhc_pre_map_backward_pack8(g_li, g_H, g_hq, g_hpre, g_proj, g_sink, *ctx.saved_tensors)
    return (*grads, None)


torch.library.register_autograd("flash_mhc::mhc_pre_map_pack8", _mhc_pre_map_pack8_backward,
                                setup_context=_setup_pre_map)


def _setup_mhc_post_res(ctx, inputs, output):
    x, x_sink, codes, scales, lo, H_merged, h_post = inputs
    # (Codes from elsewhere, or from another compiled graph, have no version; a copy of the streams has its own.)
    packed, version = getattr(codes, "_streams", (None, None))
    if packed == id(x):
        _check_version(x, version)
    _out, lo_codes, lo_scales = output
    ctx.save_for_backward(codes, scales, lo_codes, lo_scales, H_merged, h_post, graph_link(x_sink, lo))
    ctx.set_materialize_grads(False)


@differentiable_once
def _mhc_post_res_pack8_backward(ctx, grad_out, _gc, _gs):
    if grad_out is None:
        return (None,) * 7
    g_x, g_lo, g_H, g_hp = torch.ops.flash_mhc.fused_post_res_backward_pack8(grad_out, *ctx.saved_tensors[:-1])
    return None, g_x, None, None, g_lo, g_H, g_hp  # x's gradient goes to the sink


torch.library.register_autograd("flash_mhc::mhc_post_res_pack8", _mhc_post_res_pack8_backward,
                                setup_context=_setup_mhc_post_res)


def _stream_of(t) -> int:
    return _abi.stream_of(t) if t.is_cuda else 0


def _borrow(tensors, stream: int) -> None:
    """Use tensors that were made on `stream` on the current one: after what made
    them, and their memory is not given away before that use is over."""
    dev = tensors[0].device
    now = torch.cuda.current_stream(dev)
    now.wait_stream(torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev))
    for t in tensors:
        t.record_stream(now)


class _Kept:
    """The codes of a block's streams, on their way from post-res, whose forward
    makes and saves them, to the pre-map's backward, which runs after
    post-res's."""

    __slots__ = ("version", "post", "stream", "codes")

    def __init__(self, version):
        self.version = version  # of the streams when the pre-map read them
        self.post = None        # weak: post-res's node leads to the pre-map's
        self.stream = 0         # that post-res ran on, the pre-map's unless the layer left another one current
        self.codes = None

    def take(self):
        """(x_codes, x_scales).  Post-res's backward has left them here; where it
        was not part of this backward (a loss on the layer's input alone), they
        are still with post-res's node."""
        codes, self.codes = self.codes, None
        if codes is None:
            post = self.post() if self.post is not None else None
            if post is None:
                raise RuntimeError(
                    "activation_bits=8: the block's output is gone, and its 8-bit activations with it; keep the output "
                    "until its layer input's gradient is taken, or use activation_bits=16")
            codes = post.saved_tensors[:2]
        if _stream_of(codes[0]) != self.stream:
            _borrow(codes, self.stream)
        return codes


class _PreMapEager(torch.autograd.Function):
    """mhc_pre_map without the op's dispatch (ops._PreMapEager), whose backward
    reads the streams' codes from `kept`.  Returns (layer_input, H_merged,
    h_post, x_sink)."""

    @staticmethod
    def forward(ctx, x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat, kept):
        li, H, hq, h_pre, proj, inv_rms, x_sink = _mhc_pre_map_cuda(x_streams, W, alpha_pre, alpha_post, alpha_res,
                                                                     bias, perm_mat)
        ctx.kept = kept
        # (h_post, an output that post-res keeps as well, for differentiable_once)
        ctx.save_for_backward(W, alpha_pre, alpha_post, alpha_res, bias, perm_mat, h_pre, proj, inv_rms, hq)
        ctx.set_materialize_grads(False)
        return li, H, hq, x_sink

    @staticmethod
    @differentiable_once
    def backward(ctx, g_li, g_H, g_hq, g_sink):
        *saved, _hq = ctx.saved_tensors
        grads = _mhc_pre_map_backward_pack8_cuda(g_li, g_H, g_hq, None, None, g_sink, *ctx.kept.take(), *saved)
        return (*grads, None, None)


class _PostResEager(torch.autograd.Function):
    """mhc_post_res without the op's dispatch, which packs x and the layer output
    in its own pass (fused_post_res_pack8's kernel): x's gradient goes to x_sink.
    With a residual the layer output is residual + layer_output."""

    @staticmethod
    def forward(ctx, x_streams, x_sink, layer_output, H_merged, h_post, kept, residual):
        _check_version(x_streams, kept.version)
        out, *codes = _k.k4_fwd_pack8(x_streams.contiguous(), layer_output.contiguous(), _coeff(H_merged),
                                      _coeff(h_post), residual=None if residual is None else residual.contiguous())
        ctx.kept = kept
        ctx.residual = residual is not None
        kept.post = weakref.ref(ctx)
        kept.stream = _stream_of(out)
        link = h_post.detach()  # h_post as a second output, for differentiable_once
        ctx.save_for_backward(*codes, H_merged, link)
        ctx.set_materialize_grads(False)
        return out, link

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_out, _link):
        if grad_out is None:
            return (None,) * 7
        *codes, H_merged, h_post = ctx.saved_tensors
        # Not where no pre-map's backward will take them (frozen streams and coefficients).
        _x, x_sink, _lo, H, hp, _kept, _res = ctx.needs_input_grad
        if x_sink or H or hp:
            ctx.kept.codes = codes[:2]
        g_x, g_lo, g_H, g_hp = _k.k4_bwd_pack8_saved(grad_out.contiguous(), *codes, _coeff(H_merged), _coeff(h_post))
        return None, g_x, g_lo, g_H, g_hp, None, g_lo if ctx.residual else None


def pre_map_eager(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat):
    """(layer_input, H_merged, h_post, x_sink, kept) of mhc_pre_map, recorded for
    autograd without the op's dispatch; `kept` goes to post_res_eager for the
    same streams, whose forward packs them for this one's backward."""
    kept = _Kept(_version(x_streams))
    return (*_PreMapEager.apply(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm_mat, kept), kept)


def post_res_eager(x_streams, x_sink, layer_output, H_merged, h_post, kept, residual=None):
    """mhc_post_res of layer_output, or of residual + layer_output, recorded for
    autograd without the op's dispatch, keeping codes."""
    if residual is not None and (layer_output.shape != residual.shape or layer_output.dtype is not residual.dtype
                                 or layer_output.device != residual.device):
        layer_output, residual = residual + layer_output, None  # as PyTorch adds them
    return _PostResEager.apply(x_streams, x_sink, layer_output, H_merged, h_post, kept, residual)[0]


# ---------------------------------------------------------------------------
# Public functions


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (..., C), bf16, fp16 or fp32 on the GPU, as (codes, scales): int8 (..., C)
    and uint8 (..., ceil(C / 32)).  Not differentiable.

    A group of 32 columns whose largest magnitude is in [2^e, 2^(e + 1)) has the
    scale byte e + 127 (at least 7) and stands for code * 2^(e - 6); a group
    with an Inf or NaN has 255 and stands for NaN throughout."""
    if _block._plain_eager(x):
        return _pack8_cuda(x)
    return torch.ops.flash_mhc.pack8(x)


def unpack8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The tensor that pack8's codes and scales stand for, exact in bf16 and fp32
    (and in fp16 for what was packed from fp16)."""
    if _block._plain_eager(codes):
        return _unpack8_cuda(codes, scales, dtype)
    return torch.ops.flash_mhc.unpack8(codes, scales, dtype)
