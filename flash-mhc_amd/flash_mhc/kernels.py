"""Launchers for the gfx950 HIP kernels (drop-in for the reference's Triton
``kernels.py``).

Each function validates its tensors, allocates any output that was not passed
in, and enqueues one kernel through the C ABI on torch's current stream of
the tensors' device.  Nothing here falls back to another implementation: a
missing extension or a bad argument raises.

Reference counterparts (alint77/flash-mHC):
  k1_fwd     <- src/flash_mhc/kernels.py:250-303  _fused_rmsnorm_project_fwd_kernel
  k1_bwd_dx  <- src/flash_mhc/kernels.py:306-376  _fused_rmsnorm_project_bwd_dx_kernel
  k1_bwd     <- the above plus the grad_W matmul of src/flash_mhc/ops.py:683-684, fused
  k2_fwd     <- src/flash_mhc/block.py:161-170 (PyTorch ops) and the .float() casts of :176-177
  k2_bwd     <- autograd through the same ops
  premap_fwd <- K1 + K2 + K3 of src/flash_mhc/block.py:157-177 (one entry point)
  premap_bwd <- autograd through the same, x's two gradients summed in K1's store
  k3_fwd     <- src/flash_mhc/kernels.py:673-717  _fused_pre_map_fwd_kernel
  k3_bwd     <- src/flash_mhc/kernels.py:720-853  _fused_pre_map_bwd_fused_kernel_n4
  k4_fwd     <- src/flash_mhc/kernels.py:384-481  _fused_post_res_fwd_kernel_n4
  k4_bwd     <- src/flash_mhc/kernels.py:487-665  _fused_post_res_bwd_fused_kernel_n4

Without a counterpart there:
  pack8, unpack8             activations to 8 bits and back
  k4_fwd_pack8, k4_bwd_pack8, k1_bwd_pack8, premap_bwd_pack8
                             K4's forward that keeps its inputs in 8 bits, and
                             the backward passes that read them
  layer_norm_fwd, layer_norm_bwd
  rms_norm_fwd, rms_norm_bwd
  pack8_rows, rms_norm_pack8_rows, linear8
                             rows in 8 bits with a scale each, and their product
"""

from __future__ import annotations

import torch

from . import _abi

N_STREAMS = 4
D_OUT = 32  # 2n + n! at n = 4

_BF16 = torch.bfloat16
_F32 = torch.float32


def _require(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...], device) -> None:
    # One compound test on the common path; the messages come from _reject.
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or t.device != device
            or not t.is_contiguous()):
        _reject(t, name, dtype, shape, device)


def _reject(t, name: str, dtype: torch.dtype, shape: tuple[int, ...], device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:  # torch.Size compares equal to a tuple of the same ints
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _device_of(x: torch.Tensor) -> torch.device:
    if not isinstance(x, torch.Tensor):
        raise TypeError("expected a torch.Tensor")
    if x.device.type != "cuda":
        raise ValueError(f"flash_mhc HIP kernels need a GPU tensor, got device {x.device}")
    return x.device


class _OnDevice:
    """Make ``device`` current for the launch (cheap when it already is)."""

    __slots__ = ("idx", "prev")

    def __init__(self, device: torch.device):
        idx = device.index
        self.idx = torch.cuda.current_device() if idx is None else idx
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


def k1_fwd(x_flat: torch.Tensor, W: torch.Tensor, out: torch.Tensor | None = None,
           inv_rms: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """proj (T, 32) bf16 and inv_rms (T,) fp32 from x_flat (T, nC) bf16, W (32, nC) bf16
    (fmhc_k1_fwd_ws: few tokens split the nC axis over workgroups)."""
    dev = _device_of(x_flat)
    if x_flat.dim() != 2:
        raise ValueError(f"x_flat must be 2-D (T, nC), got shape {tuple(x_flat.shape)}")
    T, nC = x_flat.shape
    _require(x_flat, "x_flat", _BF16, (T, nC), dev)
    if W.dim() != 2 or W.shape[0] != D_OUT:
        raise ValueError(f"W must have shape ({D_OUT}, nC); got {tuple(W.shape)}")
    _require(W, "W", _BF16, (D_OUT, nC), dev)
    if out is None:
        out = torch.empty((T, D_OUT), device=dev, dtype=_BF16)
    if inv_rms is None:
        inv_rms = torch.empty((T,), device=dev, dtype=_F32)
    _require(out, "out", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    lib = _abi.load()
    ws = _workspace(int(lib.fmhc_k1_fwd_workspace_bytes(T, nC)), dev)
    with _OnDevice(dev):
        st = lib.fmhc_k1_fwd_ws(x_flat.data_ptr(), W.data_ptr(), out.data_ptr(), inv_rms.data_ptr(),
                                _ptr_or_none(ws), 0 if ws is None else ws.numel(), T, nC, D_OUT,
                                _abi.stream_of(x_flat))
    _abi.check(st, "k1_fwd")
    return out, inv_rms


def k1_bwd_dx(grad_out: torch.Tensor, x_flat: torch.Tensor, W: torch.Tensor,
              proj_out: torch.Tensor, inv_rms: torch.Tensor,
              grad_x: torch.Tensor | None = None) -> torch.Tensor:
    """grad of x_flat for K1, from the stored bf16 projection and inv_rms."""
    dev = _device_of(x_flat)
    if x_flat.dim() != 2:
        raise ValueError(f"x_flat must be 2-D (T, nC), got shape {tuple(x_flat.shape)}")
    T, nC = x_flat.shape
    _require(x_flat, "x_flat", _BF16, (T, nC), dev)
    _require(W, "W", _BF16, (D_OUT, nC), dev)
    _require(grad_out, "grad_out", _BF16, (T, D_OUT), dev)
    _require(proj_out, "proj_out", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    if grad_x is None:
        grad_x = torch.empty_like(x_flat)
    _require(grad_x, "grad_x", _BF16, (T, nC), dev)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k1_bwd_dx(x_flat.data_ptr(), W.data_ptr(), grad_out.data_ptr(),
                                proj_out.data_ptr(), inv_rms.data_ptr(), grad_x.data_ptr(),
                                T, nC, D_OUT, _abi.stream_of(x_flat))
    _abi.check(st, "k1_bwd_dx")
    return grad_x


def k1_bwd(grad_out: torch.Tensor, x_flat: torch.Tensor, W: torch.Tensor,
           proj_out: torch.Tensor, inv_rms: torch.Tensor,
           grad_x: torch.Tensor | None = None,
           grad_W: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(grad_x, grad_W) of K1 in one pass over x; grad_W is (32, nC) bf16 and
    equals bf16(bf16(grad_out * inv_rms)^T @ x_flat) up to fp32 summation order."""
    dev = _device_of(x_flat)
    if x_flat.dim() != 2:
        raise ValueError(f"x_flat must be 2-D (T, nC), got shape {tuple(x_flat.shape)}")
    T, nC = x_flat.shape
    _require(x_flat, "x_flat", _BF16, (T, nC), dev)
    _require(W, "W", _BF16, (D_OUT, nC), dev)
    _require(grad_out, "grad_out", _BF16, (T, D_OUT), dev)
    _require(proj_out, "proj_out", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    if grad_x is None:
        grad_x = torch.empty_like(x_flat)
    if grad_W is None:
        grad_W = torch.empty((D_OUT, nC), device=dev, dtype=_BF16)
    _require(grad_x, "grad_x", _BF16, (T, nC), dev)
    _require(grad_W, "grad_W", _BF16, (D_OUT, nC), dev)
    lib = _abi.load()
    nbytes = int(lib.fmhc_k1_bwd_workspace_bytes(T, nC))
    ws = torch.empty((max(nbytes, 16),), device=dev, dtype=torch.uint8)
    with _OnDevice(dev):
        st = lib.fmhc_k1_bwd(x_flat.data_ptr(), W.data_ptr(), grad_out.data_ptr(), proj_out.data_ptr(),
                             inv_rms.data_ptr(), grad_x.data_ptr(), grad_W.data_ptr(), ws.data_ptr(),
                             ws.numel(), T, nC, D_OUT, _abi.stream_of(x_flat))
    _abi.check(st, "k1_bwd")
    return grad_x, grad_W


N_PERM = 24  # n! at n = 4


PARAM_DTYPES = {_F32: 0, _BF16: 1}  # FMHC_PARAM_F32, FMHC_PARAM_BF16


_K2_NAMES = ("alpha_pre", "alpha_post", "alpha_res", "bias", "perm")
_K2_SHAPES = ((1,), (1,), (1,), (D_OUT,), (N_PERM, N_STREAMS * N_STREAMS))


def _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev) -> int:
    """Check K2's parameters (all fp32 or all bf16) and return the ABI's dtype code."""
    dt = alpha_pre.dtype if isinstance(alpha_pre, torch.Tensor) else None
    code = PARAM_DTYPES.get(dt)
    if code is None:
        raise TypeError(f"K2 parameters must be float32 or bfloat16, got {dt}")
    ps = (alpha_pre, alpha_post, alpha_res, bias, perm)
    for t, shape in zip(ps, _K2_SHAPES):
        if (not isinstance(t, torch.Tensor) or t.dtype is not dt or t.shape != shape or t.device != dev
                or not t.is_contiguous()):
            break
    else:
        return code
    for t, name, shape in zip(ps, _K2_NAMES, _K2_SHAPES):
        _require(t, name, dt, shape, dev)
    return code


def k2_fwd(proj: torch.Tensor, alpha_pre: torch.Tensor, alpha_post: torch.Tensor,
           alpha_res: torch.Tensor, bias: torch.Tensor, perm: torch.Tensor
           ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(h_pre (T,4), h_post (T,4), H_merged (T,4,4)) fp32 from proj (T,32) bf16,
    with the bf16 rounding points of the reference's coefficient ops.
    Parameters: alphas (1,), bias (32,), perm (24,16), all fp32 or all bf16."""
    dev = _device_of(proj)
    if proj.dim() != 2:
        raise ValueError(f"proj must be 2-D (T, 32), got shape {tuple(proj.shape)}")
    T = proj.shape[0]
    _require(proj, "proj", _BF16, (T, D_OUT), dev)
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    h_pre = torch.empty((T, N_STREAMS), device=dev, dtype=_F32)
    h_post = torch.empty((T, N_STREAMS), device=dev, dtype=_F32)
    H = torch.empty((T, N_STREAMS, N_STREAMS), device=dev, dtype=_F32)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k2_fwd(proj.data_ptr(), alpha_pre.data_ptr(), alpha_post.data_ptr(),
                             alpha_res.data_ptr(), bias.data_ptr(), perm.data_ptr(), pdt, h_pre.data_ptr(),
                             h_post.data_ptr(), H.data_ptr(), T, N_STREAMS, _abi.stream_of(proj))
    _abi.check(st, "k2_fwd")
    return h_pre, h_post, H


def k2_bwd(proj: torch.Tensor, alpha_pre: torch.Tensor, alpha_post: torch.Tensor,
           alpha_res: torch.Tensor, bias: torch.Tensor, perm: torch.Tensor,
           grad_h_pre: torch.Tensor | None, grad_h_post: torch.Tensor | None,
           grad_H: torch.Tensor | None):
    """Gradients of k2_fwd: (grad_proj (T,32) bf16, grad_alpha_pre (1,),
    grad_alpha_post (1,), grad_alpha_res (1,), grad_bias (32,)), parameter
    gradients in the parameters' dtype.  A None output gradient counts as zero."""
    dev = _device_of(proj)
    if proj.dim() != 2:
        raise ValueError(f"proj must be 2-D (T, 32), got shape {tuple(proj.shape)}")
    T = proj.shape[0]
    _require(proj, "proj", _BF16, (T, D_OUT), dev)
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    for t, name, shape in ((grad_h_pre, "grad_h_pre", (T, N_STREAMS)),
                           (grad_h_post, "grad_h_post", (T, N_STREAMS)),
                           (grad_H, "grad_H_merged", (T, N_STREAMS, N_STREAMS))):
        if t is not None:
            _require(t, name, _F32, shape, dev)
    grad_proj = torch.empty((T, D_OUT), device=dev, dtype=_BF16)
    g_ap = torch.empty((1,), device=dev, dtype=alpha_pre.dtype)
    g_apo = torch.empty((1,), device=dev, dtype=alpha_pre.dtype)
    g_ar = torch.empty((1,), device=dev, dtype=alpha_pre.dtype)
    g_b = torch.empty((D_OUT,), device=dev, dtype=alpha_pre.dtype)
    lib = _abi.load()
    nbytes = int(lib.fmhc_k2_bwd_workspace_bytes(T))
    ws = torch.empty((max(nbytes, 16),), device=dev, dtype=torch.uint8)
    ptr = lambda t: None if t is None else t.data_ptr()
    with _OnDevice(dev):
        st = lib.fmhc_k2_bwd(proj.data_ptr(), alpha_pre.data_ptr(), alpha_post.data_ptr(),
                             alpha_res.data_ptr(), bias.data_ptr(), perm.data_ptr(), pdt, ptr(grad_h_pre),
                             ptr(grad_h_post), ptr(grad_H), grad_proj.data_ptr(), g_ap.data_ptr(),
                             g_apo.data_ptr(), g_ar.data_ptr(), g_b.data_ptr(), ws.data_ptr(), ws.numel(),
                             T, N_STREAMS, _abi.stream_of(proj))
    _abi.check(st, "k2_bwd")
    return grad_proj, g_ap, g_apo, g_ar, g_b


def premap_fwd(x_streams: torch.Tensor, W: torch.Tensor, alpha_pre: torch.Tensor,
               alpha_post: torch.Tensor, alpha_res: torch.Tensor, bias: torch.Tensor,
               perm: torch.Tensor, layer_input: bool = True, zero: tuple = ()):
    """K1 + K2 + K3: (layer_input (T,C) bf16, H_merged (T,4,4), h_post (T,4),
    h_pre (T,4) fp32, proj (T,32) bf16, inv_rms (T,) fp32).  layer_input=False:
    K1 + K2 only, the first output is None.  zero: up to two 16-bit tensors
    whose first stored element the same launches set to zero (zero-stride
    placeholders; empty ones are skipped)."""
    if len(zero) > 2 or any(z.element_size() != 2 for z in zero):
        raise ValueError("premap_fwd: zero takes up to two 16-bit tensors")
    zw = [z.data_ptr() if z.numel() > 0 else None for z in zero] + [None, None]
    T, n, C = _streams_shape(x_streams)
    dev = _device_of(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(W, "W", _BF16, (D_OUT, n * C), dev)
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    li = torch.empty((T, C), device=dev, dtype=_BF16) if layer_input else None
    proj = torch.empty((T, D_OUT), device=dev, dtype=_BF16)
    inv = torch.empty((T,), device=dev, dtype=_F32)
    h_pre = torch.empty((T, n), device=dev, dtype=_F32)
    h_post = torch.empty((T, n), device=dev, dtype=_F32)
    H = torch.empty((T, n, n), device=dev, dtype=_F32)
    lib = _abi.load()
    ws = _workspace(int(lib.fmhc_premap_fwd_workspace_bytes(T, C)), dev)
    with _OnDevice(dev):
        st = lib.fmhc_premap_fwd(x_streams.data_ptr(), W.data_ptr(), alpha_pre.data_ptr(),
                                 alpha_post.data_ptr(), alpha_res.data_ptr(), bias.data_ptr(),
                                 perm.data_ptr(), pdt, _ptr_or_none(li), proj.data_ptr(), inv.data_ptr(),
                                 h_pre.data_ptr(), h_post.data_ptr(), H.data_ptr(), zw[0], zw[1],
                                 _ptr_or_none(ws), 0 if ws is None else ws.numel(), T, C, n,
                                 _abi.stream_of(x_streams))
    _abi.check(st, "premap_fwd")
    return li, H, h_post, h_pre, proj, inv


_PREMAP_WS_BYTES: dict[tuple[int, int], int] = {}


def _premap_ws_bytes(lib, T: int, C: int) -> int:
    key = (T, C)
    n = _PREMAP_WS_BYTES.get(key)
    if n is None:
        if len(_PREMAP_WS_BYTES) > 4096:
            _PREMAP_WS_BYTES.clear()
        n = _PREMAP_WS_BYTES[key] = int(lib.fmhc_premap_fwd_workspace_bytes(T, C))
    return n


def premap_fwd_eval(x_streams: torch.Tensor, W: torch.Tensor, alpha_pre: torch.Tensor,
                    alpha_post: torch.Tensor, alpha_res: torch.Tensor, bias: torch.Tensor,
                    perm: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """premap_fwd for a forward that records no autograd graph: the same
    launch, returning (layer_input, coeffs).  coeffs is one uint8 scratch
    buffer that holds H_merged (T, 4, 4) fp32 at byte 0 and h_post (T, 4)
    fp32 at byte 64 T, the inputs k4_fwd_eval reads, followed by h_pre, proj,
    inv_rms and the workspace, which nothing reads after the call: one
    allocation instead of six."""
    dev = x_streams.device
    shape = x_streams.shape
    if (len(shape) != 3 or shape[1] != N_STREAMS or dev.type != "cuda" or x_streams.dtype is not _BF16
            or not x_streams.is_contiguous() or W.dtype is not _BF16 or W.device != dev
            or W.shape != (D_OUT, N_STREAMS * shape[2]) or not W.is_contiguous()):
        T, n, C = _streams_shape(x_streams)
        dev = _device_of(x_streams)
        _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
        _require(W, "W", _BF16, (D_OUT, n * C), dev)
    T, n, C = shape
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    lib = _abi.load()
    ws_bytes = _premap_ws_bytes(lib, T, C)
    li = torch.empty((T, C), device=dev, dtype=_BF16)
    # H_merged | h_post | h_pre | inv_rms | proj | workspace, 16-byte aligned pieces
    o_hq, o_hp, o_inv = 64 * T, 80 * T, 96 * T
    o_proj = (o_inv + 4 * T + 15) // 16 * 16
    o_ws = (o_proj + 2 * D_OUT * T + 255) // 256 * 256
    coeffs = torch.empty((o_ws + ws_bytes,), device=dev, dtype=torch.uint8)
    base = coeffs.data_ptr()
    with _OnDevice(dev):
        st = lib.fmhc_premap_fwd(x_streams.data_ptr(), W.data_ptr(), alpha_pre.data_ptr(),
                                 alpha_post.data_ptr(), alpha_res.data_ptr(), bias.data_ptr(),
                                 perm.data_ptr(), pdt, li.data_ptr(), base + o_proj, base + o_inv, base + o_hp,
                                 base + o_hq, base, None, None,
                                 base + o_ws if ws_bytes else None, ws_bytes, T, C, n, _abi.stream_of(x_streams))
    _abi.check(st, "premap_fwd")
    return li, coeffs


def premap_bwd(x_streams: torch.Tensor, W: torch.Tensor, alpha_pre: torch.Tensor,
               alpha_post: torch.Tensor, alpha_res: torch.Tensor, bias: torch.Tensor,
               perm: torch.Tensor, h_pre: torch.Tensor, proj: torch.Tensor, inv_rms: torch.Tensor,
               grad_layer_input: torch.Tensor, grad_h_post: torch.Tensor | None,
               grad_H: torch.Tensor | None, grad_x_in: torch.Tensor | None = None):
    """Gradients of premap_fwd's inputs: (grad_x (T,4,C) bf16, grad_W (32,4C) bf16,
    grad_alpha_pre, grad_alpha_post, grad_alpha_res (1,), grad_bias (32,) in the parameters' dtype).
    grad_x_in (T,4,C) bf16, optional: a further gradient of x, added (bf16) into grad_x."""
    T, n, C = _streams_shape(x_streams)
    dev = _device_of(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(W, "W", _BF16, (D_OUT, n * C), dev)
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    _require(h_pre, "h_pre", _F32, (T, n), dev)
    _require(proj, "proj", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    _require(grad_layer_input, "grad_layer_input", _BF16, (T, C), dev)
    if grad_h_post is not None:
        _require(grad_h_post, "grad_h_post", _F32, (T, n), dev)
    if grad_H is not None:
        _require(grad_H, "grad_H_merged", _F32, (T, n, n), dev)
    if grad_x_in is not None:
        _require(grad_x_in, "grad_x_in", _BF16, (T, n, C), dev)
    gx = torch.empty_like(x_streams)
    gW = torch.empty((D_OUT, n * C), device=dev, dtype=_BF16)
    ga = [torch.empty((1,), device=dev, dtype=alpha_pre.dtype) for _ in range(3)]
    gb = torch.empty((D_OUT,), device=dev, dtype=alpha_pre.dtype)
    lib = _abi.load()
    nbytes = int(lib.fmhc_premap_bwd_workspace_bytes(T, C))
    ws = torch.empty((max(nbytes, 16),), device=dev, dtype=torch.uint8)
    ptr = lambda t: None if t is None else t.data_ptr()
    with _OnDevice(dev):
        st = lib.fmhc_premap_bwd(x_streams.data_ptr(), W.data_ptr(), alpha_pre.data_ptr(),
                                 alpha_post.data_ptr(), alpha_res.data_ptr(), bias.data_ptr(),
                                 perm.data_ptr(), pdt, h_pre.data_ptr(), proj.data_ptr(), inv_rms.data_ptr(),
                                 grad_layer_input.data_ptr(), ptr(grad_h_post), ptr(grad_H), ptr(grad_x_in),
                                 gx.data_ptr(),
                                 gW.data_ptr(), ga[0].data_ptr(), ga[1].data_ptr(), ga[2].data_ptr(),
                                 gb.data_ptr(), ws.data_ptr(), ws.numel(), T, C, n, _abi.stream_of(x_streams))
    _abi.check(st, "premap_bwd")
    return gx, gW, ga[0], ga[1], ga[2], gb


def _workspace(nbytes: int, dev) -> torch.Tensor | None:
    """A uint8 device buffer of nbytes (16-byte aligned: torch's allocations are), or None for 0."""
    return torch.empty((nbytes,), device=dev, dtype=torch.uint8) if nbytes > 0 else None


def _ptr_or_none(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _streams_shape(x: torch.Tensor) -> tuple[int, int, int]:
    if x.dim() != 3:
        raise ValueError(f"x_streams must be 3-D (T, n, C), got shape {tuple(x.shape)}")
    T, n, C = x.shape
    if n != N_STREAMS:
        raise ValueError(f"flash_mhc HIP kernels support n={N_STREAMS} only, got n={n}")
    return T, n, C


def k3_fwd(x_streams: torch.Tensor, h_pre: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """layer_input (T, C) bf16 = sum_j h_pre[:, j] * x_streams[:, j, :]."""
    dev = _device_of(x_streams)
    T, n, C = _streams_shape(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(h_pre, "h_pre", _F32, (T, n), dev)
    if out is None:
        out = torch.empty((T, C), device=dev, dtype=_BF16)
    _require(out, "out", _BF16, (T, C), dev)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k3_fwd(x_streams.data_ptr(), h_pre.data_ptr(), out.data_ptr(), T, C, n,
                             _abi.stream_of(x_streams))
    _abi.check(st, "k3_fwd")
    return out


def k3_bwd(grad_out: torch.Tensor, x_streams: torch.Tensor, h_pre: torch.Tensor,
           grad_x: torch.Tensor | None = None,
           grad_h_pre: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(grad_x (T, n, C) bf16, grad_h_pre (T, n) fp32) of K3."""
    dev = _device_of(x_streams)
    T, n, C = _streams_shape(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(h_pre, "h_pre", _F32, (T, n), dev)
    _require(grad_out, "grad_out", _BF16, (T, C), dev)
    if grad_x is None:
        grad_x = torch.empty_like(x_streams)
    if grad_h_pre is None:
        grad_h_pre = torch.empty((T, n), device=dev, dtype=_F32)
    _require(grad_x, "grad_x", _BF16, (T, n, C), dev)
    _require(grad_h_pre, "grad_h_pre", _F32, (T, n), dev)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k3_bwd(x_streams.data_ptr(), h_pre.data_ptr(), grad_out.data_ptr(),
                             grad_x.data_ptr(), grad_h_pre.data_ptr(), T, C, n,
                             _abi.stream_of(x_streams))
    _abi.check(st, "k3_bwd")
    return grad_x, grad_h_pre


def k4_fwd(x_streams: torch.Tensor, layer_output: torch.Tensor, H_merged: torch.Tensor,
           h_post: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out (T, n, C) bf16 = H_merged @ x_streams + h_post (x) layer_output."""
    dev = _device_of(x_streams)
    T, n, C = _streams_shape(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(layer_output, "layer_output", _BF16, (T, C), dev)
    _require(H_merged, "H_merged", _F32, (T, n, n), dev)
    _require(h_post, "h_post", _F32, (T, n), dev)
    if out is None:
        out = torch.empty_like(x_streams)
    _require(out, "out", _BF16, (T, n, C), dev)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k4_fwd(x_streams.data_ptr(), layer_output.data_ptr(), H_merged.data_ptr(),
                             h_post.data_ptr(), out.data_ptr(), T, C, n, _abi.stream_of(x_streams))
    _abi.check(st, "k4_fwd")
    return out


def k4_fwd_eval(x_streams: torch.Tensor, layer_output: torch.Tensor, coeffs: torch.Tensor) -> torch.Tensor:
    """k4_fwd with H_merged and h_post read from premap_fwd_eval's coeffs
    buffer for the same x_streams."""
    dev = x_streams.device
    shape = x_streams.shape
    if (len(shape) != 3 or shape[1] != N_STREAMS or dev.type != "cuda" or x_streams.dtype is not _BF16
            or not x_streams.is_contiguous() or layer_output.dtype is not _BF16 or layer_output.device != dev
            or layer_output.shape != (shape[0], shape[2]) or not layer_output.is_contiguous()):
        T, n, C = _streams_shape(x_streams)
        dev = _device_of(x_streams)
        _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
        _require(layer_output, "layer_output", _BF16, (T, C), dev)
    T, n, C = shape
    if coeffs.dtype is not torch.uint8 or coeffs.numel() < 80 * T or coeffs.device != dev:
        raise ValueError("coeffs is not premap_fwd_eval's buffer for these tokens")
    out = torch.empty_like(x_streams)
    lib = _abi.load()
    base = coeffs.data_ptr()
    with _OnDevice(dev):
        st = lib.fmhc_k4_fwd(x_streams.data_ptr(), layer_output.data_ptr(), base, base + 64 * T,
                             out.data_ptr(), T, C, n, _abi.stream_of(x_streams))
    _abi.check(st, "k4_fwd")
    return out


def k4_bwd(grad_out: torch.Tensor, x_streams: torch.Tensor, layer_output: torch.Tensor,
           H_merged: torch.Tensor, h_post: torch.Tensor,
           grad_x: torch.Tensor | None = None, grad_layer_output: torch.Tensor | None = None,
           grad_H: torch.Tensor | None = None, grad_h_post: torch.Tensor | None = None):
    """(grad_x, grad_layer_output, grad_H_merged, grad_h_post) of K4."""
    dev = _device_of(x_streams)
    T, n, C = _streams_shape(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(layer_output, "layer_output", _BF16, (T, C), dev)
    _require(H_merged, "H_merged", _F32, (T, n, n), dev)
    _require(h_post, "h_post", _F32, (T, n), dev)
    _require(grad_out, "grad_out", _BF16, (T, n, C), dev)
    if grad_x is None:
        grad_x = torch.empty_like(x_streams)
    if grad_layer_output is None:
        grad_layer_output = torch.empty((T, C), device=dev, dtype=_BF16)
    if grad_H is None:
        grad_H = torch.empty((T, n, n), device=dev, dtype=_F32)
    if grad_h_post is None:
        grad_h_post = torch.empty((T, n), device=dev, dtype=_F32)
    _require(grad_x, "grad_x", _BF16, (T, n, C), dev)
    _require(grad_layer_output, "grad_layer_output", _BF16, (T, C), dev)
    _require(grad_H, "grad_H", _F32, (T, n, n), dev)
    _require(grad_h_post, "grad_h_post", _F32, (T, n), dev)
    lib = _abi.load()
    with _OnDevice(dev):
        st = lib.fmhc_k4_bwd(x_streams.data_ptr(), layer_output.data_ptr(), H_merged.data_ptr(),
                             h_post.data_ptr(), grad_out.data_ptr(), grad_x.data_ptr(),
                             grad_layer_output.data_ptr(), grad_H.data_ptr(), grad_h_post.data_ptr(),
                             T, C, n, _abi.stream_of(x_streams))
    _abi.check(st, "k4_bwd")
    return grad_x, grad_layer_output, grad_H, grad_h_post


# ---------------------------------------------------------------------------
# Activations in 8 bits (the format: include/flash_mhc_hip.h)

PACK_GROUP = 32  # columns that share a scale
DTYPES = {_F32: 0, _BF16: 1, torch.float16: 2}  # FMHC_DTYPE_*


def pack_groups(C: int) -> int:
    """Scales of a row of C columns."""
    return (C + PACK_GROUP - 1) // PACK_GROUP


def _dtype_code(dt: torch.dtype, name: str) -> int:
    code = DTYPES.get(dt)
    if code is None:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {dt}")
    return code


def _rows(x: torch.Tensor, name: str) -> tuple[int, int]:
    """(rows, C) of x (..., C), which must be contiguous."""
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"expected shape (..., C) with C >= 1, got {tuple(shape)}")
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return x.numel() // shape[-1], shape[-1]


def empty_packed(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Unwritten (codes, scales) for a contiguous x."""
    shape = x.shape
    return (torch.empty_like(x, dtype=torch.int8),
            x.new_empty((*shape[:-1], (shape[-1] + PACK_GROUP - 1) // PACK_GROUP), dtype=torch.uint8))


def _launch(what: str, dev: torch.device, fn, *args) -> None:
    """fn(*args) with dev current (it nearly always is), its status checked."""
    if torch.cuda.current_device() == dev.index:
        st = fn(*args)
    else:
        with _OnDevice(dev):
            st = fn(*args)
    if st != 0:
        _abi.check(st, what)


def _require_packed(codes, scales, name: str, shape, dev) -> None:
    shape = tuple(shape)
    _require(codes, f"{name}_codes", torch.int8, shape, dev)
    _require(scales, f"{name}_scales", torch.uint8, (*shape[:-1], pack_groups(shape[-1])), dev)


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """codes (..., C) int8 and scales (..., ceil(C / 32)) uint8 of x (..., C)."""
    dev = _device_of(x)
    code = _dtype_code(x.dtype, "x")
    rows, C = _rows(x, "x")
    codes, scales = empty_packed(x)
    _launch("pack8", dev, _abi.load().fmhc_pack8, x.data_ptr(), code, codes.data_ptr(), scales.data_ptr(), rows, C,
            _abi.stream_of(x))
    return codes, scales


def unpack8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = _BF16) -> torch.Tensor:
    """The values of pack8's codes and scales, in dtype."""
    dev = _device_of(codes)
    code = _dtype_code(dtype, "dtype")
    rows, C = _rows(codes, "x_codes")
    _require_packed(codes, scales, "x", codes.shape, dev)
    x = torch.empty_like(codes, dtype=dtype)
    _launch("unpack8", dev, _abi.load().fmhc_unpack8, codes.data_ptr(), scales.data_ptr(), x.data_ptr(), code, rows, C,
            _abi.stream_of(codes))
    return x


def k4_fwd_pack8(x_streams: torch.Tensor, layer_output: torch.Tensor, H_merged: torch.Tensor, h_post: torch.Tensor,
                 pack_x: bool = True, residual: torch.Tensor | None = None):
    """k4_fwd's out with x_streams (unless pack_x is false) and layer_output packed
    in the same pass: (out, x_codes, x_scales, lo_codes, lo_scales).  With a
    residual (T, C), and pack_x, residual + layer_output takes layer_output's place."""
    dev = _device_of(x_streams)
    T, n, C = _streams_shape(x_streams)
    _require(x_streams, "x_streams", _BF16, (T, n, C), dev)
    _require(layer_output, "layer_output", _BF16, (T, C), dev)
    _require(H_merged, "H_merged", _F32, (T, n, n), dev)
    _require(h_post, "h_post", _F32, (T, n), dev)
    out = torch.empty_like(x_streams)
    xq, xs = empty_packed(x_streams) if pack_x else (None, None)
    lq, ls = empty_packed(layer_output)
    if residual is not None:
        _require(residual, "residual", _BF16, (T, C), dev)
        if not pack_x:
            raise ValueError("k4_fwd_pack8 takes a residual where it packs x_streams")
        _launch("k4_fwd_pack8_residual", dev, _abi.load().fmhc_k4_fwd_pack8_residual, x_streams.data_ptr(),
                layer_output.data_ptr(), residual.data_ptr(), H_merged.data_ptr(), h_post.data_ptr(), out.data_ptr(),
                xq.data_ptr(), xs.data_ptr(), lq.data_ptr(), ls.data_ptr(), T, C, n, _abi.stream_of(x_streams))
        return out, xq, xs, lq, ls
    _launch("k4_fwd_pack8", dev, _abi.load().fmhc_k4_fwd_pack8, x_streams.data_ptr(), layer_output.data_ptr(),
            H_merged.data_ptr(), h_post.data_ptr(), out.data_ptr(), _ptr_or_none(xq), _ptr_or_none(xs), lq.data_ptr(),
            ls.data_ptr(), T, C, n, _abi.stream_of(x_streams))
    return out, xq, xs, lq, ls


def k4_bwd_pack8(grad_out: torch.Tensor, x_codes: torch.Tensor, x_scales: torch.Tensor, lo_codes: torch.Tensor,
                 lo_scales: torch.Tensor, H_merged: torch.Tensor, h_post: torch.Tensor):
    """k4_bwd's outputs from packed x_streams and layer_output."""
    dev = _device_of(x_codes)
    T, n, C = _streams_shape(x_codes)
    _require_packed(x_codes, x_scales, "x", (T, n, C), dev)
    _require_packed(lo_codes, lo_scales, "lo", (T, C), dev)
    _require(H_merged, "H_merged", _F32, (T, n, n), dev)
    _require(h_post, "h_post", _F32, (T, n), dev)
    _require(grad_out, "grad_out", _BF16, (T, n, C), dev)
    return k4_bwd_pack8_saved(grad_out, x_codes, x_scales, lo_codes, lo_scales, H_merged, h_post)


def k4_bwd_pack8_saved(grad_out, x_codes, x_scales, lo_codes, lo_scales, H_merged, h_post):
    """k4_bwd_pack8 for operands that need no checks: what k4_fwd_pack8 took and
    gave, and autograd's gradient of its out, contiguous."""
    T, n, C = x_codes.shape
    grad_x = torch.empty_like(grad_out)
    grad_lo = torch.empty_like(lo_codes, dtype=_BF16)
    grad_H = torch.empty_like(H_merged)
    grad_h_post = torch.empty_like(h_post)
    _launch("k4_bwd_pack8", x_codes.device, _abi.load().fmhc_k4_bwd_pack8, x_codes.data_ptr(), x_scales.data_ptr(),
            lo_codes.data_ptr(), lo_scales.data_ptr(), H_merged.data_ptr(), h_post.data_ptr(), grad_out.data_ptr(),
            grad_x.data_ptr(), grad_lo.data_ptr(), grad_H.data_ptr(), grad_h_post.data_ptr(), T, C, n,
            _abi.stream_of(x_codes))
    return grad_x, grad_lo, grad_H, grad_h_post


def k1_bwd_pack8(grad_out: torch.Tensor, x_codes: torch.Tensor, x_scales: torch.Tensor, W: torch.Tensor,
                 proj_out: torch.Tensor, inv_rms: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(grad_x (T, 4, C), grad_W (32, 4 C)) of K1 from packed streams."""
    dev = _device_of(x_codes)
    T, n, C = _streams_shape(x_codes)
    _require_packed(x_codes, x_scales, "x", (T, n, C), dev)
    _require(W, "W", _BF16, (D_OUT, n * C), dev)
    _require(grad_out, "grad_out", _BF16, (T, D_OUT), dev)
    _require(proj_out, "proj_out", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    grad_x = torch.empty((T, n, C), device=dev, dtype=_BF16)
    grad_W = torch.empty((D_OUT, n * C), device=dev, dtype=_BF16)
    lib = _abi.load()
    ws = _workspace(int(lib.fmhc_k1_bwd_pack8_workspace_bytes(T, C)), dev)
    with _OnDevice(dev):
        st = lib.fmhc_k1_bwd_pack8(x_codes.data_ptr(), x_scales.data_ptr(), W.data_ptr(), grad_out.data_ptr(),
                                   proj_out.data_ptr(), inv_rms.data_ptr(), grad_x.data_ptr(), grad_W.data_ptr(),
                                   _ptr_or_none(ws), 0 if ws is None else ws.numel(), T, C, n,
                                   _abi.stream_of(x_codes))
    _abi.check(st, "k1_bwd_pack8")
    return grad_x, grad_W


def premap_bwd_pack8(x_codes: torch.Tensor, x_scales: torch.Tensor, W: torch.Tensor, alpha_pre: torch.Tensor,
                     alpha_post: torch.Tensor, alpha_res: torch.Tensor, bias: torch.Tensor, perm: torch.Tensor,
                     h_pre: torch.Tensor, proj: torch.Tensor, inv_rms: torch.Tensor, grad_layer_input: torch.Tensor,
                     grad_h_post: torch.Tensor | None, grad_H: torch.Tensor | None,
                     grad_x_in: torch.Tensor | None = None):
    """premap_bwd's outputs from packed streams."""
    dev = _device_of(x_codes)
    T, n, C = _streams_shape(x_codes)
    _require_packed(x_codes, x_scales, "x", (T, n, C), dev)
    _require(W, "W", _BF16, (D_OUT, n * C), dev)
    pdt = _k2_params(alpha_pre, alpha_post, alpha_res, bias, perm, dev)
    _require(h_pre, "h_pre", _F32, (T, n), dev)
    _require(proj, "proj", _BF16, (T, D_OUT), dev)
    _require(inv_rms, "inv_rms", _F32, (T,), dev)
    _require(grad_layer_input, "grad_layer_input", _BF16, (T, C), dev)
    if grad_h_post is not None:
        _require(grad_h_post, "grad_h_post", _F32, (T, n), dev)
    if grad_H is not None:
        _require(grad_H, "grad_H_merged", _F32, (T, n, n), dev)
    if grad_x_in is not None:
        _require(grad_x_in, "grad_x_in", _BF16, (T, n, C), dev)
    gx = torch.empty((T, n, C), device=dev, dtype=_BF16)
    gW = torch.empty((D_OUT, n * C), device=dev, dtype=_BF16)
    ga = [torch.empty((1,), device=dev, dtype=alpha_pre.dtype) for _ in range(3)]
    gb = torch.empty((D_OUT,), device=dev, dtype=alpha_pre.dtype)
    lib = _abi.load()
    ws = torch.empty((max(int(lib.fmhc_premap_bwd_workspace_bytes(T, C)), 16),), device=dev, dtype=torch.uint8)
    with _OnDevice(dev):
        st = lib.fmhc_premap_bwd_pack8(
            x_codes.data_ptr(), x_scales.data_ptr(), W.data_ptr(), alpha_pre.data_ptr(), alpha_post.data_ptr(),
            alpha_res.data_ptr(), bias.data_ptr(), perm.data_ptr(), pdt, h_pre.data_ptr(), proj.data_ptr(),
            inv_rms.data_ptr(), grad_layer_input.data_ptr(), _ptr_or_none(grad_h_post), _ptr_or_none(grad_H),
            _ptr_or_none(grad_x_in), gx.data_ptr(), gW.data_ptr(), ga[0].data_ptr(), ga[1].data_ptr(),
            ga[2].data_ptr(), gb.data_ptr(), ws.data_ptr(), ws.numel(), T, C, n, _abi.stream_of(x_codes))
    _abi.check(st, "premap_bwd_pack8")
    return gx, gW, ga[0], ga[1], ga[2], gb


# ---------------------------------------------------------------------------
# Layer norm


def _norm_params(weight, bias, dtype: torch.dtype, C: int, dev) -> torch.dtype:
    """Check the norm's weight and bias (either may be None) and return their dtype."""
    first = weight if weight is not None else bias
    if first is None:
        return _F32
    pdt = first.dtype
    if pdt is not _F32 and pdt is not dtype:
        raise TypeError(f"weight and bias must be float32 or x's dtype {dtype}, got {pdt}")
    if weight is not None:
        _require(weight, "weight", pdt, (C,), dev)
    if bias is not None:
        _require(bias, "bias", pdt, (C,), dev)
    return pdt


def _param_ptr(t: torch.Tensor | None):
    if t is None:
        return None
    p = t.data_ptr()
    if not p:  # null stands for no parameter
        raise TypeError("weight and bias must have memory that the kernels can read (not a wrapper subclass's)")
    return p


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
                   stats: bool = True, packed: bool = False):
    """(y, mean, rstd, codes, scales) of x (..., C): y in x's dtype, mean and rstd
    (...,) fp32 (None without stats), codes and scales pack8's of x (None unless
    packed)."""
    dev = _device_of(x)
    mean = torch.empty(x.shape[:-1], device=dev, dtype=_F32) if stats else None
    rstd = torch.empty(x.shape[:-1], device=dev, dtype=_F32) if stats else None
    y, q, s, _pdt = _layer_norm_fwd(x, weight, bias, eps, dev, _ptr_or_none(mean), _ptr_or_none(rstd), packed)
    return y, mean, rstd, q, s


def layer_norm_fwd_joint(x, weight, bias, eps: float, packed: bool):
    """(y, stats, codes, scales, the parameters' dtype) of layer_norm_fwd, with mean
    and rstd the halves of stats (an allocation less, where the host is the bound)."""
    dev = _device_of(x)
    T = _rows(x, "x")[0]
    stats = x.new_empty((2 * T,), dtype=_F32)
    mean = stats.data_ptr()
    y, q, s, pdt = _layer_norm_fwd(x, weight, bias, eps, dev, mean, mean + 4 * T, packed)
    return y, stats, q, s, pdt


def _layer_norm_fwd(x, weight, bias, eps, dev, mean, rstd, packed):
    code = _dtype_code(x.dtype, "x")
    T, C = _rows(x, "x")
    pdt = _norm_params(weight, bias, x.dtype, C, dev)
    y = torch.empty_like(x)
    q, s = empty_packed(x) if packed else (None, None)
    _launch("layer_norm_fwd", dev, _abi.load().fmhc_layer_norm_fwd, x.data_ptr(), _param_ptr(weight),
            _param_ptr(bias), y.data_ptr(), mean, rstd, _ptr_or_none(q), _ptr_or_none(s), code, DTYPES[pdt], T, C, eps,
            _abi.stream_of(x))
    return y, q, s, pdt


def layer_norm_bwd(grad_y: torch.Tensor, x: torch.Tensor | None, codes: torch.Tensor | None,
                   scales: torch.Tensor | None, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None,
                   param_dtype: torch.dtype, need_weight: bool = True, need_bias: bool = True,
                   grad_x_in: torch.Tensor | None = None):
    """(grad_x, grad_weight, grad_bias) of layer_norm_fwd, from x or from its codes
    and scales; a parameter's gradient is in param_dtype, None where not needed.
    grad_x_in: a gradient of x from elsewhere, added to grad_x."""
    dev = _device_of(grad_y)
    code = _dtype_code(grad_y.dtype, "grad_y")
    T, C = _rows(grad_y, "grad_y")
    if (x is None) == (codes is None):
        raise ValueError("layer_norm_bwd takes x, or its codes and scales")
    if x is not None:
        _require(x, "x", grad_y.dtype, grad_y.shape, dev)
    else:
        _require_packed(codes, scales, "x", grad_y.shape, dev)
    _require(mean, "mean", _F32, grad_y.shape[:-1], dev)
    _require(rstd, "rstd", _F32, grad_y.shape[:-1], dev)
    if param_dtype is not _F32 and param_dtype is not grad_y.dtype:
        raise TypeError(f"param_dtype must be float32 or grad_y's dtype {grad_y.dtype}, got {param_dtype}")
    if weight is not None:
        _require(weight, "weight", param_dtype, (C,), dev)
    if grad_x_in is not None:
        _require(grad_x_in, "grad_x_in", grad_y.dtype, grad_y.shape, dev)
    return _layer_norm_bwd(grad_y, x, codes, scales, mean.data_ptr(), rstd.data_ptr(), weight, param_dtype, need_weight,
                           need_bias, grad_x_in)


def layer_norm_bwd_joint(grad_y, x, codes, scales, stats, weight, param_dtype, need_weight, need_bias, grad_x_in=None):
    """layer_norm_bwd for operands that need no checks: what layer_norm_fwd_joint
    took and gave, and autograd's gradients, contiguous."""
    mean = stats.data_ptr()
    return _layer_norm_bwd(grad_y, x, codes, scales, mean, mean + 2 * stats.numel(), weight, param_dtype, need_weight,
                           need_bias, grad_x_in)


def _layer_norm_bwd(grad_y, x, codes, scales, mean, rstd, weight, param_dtype, need_weight, need_bias, grad_x_in):
    dev = grad_y.device
    code = DTYPES[grad_y.dtype]
    C = grad_y.shape[-1]
    T = grad_y.numel() // C
    gx = torch.empty_like(grad_y)
    gw = grad_y.new_empty((C,), dtype=param_dtype) if need_weight else None
    gb = grad_y.new_empty((C,), dtype=param_dtype) if need_bias else None
    lib = _abi.load()
    ws_bytes = lib.fmhc_layer_norm_bwd_workspace_bytes(T, C) if need_weight or need_bias else 0
    ws = _workspace(ws_bytes, dev)
    _launch("layer_norm_bwd", dev, lib.fmhc_layer_norm_bwd, grad_y.data_ptr(), _ptr_or_none(x), _ptr_or_none(codes),
            _ptr_or_none(scales), mean, rstd, _param_ptr(weight), _ptr_or_none(grad_x_in), gx.data_ptr(),
            _ptr_or_none(gw), _ptr_or_none(gb), _ptr_or_none(ws), ws_bytes, code, DTYPES[param_dtype], T, C,
            _abi.stream_of(grad_y))
    return gx, gw, gb


# ---------------------------------------------------------------------------
# RMS norm


def _live_ptr(t: torch.Tensor | None, name: str):
    """The address of a tensor that is added; None, which the kernels take as nothing to add, only for None
    or where there are no elements."""
    if t is None:
        return None
    p = t.data_ptr()
    if not p and t.numel():
        raise TypeError(f"{name} has no memory that the kernels can read")
    return p


def _sum_like(x, residual, dev):
    """The tensor for x + residual (None without a residual)."""
    if residual is None:
        return None
    _require(residual, "residual", x.dtype, x.shape, dev)
    return torch.empty_like(x)


def rms_norm_fwd(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float,
                 stats: bool = True):
    """(y, sum, rstd) of x (..., C): y in x's dtype, sum = x + residual (None without
    one), rstd (...,) fp32 (None without stats)."""
    dev = _device_of(x)
    code = _dtype_code(x.dtype, "x")
    T, C = _rows(x, "x")
    pdt = _norm_params(weight, None, x.dtype, C, dev)
    total = _sum_like(x, residual, dev)
    y = torch.empty_like(x)
    rstd = x.new_empty(x.shape[:-1], dtype=_F32) if stats else None
    _launch("rms_norm_fwd", dev, _abi.load().fmhc_rms_norm_fwd, x.data_ptr(), _live_ptr(residual, "residual"),
            _param_ptr(weight), y.data_ptr(), _ptr_or_none(total), _ptr_or_none(rstd), code, DTYPES[pdt], T, C, eps,
            _abi.stream_of(x))
    return y, total, rstd


def rms_norm_bwd(grad_y: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None,
                 param_dtype: torch.dtype, need_weight: bool = True, grad_x_in: torch.Tensor | None = None):
    """(grad_x, grad_weight) of rms_norm_fwd, x its x or its sum; grad_weight is in
    param_dtype, None where not needed.  grad_x_in: a gradient of x from elsewhere,
    added to grad_x."""
    dev = _device_of(grad_y)
    code = _dtype_code(grad_y.dtype, "grad_y")
    T, C = _rows(grad_y, "grad_y")
    _require(x, "x", grad_y.dtype, grad_y.shape, dev)
    _require(rstd, "rstd", _F32, grad_y.shape[:-1], dev)
    if param_dtype is not _F32 and param_dtype is not grad_y.dtype:
        raise TypeError(f"param_dtype must be float32 or grad_y's dtype {grad_y.dtype}, got {param_dtype}")
    if weight is not None:
        _require(weight, "weight", param_dtype, (C,), dev)
    if grad_x_in is not None:
        _require(grad_x_in, "grad_x_in", grad_y.dtype, grad_y.shape, dev)
    gx = torch.empty_like(grad_y)
    gw = grad_y.new_empty((C,), dtype=param_dtype) if need_weight else None
    lib = _abi.load()
    ws_bytes = lib.fmhc_rms_norm_bwd_workspace_bytes(T, C) if need_weight else 0
    ws = _workspace(ws_bytes, dev)
    _launch("rms_norm_bwd", dev, lib.fmhc_rms_norm_bwd, grad_y.data_ptr(), x.data_ptr(), rstd.data_ptr(),
            _param_ptr(weight), _live_ptr(grad_x_in, "grad_x_in"), gx.data_ptr(), _ptr_or_none(gw), _ptr_or_none(ws),
            ws_bytes, code, DTYPES[param_dtype], T, C, _abi.stream_of(grad_y))
    return gx, gw


# ---------------------------------------------------------------------------
# Rows in 8 bits (the format: include/flash_mhc_hip.h)

ROW_PITCH = 16  # rows of codes begin at multiples of this many bytes
MOST_PITCH = 1 << 22
MOST_K = (1 << 17) - 1  # the integer sums stay in 32 bits
MOST_N = (1 << 22) - 1


def row_pitch(C: int) -> int:
    return (C + ROW_PITCH - 1) // ROW_PITCH * ROW_PITCH


def empty_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Unwritten (codes, scales) for x (..., C): codes in rows of row_pitch(C) bytes."""
    shape = x.shape
    C = shape[-1]
    scales = x.new_empty(shape[:-1], dtype=_F32)
    if C % ROW_PITCH == 0:
        return torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format), scales
    return x.new_empty((*shape[:-1], row_pitch(C)), dtype=torch.int8)[..., :C], scales


def pack8_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """codes (..., C) int8 and scales (...,) fp32 of the rows of x (..., C)."""
    dev = _device_of(x)
    code = _dtype_code(x.dtype, "x")
    rows, C = _rows(x, "x")
    codes, scales = empty_rows(x)
    _launch("pack8_rows", dev, _abi.load().fmhc_pack8_rows, x.data_ptr(), code, codes.data_ptr(), scales.data_ptr(),
            rows, C, row_pitch(C), _abi.stream_of(x))
    return codes, scales


def rms_norm_pack8_rows(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float):
    """(codes, scales, sum): rms_norm_fwd's y in 8 bits."""
    dev = _device_of(x)
    code = _dtype_code(x.dtype, "x")
    T, C = _rows(x, "x")
    pdt = _norm_params(weight, None, x.dtype, C, dev)
    total = _sum_like(x, residual, dev)
    codes, scales = empty_rows(x)
    _launch("rms_norm_pack8_rows", dev, _abi.load().fmhc_rms_norm_pack8_rows, x.data_ptr(), _live_ptr(residual, "residual"),
            _param_ptr(weight), codes.data_ptr(), scales.data_ptr(), _ptr_or_none(total), code, DTYPES[pdt], T, C,
            row_pitch(C), eps, _abi.stream_of(x))
    return codes, scales, total


def _code_rows(codes: torch.Tensor, name: str, dev, shape) -> tuple[torch.Tensor, int, int]:
    """(codes, rows, bytes between rows) of codes of shape (..., K) as fmhc_linear8 takes them: as
    they are, or a copy in rows of row_pitch(K) bytes."""
    if not isinstance(codes, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if codes.dtype is not torch.int8:
        raise TypeError(f"{name} must be {torch.int8}, got {codes.dtype}")
    if codes.device != dev:
        raise ValueError(f"{name} is on {codes.device}, expected {dev}")
    K = shape[-1]
    rows = codes.numel() // K
    if K % ROW_PITCH == 0 and codes.is_contiguous() and codes.data_ptr() % ROW_PITCH == 0:
        return codes, rows, K
    pitch = row_pitch(K)
    flat = codes if len(shape) == 2 else codes.reshape(rows, K)
    ld, one = flat.stride()
    if rows <= 1:
        ld = pitch
    if (rows > 0 and one == 1 and pitch <= ld <= MOST_PITCH and ld % ROW_PITCH == 0
            and flat.data_ptr() % ROW_PITCH == 0
            and flat.storage_offset() + (rows - 1) * ld + pitch <= flat.untyped_storage().nbytes()):
        return flat, rows, ld
    copy = flat.new_empty((rows, pitch))
    copy[:, :K].copy_(flat)
    return copy, rows, pitch


def linear8(codes: torch.Tensor, scales: torch.Tensor, weight_codes: torch.Tensor, weight_scales: torch.Tensor,
            bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
            dtype: torch.dtype = _BF16) -> torch.Tensor:
    """out (..., N) in dtype, of codes (..., K), scales (...,), weight_codes (N, K) and
    weight_scales (N,); bias (N,) in fp32 or dtype, residual (..., N) in dtype."""
    dev = _device_of(codes)
    code = _dtype_code(dtype, "dtype")
    shape, wshape = codes.shape, weight_codes.shape
    if len(shape) == 0 or not 1 <= shape[-1] <= MOST_K:
        raise ValueError(f"codes must have shape (..., K) with 1 <= K <= {MOST_K}, got {tuple(shape)}")
    K, lead = shape[-1], shape[:-1]
    if len(wshape) != 2 or wshape[1] != K or not 1 <= wshape[0] <= MOST_N:
        raise ValueError(f"weight_codes must have shape (N, {K}) with 1 <= N <= {MOST_N}, got {tuple(wshape)}")
    x, T, ldx = _code_rows(codes, "codes", dev, shape)
    w, N, ldw = _code_rows(weight_codes, "weight_codes", dev, wshape)
    _require(scales, "scales", _F32, lead, dev)
    _require(weight_scales, "weight_scales", _F32, (N,), dev)
    bias_code = 0
    if bias is not None:
        if bias.dtype is not _F32 and bias.dtype is not dtype:
            raise TypeError(f"bias must be float32 or dtype {dtype}, got {bias.dtype}")
        _require(bias, "bias", bias.dtype, (N,), dev)
        bias_code = DTYPES[bias.dtype]
    if residual is not None:
        _require(residual, "residual", dtype, (*lead, N), dev)
    out = codes.new_empty((*lead, N), dtype=dtype) if residual is None else torch.empty_like(residual)
    _launch("linear8", dev, _abi.load().fmhc_linear8, x.data_ptr(), ldx, scales.data_ptr(), w.data_ptr(), ldw,
            weight_scales.data_ptr(), _live_ptr(bias, "bias"), _live_ptr(residual, "residual"), out.data_ptr(), code, bias_code, T, N, K,
            _abi.stream_of(codes))
    return out
