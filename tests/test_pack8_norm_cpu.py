"""CPU tests of the 8-bit activation and layer norm operators: what they refuse, their fakes, and the block around them.

The C entry points check their arguments on the host before any launch; nothing
is launched here."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_mhc
from flash_mhc import _abi
from flash_mhc import kernels as K
from oracle import act8_oracle as A

BF16 = torch.bfloat16
_FAKE = 4096  # a non-null address that the host-side checks never dereference
OPS = torch.ops.flash_mhc

NEW_OPS = ("pack8", "unpack8", "fused_post_res_pack8", "fused_post_res_backward_pack8",
           "fused_rmsnorm_project_bwd_pack8", "mhc_pre_map_pack8", "mhc_pre_map_backward_pack8", "mhc_post_res_pack8",
           "layer_norm", "layer_norm_pack8", "layer_norm_backward")


@pytest.mark.parametrize("name", NEW_OPS)
def test_device_kernels_only(name):
    assert torch._C._dispatch_has_kernel_for_dispatch_key(f"flash_mhc::{name}", "CUDA")
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"flash_mhc::{name}", "CPU")


F = _FAKE


@pytest.mark.parametrize(
    "call",
    [
        lambda L: L.fmhc_pack8(F, 3, F, F, 2, 8, None),  # no such dtype
        lambda L: L.fmhc_pack8(F, 1, F, F, -1, 8, None),
        lambda L: L.fmhc_pack8(F, 1, F, F, 2, 0, None),
        lambda L: L.fmhc_pack8(F, 1, F, F, 2, (1 << 30) + 1, None),
        lambda L: L.fmhc_pack8(F, 1, F, F, 1 << 60, 1 << 20, None),  # more elements than an address
        lambda L: L.fmhc_pack8(None, 1, F, F, 2, 8, None),
        lambda L: L.fmhc_pack8(F, 1, F, None, 2, 8, None),
        lambda L: L.fmhc_unpack8(F, F, F, -1, 2, 8, None),
        lambda L: L.fmhc_unpack8(F, None, F, 1, 2, 8, None),
        lambda L: L.fmhc_k4_fwd_pack8(*[F] * 9, 2, 8, 3, None),  # n != 4
        lambda L: L.fmhc_k4_fwd_pack8(*[F] * 8, None, 2, 8, 4, None),
        lambda L: L.fmhc_k4_fwd_pack8(*[F] * 9, 2, 0, 4, None),
        lambda L: L.fmhc_k4_fwd_pack8_residual(*[F] * 10, 2, 8, 3, None),
        lambda L: L.fmhc_k4_fwd_pack8_residual(*[F] * 2, None, *[F] * 7, 2, 8, 4, None),
        lambda L: L.fmhc_k4_fwd_pack8_residual(*[F] * 6, None, *[F] * 3, 2, 8, 4, None),
        lambda L: L.fmhc_k4_bwd_pack8(*[F] * 11, -2, 8, 4, None),
        lambda L: L.fmhc_k4_bwd_pack8(F, None, *[F] * 9, 2, 8, 4, None),
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 9, 1 << 40, 2, 8, 5, None),
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 8, None, 0, 2, 8, 4, None),  # no workspace
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 9, 16, 2, 8, 4, None),  # too small a one
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 8, F + 4, 1 << 40, 2, 8, 4, None),  # off 16 bytes
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 9, 1 << 40, 2, (1 << 24) + 1, 4, None),
        lambda L: L.fmhc_k1_bwd_pack8(*[F] * 7, None, F, 1 << 40, 2, 8, 4, None),  # no grad_W
        lambda L: L.fmhc_premap_bwd_pack8(*[F] * 8, 2, *[F] * 14, 1 << 40, 8, 16, 4, None),  # param dtype
        lambda L: L.fmhc_premap_bwd_pack8(F, None, *[F] * 6, 0, *[F] * 14, 1 << 40, 8, 16, 4, None),
        lambda L: L.fmhc_premap_bwd_pack8(*[F] * 8, 0, *[F] * 14, 1 << 40, 8, (1 << 24) + 8, 4, None),
        lambda L: L.fmhc_layer_norm_fwd(*[F] * 8, 3, 0, 2, 8, 1e-5, None),
        lambda L: L.fmhc_layer_norm_fwd(*[F] * 8, 0, 1, 2, 8, 1e-5, None),  # fp32 x with bf16 parameters
        lambda L: L.fmhc_layer_norm_fwd(*[F] * 8, 1, 2, 2, 8, 1e-5, None),  # bf16 x with fp16 parameters
        lambda L: L.fmhc_layer_norm_fwd(*[F] * 7, None, 1, 0, 2, 8, 1e-5, None),  # codes without scales
        lambda L: L.fmhc_layer_norm_fwd(None, *[F] * 7, 1, 0, 2, 8, 1e-5, None),
        lambda L: L.fmhc_layer_norm_fwd(*[F] * 8, 1, 0, 2, 0, 1e-5, None),
        lambda L: L.fmhc_layer_norm_bwd(*[F] * 12, 1 << 40, 1, 0, 2, 8, None),  # x and codes
        lambda L: L.fmhc_layer_norm_bwd(F, None, None, None, *[F] * 8, 1 << 40, 1, 0, 2, 8, None),  # neither
        lambda L: L.fmhc_layer_norm_bwd(F, F, None, None, *[F] * 3, None, *[F] * 4, 8, 1, 0, 2, 8, None),  # workspace too small
        lambda L: L.fmhc_layer_norm_bwd(F, F, None, None, *[F] * 3, None, *[F] * 3, F + 8, 1 << 40, 1, 0, 2, 8, None),
        lambda L: L.fmhc_layer_norm_bwd(F, F, None, None, F, None, F, None, *[F] * 4, 1 << 40, 1, 0, 2, 8, None),  # no rstd
    ],
)
def test_entry_points_refuse(call):
    assert call(_abi.load()) == 1


def test_entry_points_take_empty_batches():
    L = _abi.load()
    assert L.fmhc_pack8(None, 1, None, None, 0, 8, None) == 0
    assert L.fmhc_unpack8(None, None, None, 0, 0, 8, None) == 0
    assert L.fmhc_k4_fwd_pack8(*[None] * 9, 0, 8, 4, None) == 0
    assert L.fmhc_k4_bwd_pack8(*[None] * 11, 0, 8, 4, None) == 0
    assert L.fmhc_layer_norm_fwd(*[None] * 8, 1, 0, 0, 8, 1e-5, None) == 0
    assert L.fmhc_k1_bwd_pack8_workspace_bytes(0, 8) == 0 and L.fmhc_layer_norm_bwd_workspace_bytes(0, 8) == 0


def test_launchers_refuse():
    x = torch.zeros(4, 4, 8, dtype=BF16)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.pack8(x)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.layer_norm_fwd(x, None, None, 1e-5)
    with pytest.raises(TypeError):
        K.pack8("x")
    with pytest.raises(NotImplementedError):
        OPS.pack8(x)
    with pytest.raises(NotImplementedError):
        flash_mhc.layer_norm(x)
    with pytest.raises(ValueError, match="activation_bits"):
        flash_mhc.layer_norm(x, activation_bits=4)
    with pytest.raises(ValueError, match="weight must have shape"):
        flash_mhc.layer_norm(x, torch.ones(9))
    with pytest.raises(ValueError, match="C >= 1"):
        flash_mhc.layer_norm(torch.zeros(()))


def _meta(shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_launchers_name_what_is_wrong(monkeypatch):
    """Shape, dtype and layout errors before the library is asked."""
    monkeypatch.setattr(K, "_device_of", lambda t: t.device)
    i8, u8, f32 = torch.int8, torch.uint8, torch.float32
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        K.pack8(_meta((2, 8), torch.float64))
    with pytest.raises(ValueError, match="contiguous"):
        K.pack8(_meta((2, 8)).t())
    with pytest.raises(ValueError, match="C >= 1"):
        K.pack8(_meta((2, 0)))
    with pytest.raises(TypeError, match="x_codes must be torch.int8"):
        K.unpack8(_meta((2, 40), u8), _meta((2, 2), u8))
    with pytest.raises(ValueError, match=r"x_scales must have shape \(2, 2\)"):
        K.unpack8(_meta((2, 40), i8), _meta((2, 1), u8))
    with pytest.raises(ValueError, match="n=4 only"):
        K.k4_bwd_pack8(_meta((2, 3, 8)), _meta((2, 3, 8), i8), *[None] * 5)
    with pytest.raises(ValueError, match="lo_codes must have shape"):
        K.k4_bwd_pack8(_meta((2, 4, 8)), _meta((2, 4, 8), i8), _meta((2, 4, 1), u8), _meta((3, 8), i8),
                       _meta((3, 1), u8), None, None)
    with pytest.raises(ValueError, match="W must have shape"):
        K.k1_bwd_pack8(_meta((2, 32)), _meta((2, 4, 8), i8), _meta((2, 4, 1), u8), _meta((32, 30)), None, None)
    with pytest.raises(TypeError, match="weight and bias must be float32 or x's dtype"):
        K.layer_norm_fwd(_meta((2, 8)), _meta((8,), torch.float16), None, 1e-5)
    with pytest.raises(TypeError, match="bias must be torch.float32"):
        K.layer_norm_fwd(_meta((2, 8)), _meta((8,), f32), _meta((8,)), 1e-5)
    with pytest.raises(ValueError, match="x, or its codes"):
        K.layer_norm_bwd(_meta((2, 8)), None, None, None, None, None, None, f32)
    with pytest.raises(TypeError, match="x must be torch.bfloat16"):
        K.layer_norm_bwd(_meta((2, 8)), _meta((2, 8), f32), None, None, None, None, None, f32)


def test_fakes():
    with FakeTensorMode():
        T, C = 7, 40
        x, W = torch.empty(T, 4, C, dtype=BF16), torch.empty(32, 4 * C, dtype=BF16)
        q, s = OPS.pack8(x)
        assert (q.shape, q.dtype, s.shape, s.dtype) == (x.shape, torch.int8, (T, 4, 2), torch.uint8)
        assert OPS.unpack8(q, s, torch.float32).dtype is torch.float32
        lo, H, hp = torch.empty(T, C, dtype=BF16), torch.empty(T, 4, 4), torch.empty(T, 4)
        out, xq, xs, lq, ls = OPS.fused_post_res_pack8(x, lo, H, hp)
        assert out.shape == x.shape and lq.shape == lo.shape and ls.shape == (T, 2)
        g = OPS.fused_post_res_backward_pack8(out, xq, xs, lq, ls, H, hp)
        assert [t.shape for t in g] == [x.shape, lo.shape, H.shape, hp.shape]
        assert [t.dtype for t in g] == [BF16, BF16, torch.float32, torch.float32]
        p, inv = torch.empty(T, 32, dtype=BF16), torch.empty(T)
        gx, gW = OPS.fused_rmsnorm_project_bwd_pack8(p, xq, xs, W, p, inv)
        assert gx.shape == x.shape and gW.shape == W.shape and gx.dtype is BF16
        a, b, perm = torch.empty(1), torch.empty(32), torch.empty(24, 16)
        outs = OPS.mhc_pre_map_pack8(x, W, a, a, a, b, perm)
        assert outs[0].shape == (T, C) and outs[7].shape == x.shape and outs[8].shape == (T, 4, 2)
        g = OPS.mhc_pre_map_backward_pack8(lo, H, hp, None, None, None, xq, xs, W, a, a, a, b, perm, hp, p, inv)
        assert g[0].shape == x.shape and g[0].dtype is BF16 and g[5].shape == (32,)
        out, lq, ls = OPS.mhc_post_res_pack8(x, outs[6], xq, xs, lo, H, hp)
        assert out.shape == x.shape and lq.shape == lo.shape
        y, mean, rstd = OPS.layer_norm(lo, a.new_empty(C), None, 1e-5)
        assert y.shape == lo.shape and mean.shape == rstd.shape == (T,) and mean.dtype is torch.float32
        g = OPS.layer_norm_backward(y, lo, None, None, mean, rstd, a.new_empty(C), torch.float32, True, False)
        assert g[0].shape == lo.shape and g[1].shape == (C,) and g[2].shape == (0,)


def test_oracle_format():
    """The oracle's format: ties to even, the clamp, zeros, Inf."""
    x = torch.zeros(1, 64)
    x[0, :4] = torch.tensor([1.0, 0.5 / 64, 1.5 / 64, 255 / 128])
    x[0, 32], x[0, 33] = float("inf"), 1.0
    q, s = A.pack8(x)
    assert s.tolist() == [[127, 255]]
    assert q[0, :4].tolist() == [64, 0, 2, 127] and q[0, 32:].abs().sum() == 0
    v = A.unpack8(q, s)
    assert v[0, 0] == 1.0 and torch.isnan(v[0, 32:]).all()
    y = torch.randn(50, 100, generator=torch.Generator().manual_seed(1)).to(BF16)
    v = A.unpack8(*A.pack8(y))
    assert torch.equal(v.to(BF16).double(), v)  # every value is a bf16
    # Off by at most half a unit, a 128th of the group's power of two.
    assert float((v - y.double()).abs().max()) <= 4 / 128
    q2, s2 = A.pack8(v.float())
    assert torch.equal(q2.double() * 2.0 ** (s2.repeat_interleave(32, -1)[..., :100].double() - 133), v)


def test_block_options():
    lin = lambda: torch.nn.Linear(16, 16)
    with pytest.raises(ValueError, match="activation_bits"):
        flash_mhc.MHCLiteBlock(4, 16, lin(), activation_bits=4)
    with pytest.raises(ValueError, match="activation_bits"):
        flash_mhc.LayerNorm(16, activation_bits=32)
    torch.manual_seed(0)
    plain = flash_mhc.MHCLiteBlock(4, 16, lin())
    torch.manual_seed(0)
    blk = flash_mhc.MHCLiteBlock(4, 16, lin(), activation_bits=8, pre_norm=True, norm_eps=1e-3)
    assert [n for n, _ in plain.named_parameters()] == [n for n, _ in blk.named_parameters() if not n.startswith("norm.")]
    assert {n for n, _ in blk.named_parameters()} - {n for n, _ in plain.named_parameters()} == {"norm.weight", "norm.bias"}
    assert blk.norm.eps == 1e-3 and blk.norm.activation_bits == 8
    assert torch.equal(plain.W_all.weight, blk.W_all.weight)
    # On the CPU: the plain formulation, with the norm and its residual.
    x = torch.randn(5, 4, 16)
    li, H, hq = blk._mhc_pre_map_pytorch(x)
    want = blk._mhc_post_res_pytorch(x, li + blk.layer(torch.nn.functional.layer_norm(li, (16,), eps=1e-3)), H, hq)
    torch.testing.assert_close(blk(x), want)


def test_exports():
    for name in ("pack8", "unpack8", "layer_norm", "LayerNorm"):
        assert hasattr(flash_mhc, name)
