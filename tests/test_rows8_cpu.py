"""CPU tests of RMS norm and of layers in 8-bit integers: what they refuse, their fakes, modules and autograd.

The C entry points check their arguments on the host before any launch; nothing is launched here."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_mhc
import rows8_cpu_kernels as cpu
from flash_mhc import _abi, rows8
from flash_mhc import kernels as K
from oracle import rows8_oracle as R

BF16, F32 = torch.bfloat16, torch.float32
OPS = torch.ops.flash_mhc
NEW_OPS = ("rms_norm", "add_rms_norm", "rms_norm_backward", "pack8_rows", "rms_norm_pack8_rows",
           "add_rms_norm_pack8_rows", "linear8")
F = 4096  # a non-null address that the host-side checks never dereference


def rnd(shape, seed, scale=1.0, dtype=F32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _grad(t):
    return t.requires_grad_(True)


@pytest.mark.parametrize("name", NEW_OPS)
def test_device_kernels_only(name):
    assert torch._C._dispatch_has_kernel_for_dispatch_key(f"flash_mhc::{name}", "CUDA")
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"flash_mhc::{name}", "CPU")


def _linear8(**changes):
    a = dict(x=F, ldx=48, xs=F, w=F, ldw=48, ws=F, bias=None, res=None, out=F, dt=1, bdt=0, T=2, N=8, K=40)
    a.update(changes)
    return lambda L: L.fmhc_linear8(*a.values(), None)


@pytest.mark.parametrize(
    "call",
    [
        lambda L: L.fmhc_rms_norm_fwd(*[F] * 6, 3, 0, 2, 8, 1e-6, None),  # no such dtype
        lambda L: L.fmhc_rms_norm_fwd(*[F] * 6, 0, 1, 2, 8, 1e-6, None),  # fp32 x with a bf16 weight
        lambda L: L.fmhc_rms_norm_fwd(*[F] * 6, 1, 2, 2, 8, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, F, F, F, None, F, 1, 0, 2, 8, 1e-6, None),  # a residual without the sum
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, F, F, F, 1, 0, 2, 8, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(None, None, F, F, None, F, 1, 0, 2, 8, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, None, None, F, 1, 0, 2, 8, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, F, None, F, 1, 0, -1, 8, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, F, None, F, 1, 0, 2, 0, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, F, None, F, 1, 0, 2, (1 << 28) + 1, 1e-6, None),
        lambda L: L.fmhc_rms_norm_fwd(F, None, F, F, None, F, 1, 0, 1 << 60, 1 << 20, 1e-6, None),
        lambda L: L.fmhc_rms_norm_bwd(F, None, *[F] * 3, None, *[F] * 2, 1 << 40, 1, 0, 2, 8, None),  # no x
        lambda L: L.fmhc_rms_norm_bwd(F, F, None, F, None, *[F] * 3, 1 << 40, 1, 0, 2, 8, None),  # no rstd
        lambda L: L.fmhc_rms_norm_bwd(*[F] * 8, 1 << 40, 1, 0, 2, 8, None),  # grad_x_in is grad_x
        lambda L: L.fmhc_rms_norm_bwd(*[F] * 4, None, *[F] * 3, 8, 1, 0, 2000, 8, None),  # workspace too small
        lambda L: L.fmhc_rms_norm_bwd(*[F] * 4, None, F, F, None, 1 << 40, 1, 0, 2000, 8, None),
        lambda L: L.fmhc_rms_norm_bwd(*[F] * 4, None, F, F, F + 8, 1 << 40, 1, 0, 2000, 8, None),  # off 16 bytes
        lambda L: L.fmhc_rms_norm_bwd(*[F] * 4, None, F, F, None, 0, 1, 0, 2, 5, None),
        lambda L: L.fmhc_pack8_rows(F, 3, F, F, 2, 8, 16, None),
        lambda L: L.fmhc_pack8_rows(F, 1, F, F, 2, 8, 7, None),  # rows overlap
        lambda L: L.fmhc_pack8_rows(F, 1, F, F, 1 << 30, 8, 1 << 40, None),
        lambda L: L.fmhc_pack8_rows(F, 1, None, F, 2, 8, 16, None),
        lambda L: L.fmhc_pack8_rows(F, 1, F, None, 2, 8, 16, None),
        lambda L: L.fmhc_pack8_rows(F, 1, F, F, -2, 8, 16, None),
        lambda L: L.fmhc_rms_norm_pack8_rows(F, F, F, F, F, None, 1, 0, 2, 8, 16, 1e-6, None),
        lambda L: L.fmhc_rms_norm_pack8_rows(F, None, F, F, F, None, 1, 2, 2, 8, 16, 1e-6, None),
        lambda L: L.fmhc_rms_norm_pack8_rows(F, None, F, F, F, None, 1, 0, 2, 8, 4, 1e-6, None),
        lambda L: L.fmhc_rms_norm_pack8_rows(None, None, F, F, F, None, 1, 0, 2, 8, 16, 1e-6, None),
        _linear8(dt=3),
        _linear8(dt=0, bdt=1, bias=F),
        _linear8(T=-1),
        _linear8(T=1 << 31),
        _linear8(N=0),
        _linear8(N=1 << 22),
        _linear8(K=0),
        _linear8(K=1 << 17, ldx=1 << 17, ldw=1 << 17),  # sums past 32 bits
        _linear8(T=1 << 22, N=1 << 20),  # more outputs than 2^40
        _linear8(ldx=40),  # no multiple of 16
        _linear8(ldw=40),
        _linear8(ldx=32),  # shorter than a row
        _linear8(ldw=(1 << 22) + 16),
        _linear8(x=F + 8),
        _linear8(w=F + 1),
        _linear8(x=None),
        _linear8(w=None),
        _linear8(xs=None),
        _linear8(ws=None),
        _linear8(out=None),
    ],
)
def test_entry_points_refuse(call):
    assert call(_abi.load()) == 1


@pytest.mark.parametrize("T,C", [(4, 1024), (4, 5), (3, 20000), (2000, 1024)])
@pytest.mark.parametrize("same", ["grad_y", "x", "grad_x_in"])
def test_rms_backward_refuses_grad_x_over_its_inputs(same, T, C):
    """grad_weight's workgroups read the inputs while grad_x is stored, or afterwards."""
    L = _abi.load()
    at = dict(grad_y=F, x=2 * F, grad_x_in=None)
    gx = 4 * F
    at[same] = gx
    assert L.fmhc_rms_norm_bwd(at["grad_y"], at["x"], 3 * F, None, at["grad_x_in"], gx, 5 * F, 6 * F, 1 << 40, 1, 0, T, C,
                               None) == 1


def test_entry_points_take_empty_batches():
    L = _abi.load()
    assert L.fmhc_rms_norm_fwd(*[None] * 6, 1, 0, 0, 8, 1e-6, None) == 0
    assert L.fmhc_pack8_rows(None, 1, None, None, 0, 8, 16, None) == 0
    assert L.fmhc_rms_norm_pack8_rows(*[None] * 6, 1, 0, 0, 8, 16, 1e-6, None) == 0
    assert _linear8(T=0, x=None, out=None)(L) == 0
    assert L.fmhc_rms_norm_bwd_workspace_bytes(0, 8) == 0 and L.fmhc_rms_norm_bwd_workspace_bytes(3, 5) == 3 * 8 * 4
    # Partial sums of 512 rows at most, of very long rows fewer, none for few rows.
    ws = L.fmhc_rms_norm_bwd_workspace_bytes
    assert ws(1 << 20, 2048) == 512 * 2048 * 4 == ws(513, 2048) and ws(1 << 20, 5) == 512 * 8 * 4
    assert ws(512, 2048) == ws(1024, 1024) == ws(1, 8) == 0 and ws(1025, 1024) == 512 * 1024 * 4
    assert ws(1 << 20, 1 << 28) == 4 << 28 and ws(1 << 20, 20000) == 102 * 20000 * 4


def test_refusals():
    x = torch.zeros(4, 8, dtype=BF16)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for f in (K.pack8_rows, lambda t: K.rms_norm_fwd(t, None, None, 1e-6),
              lambda t: K.rms_norm_pack8_rows(t, None, None, 1e-6), lambda t: K.linear8(q, s, q, s)):
        with pytest.raises(ValueError, match="GPU tensor"):
            f(x)
    for f in (flash_mhc.pack8_rows, flash_mhc.rms_norm, flash_mhc.rms_norm_pack8_rows,
              lambda t: flash_mhc.linear8(q, s, q, s)):
        with pytest.raises(NotImplementedError):
            f(x)
    for f in (flash_mhc.rms_norm, flash_mhc.rms_norm_pack8_rows):
        with pytest.raises(ValueError, match="weight must have shape"):
            f(x, torch.ones(9))
        with pytest.raises(ValueError, match="C >= 1"):
            f(torch.zeros(()))
        with pytest.raises(ValueError, match="residual must have x's shape"):
            f(x, residual=x[:1])
        with pytest.raises(ValueError, match="residual must have x's shape"):
            f(x, residual=x.float())
    with pytest.raises(ValueError, match="C >= 1"):
        flash_mhc.pack8_rows(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="in_features"):
        flash_mhc.Linear8(1 << 17, 4)
    with pytest.raises(ValueError, match="out_features"):
        flash_mhc.Linear8(4, 0)
    with pytest.raises(ValueError, match=r"shape \(..., 8\)"):
        flash_mhc.Linear8(8, 4)(torch.zeros(3, 9))
    with pytest.raises(ValueError, match="pre_norm must be"):
        flash_mhc.MHCLiteBlock(4, 8, torch.nn.Linear(8, 8), pre_norm="group")
    assert flash_mhc.MHCLiteBlock(4, 8, torch.nn.Linear(8, 8), pre_norm=None).norm is None
    with pytest.raises(ValueError, match="out_features"):
        flash_mhc.Linear8(4, 1 << 22)


def _meta(shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_launchers_name_what_is_wrong(monkeypatch):
    """Shape, dtype and layout errors before the library is asked."""
    monkeypatch.setattr(K, "_device_of", lambda t: t.device)
    i8 = torch.int8
    with pytest.raises(TypeError, match="weight and bias must be float32 or x's dtype"):
        K.rms_norm_fwd(_meta((2, 8)), None, _meta((8,), torch.float16), 1e-6)
    with pytest.raises(ValueError, match="residual must have shape"):
        K.rms_norm_fwd(_meta((2, 8)), _meta((1, 8)), None, 1e-6)
    with pytest.raises(TypeError, match="residual must be torch.bfloat16"):
        K.rms_norm_pack8_rows(_meta((2, 8)), _meta((2, 8), F32), None, 1e-6)
    with pytest.raises(ValueError, match="contiguous"):
        K.pack8_rows(_meta((2, 8)).t())
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        K.pack8_rows(_meta((2, 8), torch.float64))
    with pytest.raises(ValueError, match="rstd must have shape"):
        K.rms_norm_bwd(_meta((2, 8)), _meta((2, 8)), _meta((3,), F32), None, F32)
    with pytest.raises(TypeError, match="param_dtype"):
        K.rms_norm_bwd(_meta((2, 8)), _meta((2, 8)), _meta((2,), F32), None, torch.float16)
    q, s, w, ws = _meta((2, 16), i8), _meta((2,), F32), _meta((5, 16), i8), _meta((5,), F32)
    for match, args in (("codes must be torch.int8", (_meta((2, 16)), s, w, ws)),
                        ("weight_codes must be torch.int8", (q, s, _meta((5, 16), torch.uint8), ws)),
                        (r"weight_codes must have shape \(N, 16\)", (q, s, _meta((5, 17), i8), ws)),
                        (r"weight_codes must have shape \(N, 16\)", (q, s, _meta((0, 16), i8), ws)),
                        ("1 <= N", (q, s, _meta((1 << 22, 16), i8), ws)),
                        ("scales must have shape", (q, _meta((3,), F32), w, ws)),
                        ("scales must be torch.float32", (q, _meta((2,)), w, ws)),
                        ("weight_scales must have shape", (q, s, w, _meta((4,), F32))),
                        ("bias must be float32 or dtype", (q, s, w, ws, _meta((5,), torch.float16))),
                        ("bias must have shape", (q, s, w, ws, _meta((6,)))),
                        ("residual must have shape", (q, s, w, ws, None, _meta((5, 2)))),
                        ("residual must be torch.bfloat16", (q, s, w, ws, None, _meta((2, 5), F32))),
                        ("dtype must be", (q, s, w, ws, None, None, torch.float64)),
                        ("1 <= K", (_meta((2, 1 << 17), i8), s, _meta((5, 1 << 17), i8), ws))):
        with pytest.raises((TypeError, ValueError), match=match):
            K.linear8(*args)


def test_operands_without_memory_are_not_left_out(monkeypatch):
    """A null address stands for no bias, residual or second gradient in the kernels' entry points."""
    monkeypatch.setattr(K, "_device_of", lambda t: t.device)
    monkeypatch.setattr(K, "_launch", lambda what, dev, fn, *a: None)
    monkeypatch.setattr(_abi, "stream_of", lambda t: 0)
    x, w, stat = _meta((2, 16)), _meta((16,)), _meta((2,), F32)
    q, wq, ws = _meta((2, 16), torch.int8), _meta((5, 16), torch.int8), _meta((5,), F32)
    for call in (lambda: K.rms_norm_fwd(x, x, None, 1e-6), lambda: K.rms_norm_fwd(x, None, w, 1e-6),
                 lambda: K.rms_norm_pack8_rows(x, x, None, 1e-6), lambda: K.rms_norm_bwd(x, x, stat, None, F32, False, x),
                 lambda: K.linear8(q, stat, wq, ws, _meta((5,))), lambda: K.linear8(q, stat, wq, ws, None, _meta((2, 5)))):
        with pytest.raises(TypeError, match="memory that the kernels can read"):
            call()
    for call in (lambda: K.rms_norm_fwd(x, None, None, 1e-6), lambda: K.linear8(q, stat, wq, ws),
                 lambda: K.linear8(q[:0], stat[:0], wq, ws, None, _meta((0, 5)))):
        call()


def test_codes_are_copied_only_where_rows_are_off():
    def rows(t):
        out, n, ld = K._code_rows(t, "codes", t.device, t.shape)
        assert n == t.numel() // t.shape[-1] and ld % 16 == 0 and out.data_ptr() % 16 == 0
        # What the kernel may read lies inside the storage.
        end = out.data_ptr() - out.untyped_storage().data_ptr() + (n - 1) * ld + K.row_pitch(t.shape[-1])
        assert n == 0 or end <= out.untyped_storage().nbytes()
        got = out.as_strided((n, t.shape[-1]), (ld, 1))
        assert torch.equal(got, t.reshape(n, t.shape[-1]))
        return out.untyped_storage().data_ptr() == t.untyped_storage().data_ptr()

    base = torch.arange(16 * 64, dtype=torch.int32).to(torch.int8).view(16, 64)
    assert rows(base) and rows(base[:, :40]) and rows(base[:, 16:40]) and rows(base.view(2, 8, 64)[..., :33])
    assert rows(base[::2]) and rows(base[3:4, :5])
    rows(torch.zeros(0, 33, dtype=torch.int8))
    assert not rows(base[:, 1:40]) and not rows(base.t()) and not rows(base[:, ::2]) and not rows(base[:1].expand(4, 64))
    assert not rows(base[:, :40].contiguous()) and not rows(base.as_strided((16, 40), (8, 1)))
    assert not rows(torch.zeros(15 * 48 + 33, dtype=torch.int8).as_strided((16, 33), (48, 1)))  # ends with its storage
    assert rows(torch.zeros(15 * 48 + 48, dtype=torch.int8).as_strided((16, 33), (48, 1)))


def test_fakes():
    with FakeTensorMode():
        x, r, w = torch.empty(7, 3, 40, dtype=BF16), torch.empty(7, 3, 40, dtype=BF16), torch.empty(40)
        y, rstd = OPS.rms_norm(x, w, 1e-6)
        assert y.shape == x.shape and y.dtype is BF16 and rstd.shape == (7, 3) and rstd.dtype is F32
        y, s, rstd = OPS.add_rms_norm(x, r, w, 1e-6)
        assert s.shape == x.shape and s.dtype is BF16
        g = OPS.rms_norm_backward(y, s, x, rstd, w, True)
        assert g[0].shape == x.shape and g[0].dtype is BF16 and g[1].shape == (40,) and g[1].dtype is F32
        assert OPS.rms_norm_backward(y, None, x, rstd, None, False)[1].shape == (0,)
        for out in (OPS.pack8_rows(x), OPS.rms_norm_pack8_rows(x, w, 1e-6), OPS.add_rms_norm_pack8_rows(x, r, w, 1e-6)):
            assert out[0].shape == x.shape and out[0].dtype is torch.int8 and out[0].stride() == (144, 48, 1)
            assert out[1].shape == (7, 3) and out[1].dtype is F32
        turned = torch.empty(48, 5, dtype=BF16).t()  # what comes back is dense by rows
        assert OPS.pack8_rows(turned)[0].stride() == (48, 1) and OPS.rms_norm(turned, None, 1e-6)[0].stride() == (48, 1)
        assert OPS.add_rms_norm_pack8_rows(turned, turned, None, 1e-6)[0].stride() == (48, 1)
        q, s = OPS.pack8_rows(x)
        o = OPS.linear8(q, s, torch.empty(9, 40, dtype=torch.int8), torch.empty(9), None, None, torch.float16)
        assert o.shape == (7, 3, 9) and o.dtype is torch.float16


def test_oracle_rows():
    x = torch.zeros(4, 8)
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])
    x[1] = 1e-42
    x[2, 3] = float("nan")
    x[3] = 8.0
    q, s = R.pack_rows(x)
    assert q[0, :4].tolist() == [127, 0, 2, -2] and float(s[0]) == 1.0
    assert int(q[1].abs().max()) == 0 and bool(torch.isnan(s[2])) and int(q[2].abs().max()) == 0
    assert q[3].tolist() == [127] * 8
    y = rnd((30, 50), 1)
    q, s = R.pack_rows(y)
    assert float(((q * s.unsqueeze(-1)) - y).abs().div(s.unsqueeze(-1)).max()) <= 0.5 + 1e-4
    R.check_rows(q, s, y.double(), torch.zeros_like(y).double())
    with pytest.raises(AssertionError):
        R.check_rows(q + (q < 0).to(torch.int8), s, y.double(), torch.zeros_like(y).double())
    acc = (q[:4].long() @ q[4:9].long().t()).double()
    out, err = R.linear8(q[:4], s[:4], q[4:9], s[4:9])
    assert torch.equal(out, acc * s[:4].double()[:, None] * s[4:9].double()) and bool((err < 1e-5).all())


# ---------------------------------------------------------------------------
# Modules on the CPU: the plain formulas


def test_rms_norm_module():
    norm, ref = flash_mhc.RMSNorm(24, eps=1e-5), torch.nn.RMSNorm(24, eps=1e-5)
    assert list(norm.state_dict()) == list(ref.state_dict()) == ["weight"]
    with torch.no_grad():
        norm.weight.copy_(rnd((24,), 1))
    ref.load_state_dict(norm.state_dict())
    x, r = rnd((5, 24), 2), rnd((5, 24), 3)
    assert torch.equal(norm(x), ref(x))
    y, s = norm(x, r)
    assert torch.equal(s, x + r) and torch.equal(y, ref(x + r))
    a, b = norm.with_residual(x)
    assert torch.equal(a, ref(x)) and b is x
    assert flash_mhc.RMSNorm(24, elementwise_affine=False).weight is None
    with pytest.raises(ValueError, match="residual must have x's shape"):
        norm(x, r[:1])


@pytest.mark.parametrize("K_", [40, 64])
@pytest.mark.parametrize("bias", [False, True])
def test_linear8_module(K_, bias):
    torch.manual_seed(0)
    lin = torch.nn.Linear(K_, 9, bias=bias)
    layer = flash_mhc.Linear8.from_linear(lin)
    q, s = R.pack_rows(lin.weight.detach())
    assert torch.equal(layer.weight_codes[:, :K_], q) and torch.equal(layer.weight_scales, s)
    assert layer.weight_codes.shape == (9, -(-K_ // 16) * 16) and int(layer.weight_codes[:, K_:].abs().sum()) == 0
    x = rnd((3, 5, K_), 1)
    want, err = R.linear8(*R.pack_rows(x), q, s, None if lin.bias is None else lin.bias.detach())
    assert bool(((layer(x).double() - want).abs() <= err + 2 ** -23 * want.abs()).all())
    # Scales stay fp32 where the module is cast; the bias is cast.
    cast = copy.deepcopy(layer).bfloat16()
    assert cast.weight_scales.dtype is F32 and torch.equal(cast.weight_scales, s)
    assert not bias or cast.bias.dtype is BF16
    assert cast(x.bfloat16()).dtype is BF16
    assert copy.deepcopy(layer).to("meta").bfloat16().weight_scales.dtype is F32
    empty = flash_mhc.Linear8(K_, 9, bias=bias)
    assert int(empty.weight_codes.abs().sum()) == 0
    empty.load_state_dict(layer.state_dict())
    assert torch.equal(empty(x), layer(x))
    assert not list(layer.parameters())
    bad = x.clone()
    bad[0, 0, 3] = float("inf")
    out = layer(bad)
    assert bool(torch.isnan(out[0, 0]).all()) and torch.equal(out[1:], layer(x)[1:])


@pytest.mark.parametrize("dtype", [BF16, torch.float16, F32])
def test_plain_rows_are_the_formats(dtype):
    """16-bit rows hold half their largest magnitude often: 63.5, which goes to the even 64."""
    x = rnd((512, 1024), 1, dtype=dtype)
    x[0, :4] = torch.tensor([1.7, 0.85, -0.85, 0.425])
    x[0, 4:] = 0
    for rows in (x, x.double()):
        q, s = rows8._plain_rows(rows)
        want = R.pack_rows(x)
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    assert q[0, :3].tolist() == [127, 64, -64]


def test_block_on_the_cpu():
    blk = cpu.make_block(24, dtype=F32)
    assert type(blk.norm) is flash_mhc.RMSNorm and blk.norm.eps == 1e-5
    assert type(flash_mhc.MHCLiteBlock(4, 24, torch.nn.Linear(24, 24), pre_norm="layer").norm) is flash_mhc.LayerNorm
    x = rnd((5, 4, 24), 1)
    with torch.no_grad():
        li, H, hq = blk._mhc_pre_map_pytorch(x)
        lo = li + blk.layer(torch.nn.functional.rms_norm(li, (24,), blk.norm.weight, 1e-5))
        torch.testing.assert_close(blk(x), blk._mhc_post_res_pytorch(x, lo, H, hq))


# ---------------------------------------------------------------------------
# Autograd, with stand-ins for the launchers


@pytest.fixture
def eager(monkeypatch):
    cpu.eager(monkeypatch)


def _twice(loss, leaf):
    """A gradient of the gradients raises, through all nodes and through those that lead to the leaf."""
    (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
    total = loss + g.float().square().sum()
    for f in (lambda: total.backward(retain_graph=True), lambda: torch.autograd.grad(total, leaf, retain_graph=True)):
        with pytest.raises(RuntimeError, match="once_differentiable"):
            f()


def _norms(route):
    if route == "eager":
        return flash_mhc.rms_norm
    return lambda x, w=None, eps=1e-6, residual=None: (
        OPS.rms_norm(x, w, eps)[0] if residual is None else OPS.add_rms_norm(x, residual, w, eps)[:2])


@pytest.fixture(params=["eager", "ops"])
def route(request, monkeypatch):
    if request.param == "eager":
        cpu.eager(monkeypatch)
        yield request.param
    else:
        with cpu.registered():
            yield request.param


@pytest.mark.parametrize("score", [lambda y: y.square().sum(), lambda y: (y * rnd(y.shape, 9)).sum(), lambda y: y.sum()])
def test_once(route, score):
    norm = _norms(route)
    x, r, w = _grad(rnd((5, 48), 1)), _grad(rnd((5, 48), 2)), rnd((48,), 3)
    for weight in (w, _grad(w.clone()), None):
        _twice(score(norm(x, weight)), x)
        u = x * 1.5
        _twice(score(norm(u * 1, weight)), u)
        u = x.t().contiguous() * 1.5
        _twice(score(norm(u.t(), weight)), u)
        y, s = norm(x, weight, residual=r)
        for leaf in (x, r):
            _twice(score(y) + score(s), leaf)
            _twice(score(y), leaf)
        # The sum is linear: all its derivatives.
        g, = torch.autograd.grad(s.square().sum(), x, create_graph=True)
        assert torch.equal(torch.autograd.grad(g.sum(), r)[0], torch.full_like(r, 2.0))
    wide = _grad(rnd((48, 2), 4))
    _twice(score(norm(x, wide[:, 0])), wide)
    weight = _grad(w.clone())
    _twice(score(norm(x, weight)), weight)
    _twice(score(norm(x, weight, residual=r)[0]), weight)


def test_gradients(route):
    """The formulas against autograd's own of the plain form in 64 bits."""
    norm = _norms(route)
    x, r, w, gy, gs = rnd((5, 48), 1), rnd((5, 48), 2), rnd((48,), 3), rnd((5, 48), 4), rnd((5, 48), 5)
    leaves = [_grad(t.clone()) for t in (x, r, w)]
    got = torch.autograd.grad(list(norm(leaves[0], leaves[2], 1e-6, residual=leaves[1])), leaves, [gy, gs])
    ref = [_grad(t.double().clone()) for t in (x, r, w)]
    s = ref[0] + ref[1]
    y = s * (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * ref[2]
    want = torch.autograd.grad([y, s], ref, [gy.double(), gs.double()])
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, rtol=1e-5, atol=1e-5)
    # Under a graph of the gradients the same values; a gradient that is not asked for is not computed.
    again = torch.autograd.grad(list(norm(leaves[0], leaves[2], 1e-6, residual=leaves[1])), leaves, [gy, gs],
                                create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    y, s = norm(x, _grad(w.clone()), residual=r)
    assert y.requires_grad


def test_with_residual(eager):
    norm = flash_mhc.RMSNorm(48)
    x, g = rnd((5, 48), 1), rnd((5, 48), 2)
    a, b = _grad(x.clone()), _grad(x.clone())
    y, res = norm.with_residual(a)
    assert res is not a and torch.equal(res, a)
    got = torch.autograd.grad(y * 2 + res, [a, norm.weight], g)
    want = torch.autograd.grad(norm(b) * 2 + b, [b, norm.weight], g)
    for p, q in zip(got, want):
        torch.testing.assert_close(p, q)
    norm.register_forward_hook(lambda *args: None)
    assert norm.with_residual(a)[1] is a


def test_saved_tensors_are_checked(eager, monkeypatch):
    """What a hook for saved tensors gives back goes through the launcher's checks, on its way to a GPU."""
    seen = []
    bwd = cpu.rms_norm_bwd
    monkeypatch.setattr(K, "rms_norm_bwd", lambda *a: (seen.append([t.is_contiguous() for t in a[:4]]), bwd(*a))[1])
    x, w, g = _grad(rnd((6, 5), 1)), _grad(rnd((5,), 2)), rnd((6, 5), 3)
    want = torch.autograd.grad(flash_mhc.rms_norm(x, w), [x, w], g)
    spread = lambda t: torch.stack([t, t], -1)[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), spread):
        y = flash_mhc.rms_norm(x, w)
    got = torch.autograd.grad(y, [x, w], g)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and seen[-1] == [True] * 4


def test_dual_tensors_are_refused(route):
    norm = _norms(route)
    x, w = rnd((5, 48), 1), rnd((48,), 2)
    q, s = cpu.pack8_rows(x)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        ds = fwAD.make_dual(s, torch.ones_like(s))
        calls = [lambda: norm(d, w), lambda: norm(x, w, residual=d), lambda: norm(_grad(d.clone()), w),
                 lambda: flash_mhc.pack8_rows(d) if route == "eager" else OPS.pack8_rows(d),
                 lambda: flash_mhc.rms_norm_pack8_rows(d, w) if route == "eager" else OPS.rms_norm_pack8_rows(d, w, 1e-6),
                 lambda: flash_mhc.linear8(q, ds, q, s) if route == "eager"
                 else OPS.linear8(q, ds, q, s, None, None, F32)]
        for call in calls:
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()


def test_eight_bit_operators_have_no_gradient(monkeypatch):
    """Their outputs' backward raises, through the functions and the ops, instead of losing a term."""
    cpu.eager(monkeypatch)
    with cpu.registered():
        x, w, res = _grad(rnd((5, 48), 1)), _grad(rnd((48,), 2)), _grad(rnd((5, 7), 3))
        q, s = cpu.pack8_rows(rnd((5, 48), 4))
        wq, ws = cpu.pack8_rows(rnd((7, 48), 5))
        outs = [flash_mhc.pack8_rows(x)[1], flash_mhc.rms_norm_pack8_rows(x, w)[1],
                flash_mhc.rms_norm_pack8_rows(x.detach(), None, residual=x)[2],
                flash_mhc.linear8(q, s, wq, ws, residual=res, dtype=F32), flash_mhc.linear8(q, _grad(s.clone()), wq, ws),
                flash_mhc.Linear8.from_linear(torch.nn.Linear(48, 7))(x)]
        for out in outs:
            assert out.requires_grad
            with pytest.raises(RuntimeError, match="has no gradient"):
                out.float().sum().backward()
        with torch.no_grad():
            assert not flash_mhc.Linear8.from_linear(torch.nn.Linear(48, 7))(x).requires_grad


@pytest.mark.parametrize("dtype", [torch.int32, torch.int8, torch.bool, torch.complex64])
def test_linear8_refuses_rows_of_other_types(dtype):
    """Their outputs would be cut to whole numbers, or to a real part."""
    layer = flash_mhc.Linear8.from_linear(torch.nn.Linear(48, 7))
    with pytest.raises(TypeError, match="floating-point"):
        layer(torch.ones(5, 48, dtype=dtype))


def test_linear8_off_the_kernels_has_no_gradient():
    """The plain formula's codes are constants and its scales are not: a part of a gradient, which it does not give."""
    layer = flash_mhc.Linear8.from_linear(torch.nn.Linear(48, 48))
    x = rnd((5, 48), 1)
    blocks = [flash_mhc.MHCLiteBlock(4, 48, layer, pre_norm=norm, **kw)
              for norm in ("rms", "layer", False) for kw in ({}, {"activation_checkpointing": True})]
    streams = _grad(rnd((5, 4, 48), 2))
    scaled = copy.deepcopy(layer)
    scaled.weight_scales.requires_grad_(True)
    for f in (lambda: layer(_grad(x.clone())).sum().backward(), lambda: layer(_grad(x.double())).sum().backward(),
              lambda: torch.compile(layer, backend="aot_eager")(_grad(x.clone())).sum().backward(),
              lambda: torch.func.grad(lambda t: layer(t).sum())(x), lambda: scaled(x).sum().backward(),
              *(lambda blk=blk: blk(streams).sum().backward() for blk in blocks)):
        with pytest.raises(RuntimeError, match="has no gradient"):
            f()
    with fwAD.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="dual tensor"):
        layer(fwAD.make_dual(x, x))
    with pytest.raises(NotImplementedError, match="dual tensor"):
        torch.func.jvp(layer, (x,), (x,))
    with torch.no_grad():
        want = layer(x)
        assert not layer(_grad(x.clone())).requires_grad
    out = layer(_grad(x.clone()))
    assert out.requires_grad and torch.equal(out, want) and not layer(x).requires_grad
    assert torch.equal(torch.func.vmap(layer)(x.view(5, 1, 48)).view(5, 48), want)


def test_opcheck():
    with cpu.registered():
        x, r, w = _grad(rnd((5, 40), 1)), _grad(rnd((5, 40), 2)), _grad(rnd((40,), 3))
        tests = ("test_schema", "test_faketensor", "test_autograd_registration")
        torch.library.opcheck(OPS.rms_norm.default, (x, w, 1e-6), test_utils=(*tests, "test_aot_dispatch_static"))
        torch.library.opcheck(OPS.rms_norm.default, (x, None, 1e-6), test_utils=tests)
        torch.library.opcheck(OPS.add_rms_norm.default, (x, r, w, 1e-6), test_utils=(*tests, "test_aot_dispatch_static"))
        d = x.detach()
        torch.library.opcheck(OPS.pack8_rows.default, (d,), test_utils=tests)
        torch.library.opcheck(OPS.rms_norm_pack8_rows.default, (d, None, 1e-6), test_utils=tests)
        torch.library.opcheck(OPS.add_rms_norm_pack8_rows.default, (d, d.clone(), None, 1e-6), test_utils=tests)
        q, s = cpu.pack8_rows(d)
        wq, ws = cpu.pack8_rows(rnd((7, 40), 5))
        torch.library.opcheck(OPS.linear8.default, (q, s, wq, ws, None, None, BF16), test_utils=tests)


def test_block_calls_what_is_put_around_its_norm_and_layer(monkeypatch):
    """Without a graph the norm's codes go to the product; a hook, another class or keyword arguments and the
    modules are called."""
    cpu.eager(monkeypatch)
    blk = cpu.make_block(32, dtype=F32)
    u = rnd((6, 32), 1)
    with torch.no_grad():
        want = blk._apply_layer(u, {})
        q, s, _t = cpu.rms_norm_pack8_rows(u, None, blk.norm.weight, blk.norm.eps)
        assert torch.equal(want, blk.layer.product(q, s, F32, residual=u))
        seen = []
        for module in (blk.norm, blk.layer):
            handle = module.register_forward_hook(lambda m, i, o: seen.append(type(m).__name__))
            out = blk._apply_layer(u, {})
            handle.remove()
            torch.testing.assert_close(out, want, rtol=0, atol=0.05)
        assert seen == ["RMSNorm", "Linear8"]

        class Twice(flash_mhc.Linear8):
            def forward(self, x):
                return super().forward(x) * 2

        plain = blk._apply_layer(u, {}) - u
        blk.layer.__class__ = Twice
        torch.testing.assert_close(blk._apply_layer(u, {}) - u, plain * 2, rtol=0, atol=0.1)
        blk.layer.__class__ = flash_mhc.Linear8
        with pytest.raises(TypeError):
            blk._apply_layer(u, {"mask": None})
    # With a graph the layer is called as it is, and its backward raises.
    with cpu.registered():
        out = blk._apply_layer(_grad(u.clone()), {})
        with pytest.raises(RuntimeError, match="has no gradient"):
            out.sum().backward()


@pytest.mark.parametrize("dtype,kept", [(torch.float16, BF16), (BF16, torch.float16), (BF16, torch.float64),
                                        (torch.float16, F32), (F32, BF16), (BF16, BF16)])
def test_bias_of_another_type(dtype, kept):
    """The bias is added as it is: neither cut to the output's bits nor past its range before the sum."""
    layer = flash_mhc.Linear8.from_linear(torch.nn.Linear(40, 4).to(kept))
    layer.bias.copy_(torch.tensor([65000.0, 1.0 + 2.0 ** -7, 2.0 ** -12 * 1.25, 99840.0], dtype=torch.float64))
    b = layer._bias(dtype)
    assert torch.equal(b.double(), layer.bias.float().double()) and b.dtype in (dtype, F32)
    assert layer._bias(layer.bias.dtype) is layer.bias


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("x,w", [(1e33, 0.01), (1e38, 1e-6), (1e-6, 1e33), (-1e35, 1e-4), (1e-25, 1e38)])
def test_products_past_the_range_on_the_way(x, w, dtype):
    """4096 products of codes 127 times a large scale are past fp32; times the small one too they are not."""
    lin = torch.nn.Linear(4096, 3, bias=False)
    torch.nn.init.constant_(lin.weight, w)
    layer = flash_mhc.Linear8.from_linear(lin)
    out = layer(torch.full((2, 4096), x, dtype=F32).to(dtype))
    q, s = R.pack_rows(torch.full((2, 4096), x, dtype=F32).to(dtype))
    want, err = R.linear8(q, s, layer.weight_codes, layer.weight_scales)
    assert bool(torch.isfinite(out).all())
    assert bool(((out.double() - want).abs() <= err + want.abs() * torch.finfo(dtype).eps / 2).all())


def test_block_of_another_width(eager):
    """A layer that is no map of (T, C) to itself is left to the ordinary path and its error."""
    blk = cpu.make_block(32, layer=flash_mhc.Linear8(32, 16), dtype=F32)
    with torch.no_grad(), pytest.raises(RuntimeError):
        blk._apply_layer(rnd((6, 32), 1), {})


def test_exports():
    for name in ("rms_norm", "RMSNorm", "pack8_rows", "rms_norm_pack8_rows", "linear8", "Linear8"):
        assert hasattr(flash_mhc, name)
