"""GPU tests of activations kept in 8 bits: the format itself, and the kernels that write and read it.

Codes and scales are whole numbers with one right value, and a kernel that reads
codes gives the bits of the bf16 kernel on the unpacked tensor, so nearly all of
this is equality."""

from __future__ import annotations

import pytest
import torch

import flash_mhc
from flash_mhc import ops as _ops  # noqa: F401
from oracle import act8_oracle as A
from oracle import mhc_oracle as O
from parity import block_close, check_bf16, check_fp32

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
DEV = "cuda"
OPS = torch.ops.flash_mhc


def rnd(shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def streams(T, C, seed, dtype=BF16):
    x = rnd((T, 4, C), seed, dtype=dtype)
    x[::7] *= 100
    return x


def same(a, b, what=""):
    assert a.dtype == b.dtype and a.shape == b.shape, what
    a, b = a.contiguous(), b.contiguous()
    if a.is_floating_point():
        a, b = (t.view(torch.int16 if t.element_size() == 2 else torch.int32) for t in (a, b))
    assert torch.equal(a.cpu(), b.cpu()), what


# ---------------------------------------------------------------------------
# pack8 and unpack8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 4, 40), (7, 4, 100), (64, 4, 256), (13, 1001),
                                   (1, 4, 4096), (257, 65), (2, 3, 5, 96)])
def test_codes_and_values(dtype, shape):
    x = rnd(shape, 1, dtype=torch.float32)
    x = (x * 10.0 ** rnd(shape[:-1] + (1,), 2, dtype=torch.float32)).clamp(-6e4, 6e4).to(dtype)
    codes, scales = flash_mhc.pack8(x.to(DEV))
    rc, rs = A.pack8(x)
    same(codes.cpu(), rc, "codes")
    same(scales.cpu(), rs, "scales")
    for out in (torch.bfloat16, torch.float32, dtype):
        v = flash_mhc.unpack8(codes, scales, out)
        assert v.dtype is out
        assert torch.equal(v.double().cpu(), A.unpack8(rc, rs)), out  # exact
    for op_out, fn_out in zip(OPS.pack8(x.to(DEV)), (codes, scales)):
        same(op_out, fn_out)
    same(OPS.unpack8(codes, scales, dtype), flash_mhc.unpack8(codes, scales, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_borders(dtype):
    """Ties, the clamp at 127, zeros, the ends of the exponent range, Inf and NaN."""
    info = torch.finfo(dtype)
    rows = torch.zeros(12, 70, dtype=torch.float64)
    rows[1, :5] = torch.tensor([1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64], dtype=torch.float64)  # ties
    rows[2, 3] = 255 / 128  # rounds to 128, clamped
    rows[2, 4] = -255 / 128
    rows[3, :] = info.max
    rows[4, :] = -info.max
    rows[5, 0], rows[5, 1] = 2.0 ** -126, 2.0 ** -120  # the smallest unit
    rows[6, 0], rows[6, 1], rows[6, 2] = 2.0 ** -133, 2.0 ** -127, 2.0 ** -128  # subnormal: around half a unit
    rows[7, 40] = float("inf")
    rows[8, 69] = float("nan")
    rows[9, 0], rows[9, 33] = -float("inf"), 3.0
    rows[10, 64:] = 1e-3
    rows[11, 0], rows[11, 1] = 2.0 ** 127, 2.0 ** 120
    x = rows.to(dtype)
    codes, scales = flash_mhc.pack8(x.to(DEV))
    rc, rs = A.pack8(x)
    same(codes.cpu(), rc)
    same(scales.cpu(), rs)
    v = flash_mhc.unpack8(codes, scales, torch.float32).cpu()
    assert torch.equal(torch.isnan(v), torch.isnan(A.unpack8(rc, rs)))
    assert torch.isnan(v[7, 32:64]).all() and not torch.isnan(v[7, :32]).any() and not torch.isnan(v[7, 64:]).any()
    assert torch.isnan(v[8, 64:]).all() and torch.isnan(v[9, :32]).all() and v[9, 33] == 3.0
    fine = ~torch.isnan(v)
    assert torch.equal(v.double()[fine], A.unpack8(rc, rs)[fine])


def test_unaligned_and_strided():
    base = rnd((1 + 6 * 4 * 104,), 3).to(DEV)
    x = base[1:].view(6, 4, 104)  # 2 bytes off
    rc, rs = A.pack8(x)
    codes, scales = flash_mhc.pack8(x)
    same(codes.cpu(), rc)
    same(scales.cpu(), rs)
    y = rnd((6, 208, 4), 4).to(DEV).transpose(1, 2)[..., ::2]
    codes, scales = flash_mhc.pack8(y)
    same(codes.cpu(), A.pack8(y)[0])
    off = torch.empty(codes.numel() + 3, device=DEV, dtype=torch.int8)[3:].view(codes.shape)
    off.copy_(codes)
    same(flash_mhc.unpack8(off, scales), flash_mhc.unpack8(codes, scales))


def test_empty():
    codes, scales = flash_mhc.pack8(torch.empty(0, 4, 40, device=DEV, dtype=BF16))
    assert codes.shape == (0, 4, 40) and scales.shape == (0, 4, 2)
    assert flash_mhc.unpack8(codes, scales).shape == (0, 4, 40)


def test_other_stream():
    x = streams(512, 1024, 5).to(DEV)
    want = flash_mhc.pack8(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = flash_mhc.pack8(x)
        back = flash_mhc.unpack8(*got)
    torch.cuda.current_stream().wait_stream(s)
    same(got[0], want[0])
    same(back, flash_mhc.unpack8(*want))


# ---------------------------------------------------------------------------
# The post-residual mix


SIZES = [(1, 8), (1, 33), (5, 1), (3, 40), (2, 65), (17, 100), (64, 256), (9, 300), (33, 512), (10, 1000), (6, 1001),
         (257, 1024), (7, 2056), (5, 2560), (3, 4096), (2, 4100)]


def mix_inputs(T, C, seed=0):
    x, lo = streams(T, C, seed).to(DEV), rnd((T, C), seed + 1).to(DEV)
    H = rnd((T, 4, 4), seed + 2, dtype=torch.float32).to(DEV)
    hp = rnd((T, 4), seed + 3, dtype=torch.float32).to(DEV)
    return x, lo, H, hp, rnd((T, 4, C), seed + 4).to(DEV)


@pytest.mark.parametrize("T,C", SIZES)
def test_post_res(T, C):
    x, lo, H, hp, go = mix_inputs(T, C)
    out, xq, xs, lq, ls = OPS.fused_post_res_pack8(x, lo, H, hp)
    same(out, OPS.fused_post_res(x, lo, H, hp), "out")
    for t, q, s in ((x, xq, xs), (lo, lq, ls)):
        rc, rs = A.pack8(t)
        same(q.cpu(), rc, "codes")
        same(s.cpu(), rs, "scales")
    got = OPS.fused_post_res_backward_pack8(go, xq, xs, lq, ls, H, hp)
    xv, lv = flash_mhc.unpack8(xq, xs), flash_mhc.unpack8(lq, ls)
    for name, a, b in zip(("x", "lo", "H", "hp"), got, OPS.fused_post_res_backward(go, xv, lv, H, hp)):
        same(a, b, name)
    r = O.k4_bwd(go.cpu(), A.unpack8(xq, xs).float(), A.unpack8(lq, ls).float(), H.cpu(), hp.cpu())
    check_bf16("grad_x", got[0], *r["grad_x"], 4)
    check_bf16("grad_lo", got[1], *r["grad_lo"], 4)
    check_fp32("grad_H", got[2], *r["grad_H"], C)
    check_fp32("grad_hp", got[3], *r["grad_hp"], C)


def test_post_res_autograd():
    x, lo, H, hp, go = mix_inputs(20, 104)
    leaves = [t.clone().requires_grad_(True) for t in (x, lo, H, hp)]
    out, xq, xs, lq, ls = OPS.fused_post_res_pack8(*leaves)
    assert not any(t.requires_grad for t in (xq, xs, lq, ls))
    grads = torch.autograd.grad(out, leaves, go)
    for a, b in zip(grads, OPS.fused_post_res_backward_pack8(go, xq, xs, lq, ls, H, hp)):
        same(a, b)
    # Nothing of the inputs is kept.
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        OPS.fused_post_res_pack8(*leaves)
    assert all(t.dtype in (torch.int8, torch.uint8, torch.float32) for t in kept) and kept


def test_post_res_leaves_neighbours_alone():
    """Rows behind the last token and before the first stay as they were."""
    from flash_mhc import _abi

    T, C = 6, 65
    x, lo, H, hp, go = mix_inputs(T, C)
    lib = _abi.load()
    G = 3

    def guarded(n, dtype):
        t = torch.full((n + 512,), 77, device=DEV, dtype=dtype)
        return t, t[256:256 + n]

    o, ov = guarded(T * 4 * C, BF16)
    q, qv = guarded(T * 4 * C, torch.int8)
    s, sv = guarded(T * 4 * G, torch.uint8)
    lq, lqv = guarded(T * C, torch.int8)
    ls, lsv = guarded(T * G, torch.uint8)
    p = [t.data_ptr() for t in (x, lo, H, hp, ov, qv, sv, lqv, lsv)]
    assert lib.fmhc_k4_fwd_pack8(*p, T, C, 4, torch.cuda.current_stream().cuda_stream) == 0
    for t, v in ((o, ov), (q, qv), (s, sv), (lq, lqv), (ls, lsv)):
        assert bool((t[:256] == 77).all()) and bool((t[256 + v.numel():] == 77).all())
    same(ov.view(T, 4, C), OPS.fused_post_res(x, lo, H, hp))


# ---------------------------------------------------------------------------
# K1's backward and the pre-map backward


def project_inputs(T, C, seed=0):
    x = streams(T, C, seed).to(DEV)
    W = rnd((32, 4 * C), seed + 1, 0.05).to(DEV)
    proj, inv = OPS.fused_rmsnorm_project(x.view(T, 4 * C), W)
    return x, W, proj, inv, rnd((T, 32), seed + 2).to(DEV)


@pytest.mark.parametrize("T,C", SIZES + [(500, 264), (1027, 129)])
def test_project_backward(T, C):
    x, W, proj, inv, go = project_inputs(T, C)
    xq, xs = flash_mhc.pack8(x)
    gx, gW = OPS.fused_rmsnorm_project_bwd_pack8(go, xq, xs, W, proj, inv)
    assert gx.shape == (T, 4, C) and gW.shape == (32, 4 * C)
    xv = flash_mhc.unpack8(xq, xs).view(T, 4 * C)
    if C % 8 == 0:
        rx, rW = OPS.fused_rmsnorm_project_bwd(go, xv, W, proj, inv)
        same(gx.view(T, 4 * C), rx)
        same(gW, rW)
    R, S = O.k1_bwd_dx(go.cpu(), xv.cpu(), W.cpu(), proj.cpu(), inv.cpu())
    check_bf16("grad_x", gx.view(T, 4 * C), R, S, 33)
    R, S = O.k1_grad_W(go.cpu(), xv.cpu(), inv.cpu())
    check_bf16("grad_W", gW, R, S, T)


def pre_map_inputs(T, C, pdt=torch.float32, seed=0):
    x = streams(T, C, seed).to(DEV)
    W = rnd((32, 4 * C), seed + 1, 0.05).to(DEV)
    params = [torch.tensor([a], device=DEV, dtype=pdt) for a in (0.25, 0.375, 0.5)]
    params += [rnd((32,), seed + 2, 0.1, pdt).to(DEV), flash_mhc.build_permutation_matrices(4)[0].to(DEV, pdt)]
    return x, W, params


@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("T,C", SIZES + [(3000, 72), (2500, 1024), (300, 448)])
def test_pre_map_backward(T, C, sink):
    pdt = torch.float32 if T % 2 else BF16
    x, W, params = pre_map_inputs(T, C, pdt)
    outs = OPS.mhc_pre_map_pack8(x, W, *params)
    for a, b in zip(outs, OPS.mhc_pre_map(x, W, *params)):
        same(a, b)
    _li, _H, _hq, h_pre, proj, inv, _sink, xq, xs = outs
    rc, rs = A.pack8(x)
    same(xq.cpu(), rc)
    same(xs.cpu(), rs)
    g_li, g_H = rnd((T, C), 5).to(DEV), rnd((T, 4, 4), 6, dtype=torch.float32).to(DEV)
    g_hq = rnd((T, 4), 7, dtype=torch.float32).to(DEV)
    g_sink = rnd((T, 4, C), 8).to(DEV) if sink else None
    got = OPS.mhc_pre_map_backward_pack8(g_li, g_H, g_hq, None, None, g_sink, xq, xs, W, *params, h_pre, proj, inv)
    ref = OPS.mhc_pre_map_backward(g_li, g_H, g_hq, None, None, g_sink, flash_mhc.unpack8(xq, xs), W, *params, h_pre,
                                   proj, inv)
    for name, a, b in zip(("x", "W", "ap", "apo", "ar", "b"), got, ref):
        same(a, b, name)


def test_pre_map_backward_other_gradients():
    """Gradients into h_pre and proj, and none into the layer input."""
    T, C = 40, 96
    x, W, params = pre_map_inputs(T, C)
    _li, _H, _hq, h_pre, proj, inv, _sink, xq, xs = OPS.mhc_pre_map_pack8(x, W, *params)
    xv = flash_mhc.unpack8(xq, xs)
    g_hpre = rnd((T, 4), 5, dtype=torch.float32).to(DEV)
    g_proj, g_sink = rnd((T, 32), 6).to(DEV), rnd((T, 4, C), 7).to(DEV)
    for g in ((None, None, None, g_hpre, g_proj, g_sink), (None, None, None, None, g_proj, None)):
        got = OPS.mhc_pre_map_backward_pack8(*g, xq, xs, W, *params, h_pre, proj, inv)
        ref = OPS.mhc_pre_map_backward(*g, xv, W, *params, h_pre, proj, inv)
        for a, b in zip(got, ref):
            same(a, b)


def test_empty_batches():
    C = 40
    x, W, params = pre_map_inputs(0, C)
    outs = OPS.mhc_pre_map_pack8(x, W, *params)
    got = OPS.mhc_pre_map_backward_pack8(torch.empty(0, C, device=DEV, dtype=BF16), None, None, None, None, None,
                                         outs[7], outs[8], W, *params, outs[3], outs[4], outs[5])
    assert got[0].shape == (0, 4, C) and all(float(t.float().abs().sum()) == 0 for t in got[1:])
    gx, gW = OPS.fused_rmsnorm_project_bwd_pack8(torch.empty(0, 32, device=DEV, dtype=BF16), outs[7], outs[8], W,
                                                 outs[4], outs[5])
    assert gx.shape == (0, 4, C) and float(gW.float().abs().sum()) == 0


# ---------------------------------------------------------------------------
# The block


def make_block(C, seed=0, **kw):
    torch.manual_seed(seed)
    layer = torch.nn.Sequential(torch.nn.Linear(C, C, bias=False), torch.nn.GELU())
    blk = flash_mhc.MHCLiteBlock(4, C, layer, **kw).to(DEV).to(BF16)
    with torch.no_grad():
        blk.alpha_pre.fill_(0.8)
        blk.alpha_post.fill_(1.2)
        blk.alpha_res.fill_(1.7)
    return blk


def grads(blk, x, g):
    xs = x.clone().requires_grad_(True)
    out = blk(xs)
    gr = torch.autograd.grad(out, [xs, *blk.parameters()], g)
    return out.detach(), gr


@pytest.mark.parametrize("T,C", [(1, 32), (33, 40), (64, 256), (300, 100), (2048, 512)])
def test_block(T, C):
    """The forward is the 16-bit block's; the gradients are those of the ops on
    what the codes stand for, with the layer's own backward between them."""
    blk, ref = make_block(C, activation_bits=8), make_block(C)
    x, g = streams(T, C, 11).to(DEV), rnd((T, 4, C), 12).to(DEV)
    out, got = grads(blk, x, g)
    same(out, grads(ref, x, g)[0])
    args = (ref.W_all.weight.detach(), *(p.detach() for p in (ref.alpha_pre, ref.alpha_post, ref.alpha_res)),
            ref.W_all.bias.detach(), ref.perm_mat)
    li, H, hq, h_pre, proj, inv, _sink = OPS.mhc_pre_map(x, *args)
    li.requires_grad_(True)
    lo = ref.layer(li)
    xv, lv = (flash_mhc.unpack8(*flash_mhc.pack8(t.detach())) for t in (x, lo))
    gx, glo, gH, ghq = OPS.fused_post_res_backward(g, xv, lv, H, hq)
    gli, gl = torch.autograd.grad(lo, [li, ref.layer[0].weight], glo)
    rx, rW, ra, rq, rr, rb = OPS.mhc_pre_map_backward(gli, gH, ghq, None, None, gx, xv, *args, h_pre, proj, inv)
    want = {"alpha_pre": ra, "alpha_post": rq, "alpha_res": rr, "layer.0.weight": gl, "W_all.weight": rW, "W_all.bias": rb}
    same(got[0], rx, "x")
    for (name, _p), a in zip(blk.named_parameters(), got[1:]):
        same(a, want[name].view_as(a), name)


def test_block_keeps_codes():
    C, T = 128, 64
    x = streams(T, C, 1).to(DEV).requires_grad_(True)

    def kept(**kw):
        blk = make_block(C, **kw)
        blk.layer = torch.nn.Identity()
        seen = {}
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.__setitem__(t.data_ptr(), t), t)[1], lambda t: t):
            blk(x)
        own = {p.data_ptr() for p in blk.parameters()}
        return sum(t.untyped_storage().nbytes() for a, t in seen.items() if t.numel() >= T * C and a not in own)

    assert kept() == 2 * (T * 4 * C + T * C)
    assert kept(activation_bits=8) == T * 4 * C + T * C


def test_block_stack_norms_and_retain_graph():
    """Two blocks with their own norms: gradients twice from one graph, eager and through the ops."""
    C, T = 96, 130
    blks = torch.nn.Sequential(*(make_block(C, s, activation_bits=8, pre_norm=True) for s in (1, 2)))
    x, g = streams(T, C, 2).to(DEV).requires_grad_(True), rnd((T, 4, C), 3).to(DEV)
    leaves = [x, *blks.parameters()]
    out = blks(x)
    first = torch.autograd.grad(out, leaves, g, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(out, leaves, g)):
        same(a, b)
    assert len(leaves) == 1 + 2 * 8
    compiled = torch.compile(blks, fullgraph=True, backend="aot_eager")
    out_c = compiled(x)
    same(out_c, out)
    for a, b in zip(torch.autograd.grad(out_c, leaves, g), first):
        same(a, b)


@pytest.mark.parametrize("kw", [dict(activation_bits=8), dict(activation_bits=8, pre_norm=True)])
def test_block_close_to_16_bits(kw):
    """How far 8 bits move the gradients.  With x in [2^e, 2^(e + 1)) the largest of
    a group, a code is off by at most 2^(e - 7) uniformly, 2^-7 / sqrt(3) of the
    group's largest value (2-norm over elements no more than sqrt(32) times
    smaller than it, as here: normal values, largest about 2 of 32), so a gradient
    linear in one kept tensor moves by under 2^-7 of its norm times 2 / sqrt(3)
    = 0.9%, and one through both kept tensors and the coefficients' chain by a few
    times that: 4%."""
    C, T = 256, 2048
    x, g = rnd((T, 4, C), 2).to(DEV) + rnd((1, 4, C), 4).to(DEV), rnd((T, 4, C), 3).to(DEV) + rnd((1, 4, C), 5).to(DEV)
    kw16 = {**kw, "activation_bits": 16}
    _o, a = grads(make_block(C, 1, **kw), x, g)
    _o, b = grads(make_block(C, 1, **kw16), x, g)
    for p, q in zip(a, b):
        p, q = p.double(), q.double()
        assert float((p - q).norm()) <= 0.04 * float(q.norm()) + 1e-3


@pytest.mark.parametrize("pre_norm", [False, True])
def test_block_captured(pre_norm):
    """A training step captured into a graph, replayed with other work between."""
    C, T = 256, 512
    blk = make_block(C, activation_bits=8, pre_norm=pre_norm)
    x, g = streams(T, C, 4).to(DEV).requires_grad_(True), rnd((T, 4, C), 5).to(DEV)
    leaves = [x, *blk.parameters()]

    def step():
        out = blk(x)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        if k == 1:
            with torch.no_grad():
                x.copy_(streams(T, C, 9).to(DEV))
            want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            same(a, b)
        flash_mhc.pack8(torch.randn(100, 100, device=DEV))


def test_block_under_checkpoint_and_offload():
    """torch's own recomputation around the block, and hooks that move what it keeps."""
    from torch.utils.checkpoint import checkpoint

    C, T = 64, 40
    blk = make_block(C, activation_bits=8)
    x, g = streams(T, C, 4).to(DEV), rnd((T, 4, C), 5).to(DEV)
    _out, want = grads(blk, x, g)
    xs = x.clone().requires_grad_(True)
    out = checkpoint(blk, xs, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(out, [xs, *blk.parameters()], g), want):
        same(a, b)
    with torch.autograd.graph.save_on_cpu():
        out = blk(xs)
    for a, b in zip(torch.autograd.grad(out, [xs, *blk.parameters()], g), want):
        same(a, b)


def test_block_gradients_in_parts():
    """The pre-map's backward gets the streams' codes from post-res's node,
    whichever parts of the graph a backward runs."""
    C, T = 64, 40
    blk = make_block(C, activation_bits=8)
    x, g = streams(T, C, 4).to(DEV), rnd((T, 4, C), 5).to(DEV)
    seen = {}
    blk.layer.register_forward_hook(lambda m, i, o: seen.__setitem__("li", i[0]))
    aux = lambda: seen["li"].float().square().sum()
    xs = x.clone().requires_grad_(True)
    params = list(blk.parameters())
    out = blk(xs)
    whole = torch.autograd.grad(out, [xs, *params], g, retain_graph=True)
    both = torch.autograd.grad([out, aux()], [xs], [g, None], retain_graph=True)[0]
    alone = torch.autograd.grad(aux(), [xs], retain_graph=True)[0]  # a loss on the layer's input
    again = torch.autograd.grad(out, [xs, *params], g)
    for a, b in zip(whole, again):
        same(a, b)
    # The layer's gradient first, then the rest with another loss.
    out = blk(xs)
    at = [n for n, _p in blk.named_parameters()].index("layer.0.weight")
    same(torch.autograd.grad(out, [params[at]], g)[0], whole[1 + at])
    same(torch.autograd.grad(aux(), [xs], retain_graph=True)[0], alone)
    # Against the 16-bit block: codes of x alone come in, a few percent.
    ref = make_block(C)
    ref.layer.register_forward_hook(lambda m, i, o: seen.__setitem__("li", i[0]))
    out16 = ref(xs)
    for got, want in ((alone, torch.autograd.grad(aux(), [xs], retain_graph=True)[0]),
                      (both, torch.autograd.grad([out16, aux()], [xs], [g, None])[0])):
        got, want = got.double(), want.double()
        assert float((got - want).norm()) <= 0.04 * float(want.norm())
    # The output and its codes gone: refused, not wrong.
    out = blk(xs)
    del out
    with pytest.raises(RuntimeError, match="keep the output"):
        torch.autograd.grad(aux(), [xs])


def test_block_refuses_changed_streams():
    C, T = 64, 8
    blk = make_block(C, activation_bits=8)
    x = streams(T, C, 4).to(DEV)
    blk.layer.register_forward_pre_hook(lambda m, i: [x.mul_(2)] and None)
    with pytest.raises(RuntimeError, match="inplace"):
        blk(x)


def test_block_frozen_parts():
    """Frozen streams and coefficients, a trained layer; and the reverse."""
    C, T = 64, 24
    blk = make_block(C, activation_bits=8)
    x, g = streams(T, C, 4).to(DEV), rnd((T, 4, C), 5).to(DEV)
    _out, want = grads(blk, x, g)
    at = [n for n, _p in blk.named_parameters()].index("layer.0.weight")
    for p in blk.parameters():
        p.requires_grad_(False)
    w = blk.layer[0].weight.requires_grad_(True)
    blk(x).backward(g)
    same(w.grad, want[1 + at])
    w.requires_grad_(False)
    xs = x.clone().requires_grad_(True)
    blk(xs).backward(g)
    same(xs.grad, want[0])


def test_block_eval_keeps_nothing():
    blk, ref = make_block(64, activation_bits=8), make_block(64)
    x = streams(16, 64, 6).to(DEV)
    with torch.no_grad():
        same(blk(x), ref(x))


@pytest.mark.parametrize("flags", [dict(FLASH_MHC_FUSED_XGRAD="0"), dict(FLASH_MHC_FUSED_PREMAP="0")])
def test_block_other_switches(flags, monkeypatch):
    """Without the x-gradient sink, and on the paths that keep the tensors."""
    for k, v in flags.items():
        monkeypatch.setenv(k, v)
    C, T = 96, 50
    x, g = streams(T, C, 7).to(DEV), rnd((T, 4, C), 8).to(DEV)
    out, got = grads(make_block(C, activation_bits=8), x, g)
    ref, want = grads(make_block(C), x, g)
    same(out, ref)
    for a, b in zip(got, want):
        assert float((a.double() - b.double()).norm()) <= 0.06 * float(b.double().norm()) + 1e-3


def test_post_res_compiled_and_nograd():
    """The op in a compiled graph, without autograd and in inference mode."""
    T, C = 33, 96
    x, lo, H, hp, go = mix_inputs(T, C)
    leaves = [t.clone().requires_grad_(True) for t in (x, lo, H, hp)]
    f = lambda x, lo, H, hp: OPS.fused_post_res_pack8(x, lo, H, hp)[0] * 2
    want = f(*leaves)
    gw = torch.autograd.grad(want, leaves, go)
    comp = torch.compile(f, fullgraph=True, backend="aot_eager")
    out = comp(*leaves)
    same(out, want)
    for a, b in zip(torch.autograd.grad(out, leaves, go), gw):
        same(a, b)
    with torch.no_grad():
        for a, b in zip(OPS.fused_post_res_pack8(x, lo, H, hp), OPS.fused_post_res_pack8(*leaves)):
            same(a, b)
            assert not a.requires_grad
    with torch.inference_mode():
        same(OPS.fused_post_res_pack8(x, lo, H, hp)[0], OPS.fused_post_res(x, lo, H, hp))
    # Only some gradients asked for; gradients into the codes do not exist.
    some = [x, lo.clone().requires_grad_(True), H, hp]
    out, *codes = OPS.fused_post_res_pack8(*some)
    assert not any(c.requires_grad for c in codes)
    same(torch.autograd.grad(out, some[1], go)[0], OPS.fused_post_res_backward(go, x, lo, H, hp)[1])


def test_opcheck():
    """Schemas, fakes, autograd registration and tracing of the ops."""
    T, C = 5, 40
    x, lo, H, hp, go = mix_inputs(T, C)
    q, s = flash_mhc.pack8(x)
    lq, ls = flash_mhc.pack8(lo)
    xx, args, li, hpre, proj, inv = premap_state(T, C)
    xq, xs = flash_mhc.pack8(xx)
    grad = lambda *ts: [t.clone().requires_grad_(True) for t in ts]
    check = torch.library.opcheck
    check(OPS.pack8, (x,))
    check(OPS.unpack8, (q, s, BF16))
    check(OPS.fused_post_res_pack8, (x, lo, H, hp))
    check(OPS.fused_post_res_pack8_traced, tuple(grad(x, lo, H, hp)))
    check(OPS.fused_post_res_backward_pack8, (go, q, s, lq, ls, H, hp))
    check(OPS.fused_rmsnorm_project_bwd_pack8, (proj, xq, xs, args[0], proj, inv))
    check(OPS.mhc_pre_map_pack8, (*grad(xx, *args[:-1]), args[-1]), test_utils=("test_schema", "test_faketensor"))
    check(OPS.mhc_pre_map_backward_pack8, (li, None, None, None, None, None, xq, xs, *args, hpre, proj, inv))
    check(OPS.mhc_post_res_pack8, (x, torch.empty_like(x), q, s, lo, H, hp))


def premap_state(T, C):
    """x, mhc_pre_map's other arguments, and some of its outputs."""
    blk = make_block(C)
    x = streams(T, C, 5).to(DEV)
    args = (*(p.detach() for p in (blk.W_all.weight, blk.alpha_pre, blk.alpha_post, blk.alpha_res, blk.W_all.bias)),
            blk.perm_mat)
    li, _H, _hq, hpre, proj, inv, _sink = OPS.mhc_pre_map(x, *args)
    return x, args, li, hpre, proj, inv


@pytest.mark.parametrize("kw", [{}, {"pre_norm": True}])
def test_block_differentiable_once(kw):
    blk = make_block(64, activation_bits=8, **kw)
    x = streams(6, 64, 3).to(DEV).requires_grad_(True)
    (gx,) = torch.autograd.grad(blk(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.float().square().sum().backward()


@pytest.mark.parametrize("C", [2048, 2051])
def test_past_32_bits(C):
    """Over 2^32 elements: 530 copies of the same tokens have the same results."""
    n, reps = 1000, 530
    T = n * reps
    assert T * 4 * C > 1 << 32
    x, lo, H, hp, go = mix_inputs(n, C)
    xx, args, li, hpre, proj, inv = premap_state(n, C)
    many = lambda t: t.repeat(reps, *[1] * (t.dim() - 1))
    parts = [slice(0, n), slice((reps // 2) * n, (reps // 2 + 1) * n), slice(T - n, T)]

    def compare(outs, want):
        for o, w in zip(outs, want):
            for p in parts:
                same(o[p], w)

    big = many(x)
    codes = flash_mhc.pack8(big)
    want = flash_mhc.pack8(x)
    compare(codes, want)
    back = flash_mhc.unpack8(*codes)
    compare([back], [flash_mhc.unpack8(*want)])
    del back, codes
    rest = [many(t) for t in (lo, H, hp)]
    outs = OPS.fused_post_res_pack8(big, *rest)
    want = OPS.fused_post_res_pack8(x, lo, H, hp)
    compare(outs, want)
    del big
    rest, outs = rest[1:], outs[1:]
    big = many(go)
    got = OPS.fused_post_res_backward_pack8(big, *outs, *rest)
    compare(got, OPS.fused_post_res_backward_pack8(go, *want[1:], H, hp))
    del got, big
    xq, xs = flash_mhc.pack8(xx)
    got = OPS.fused_rmsnorm_project_bwd_pack8(many(proj), many(xq), many(xs), args[0], many(proj), many(inv))
    want = OPS.fused_rmsnorm_project_bwd_pack8(proj, xq, xs, args[0], proj, inv)
    compare(got[:1], want[:1])
    del got
    got = OPS.mhc_pre_map_backward_pack8(many(li), None, None, None, None, None, many(xq), many(xs), *args, many(hpre),
                                         many(proj), many(inv))
    want = OPS.mhc_pre_map_backward_pack8(li, None, None, None, None, None, xq, xs, *args, hpre, proj, inv)
    compare(got[:1], want[:1])
    del got
    torch.cuda.empty_cache()


def test_block_reduce_overhead_training():
    """Inductor with graphs: replays equal the first calls, and eager mode within the block's tolerance."""
    T, C = 256, 512
    torch._dynamo.reset()
    blk = make_block(C, activation_bits=8, pre_norm=True)
    data = [(streams(T, C, 300 + i).to(DEV), rnd((T, 4, C), 400 + i).to(DEV)) for i in range(3)]

    def step(fn, x, up):
        blk.zero_grad(set_to_none=True)
        xi = x.clone().requires_grad_(True)
        out = fn(xi)
        out.backward(up)
        return [out.detach().clone(), xi.grad.clone()] + [p.grad.clone() for p in blk.parameters()]

    eager = [step(blk, x, up) for x, up in data]
    f = torch.compile(blk, mode="reduce-overhead", fullgraph=True)
    rounds = []
    for _ in range(2):
        res = []
        for x, up in data:
            torch.compiler.cudagraph_mark_step_begin()
            res.append(step(f, x, up))
        rounds.append(res)
    for first, again, want in zip(*rounds, eager):
        for a, b in zip(again, first):
            same(a, b)
        block_close("out", again[0], want[0].float())
        block_close("grad_x", again[1], want[1].float(), rtol=5e-2, atol=1e-1)


@pytest.mark.parametrize("T,C", [(1, 1), (3, 7), (17, 8), (16, 33), (130, 100), (47, 300), (33, 1001), (64, 1024), (5, 2056)])
def test_writes_stay_inside(T, C):
    """The outputs of every kernel that reads or writes codes, and nothing beside them."""
    from flash_mhc import _abi

    held = []

    def out(shape, dtype):
        n = torch.empty(shape, dtype=dtype, device="meta").numel() * dtype.itemsize
        buf = torch.full((n + 1024,), 0xA5, dtype=torch.uint8, device=DEV)
        held.append((buf, n))
        return buf[512:512 + n].view(dtype).view(shape)

    f32, i8, u8 = torch.float32, torch.int8, torch.uint8
    lib, st, G = _abi.load(), torch.cuda.current_stream().cuda_stream, (C + 31) // 32
    P = lambda *ts: [None if t is None else t.data_ptr() for t in ts]
    x, lo, H, hp, go = mix_inputs(T, C)
    o, xq, xs, lq, ls = (out((T, 4, C), BF16), out((T, 4, C), i8), out((T, 4, G), u8), out((T, C), i8), out((T, G), u8))
    _abi.check(lib.fmhc_k4_fwd_pack8(*P(x, lo, H, hp, o, xq, xs, lq, ls), T, C, 4, st), "k4 forward")
    want = OPS.fused_post_res_pack8(x, lo, H, hp)
    for a, b in zip((o, xq, xs, lq, ls), want):
        same(a, b)
    gx, glo, gH, ghp = out((T, 4, C), BF16), out((T, C), BF16), out((T, 4, 4), f32), out((T, 4), f32)
    _abi.check(lib.fmhc_k4_bwd_pack8(*P(xq, xs, lq, ls, H, hp, go, gx, glo, gH, ghp), T, C, 4, st), "k4 backward")
    for a, b in zip((gx, glo, gH, ghp), OPS.fused_post_res_backward_pack8(go, *want[1:], H, hp)):
        same(a, b)
    xx, args, li, hpre, proj, inv = premap_state(T, C)
    q, s = flash_mhc.pack8(xx)
    gx, gW = out((T, 4, C), BF16), out((32, 4 * C), BF16)
    nbytes = lib.fmhc_k1_bwd_pack8_workspace_bytes(T, C)
    ws = out((nbytes,), u8)
    _abi.check(lib.fmhc_k1_bwd_pack8(*P(q, s, args[0], proj, proj, inv, gx, gW, ws if nbytes else None), nbytes, T, C, 4, st),
               "k1 backward")
    for a, b in zip((gx, gW), OPS.fused_rmsnorm_project_bwd_pack8(proj, q, s, args[0], proj, inv)):
        same(a, b)
    nbytes = max(lib.fmhc_premap_bwd_workspace_bytes(T, C), 16)
    for sink in (None, go):
        gx, gW, ws = out((T, 4, C), BF16), out((32, 4 * C), BF16), out((nbytes,), u8)
        ga, gb = [out((1,), BF16) for _ in range(3)], out((32,), BF16)
        _abi.check(lib.fmhc_premap_bwd_pack8(*P(q, s, *args), 1, *P(hpre, proj, inv, li, hp, H, sink, gx, gW, *ga, gb, ws),
                                             nbytes, T, C, 4, st), "pre-map backward")
        ref = OPS.mhc_pre_map_backward_pack8(li, H, hp, None, None, sink, q, s, *args, hpre, proj, inv)
        for a, b in zip((gx, gW, *ga, gb), ref):
            same(a, b.view_as(a))
    for buf, n in held:
        assert bool((buf[:512] == 0xA5).all()) and bool((buf[512 + n:] == 0xA5).all())


@pytest.mark.parametrize("kw", [dict(rmsnorm_weight=True), dict(activation_checkpointing=True),
                                dict(rmsnorm_weight=True, pre_norm=True, activation_checkpointing=True)])
def test_block_options_eager_and_compiled(kw):
    """The block's other options beside activation_bits=8: the same bits through the
    Functions and through the ops, from a strided x too."""
    T, C = 70, 96
    torch._dynamo.reset()
    blk = make_block(C, 3, activation_bits=8, **kw)
    x, g = streams(T, C, 2).to(DEV), rnd((T, 4, C), 3).to(DEV)
    out, want = grads(blk, x, g)
    compiled = torch.compile(blk, fullgraph=True, backend="aot_eager")
    for fn in (blk, compiled):
        xs = x.clone().requires_grad_(True)
        o = fn(xs)
        same(o, out)
        for a, b in zip(torch.autograd.grad(o, [xs, *blk.parameters()], g), want):
            same(a, b)
    wide = torch.empty(T, C, 4, device=DEV, dtype=BF16).copy_(x.transpose(1, 2)).transpose(1, 2).requires_grad_(True)
    assert not wide.is_contiguous()
    o = blk(wide)
    same(o, out)
    for a, b in zip(torch.autograd.grad(o, [wide, *blk.parameters()], g.transpose(1, 2).contiguous().transpose(1, 2)), want):
        same(a, b)


@pytest.mark.parametrize("T,C", SIZES)
def test_post_res_with_residual(T, C):
    """The bits of post-res of the added tensors, rows of every kind."""
    from flash_mhc import kernels as K

    x, lo, H, hp, _go = mix_inputs(T, C)
    r = rnd((T, C), 77).to(DEV)
    for a, b in zip(K.k4_fwd_pack8(x, lo, H, hp, residual=r), K.k4_fwd_pack8(x, r + lo, H, hp)):
        same(a, b)
    off = torch.empty(T * C + 1, device=DEV, dtype=BF16)[1:].view(T, C).copy_(r)  # 2 bytes off
    for a, b in zip(K.k4_fwd_pack8(x, lo, H, hp, residual=off), K.k4_fwd_pack8(x, r + lo, H, hp)):
        same(a, b)
    with pytest.raises(ValueError, match="packs x_streams"):
        K.k4_fwd_pack8(x, lo, H, hp, pack_x=False, residual=r)


class Layer(torch.nn.Module):
    """A layer with an output of another dtype, another shape, or its input itself."""

    def __init__(self, C, kind):
        super().__init__()
        self.lin, self.kind = torch.nn.Linear(C, C, bias=False), kind

    def forward(self, u):
        if self.kind == "input":
            return u
        out = self.lin(u)
        return {"wide": out.to(torch.bfloat16)[None].squeeze(0), "row": out.mean(0, keepdim=True),
                "strided": out.t().contiguous().t(), "frozen": out.detach()}[self.kind]


@pytest.mark.parametrize("kind", ["input", "wide", "row", "strided", "frozen"])
def test_block_residual_kinds(kind):
    """pre_norm in 8 bits: the residual is added in post-res where it can be, with
    the bits of PyTorch's addition (the op path)."""
    T, C = 37, 96
    torch.manual_seed(0)
    blk = flash_mhc.MHCLiteBlock(4, C, Layer(C, kind), activation_bits=8, pre_norm=True).to(DEV).to(BF16)
    x, g = streams(T, C, 2).to(DEV), rnd((T, 4, C), 3).to(DEV)
    xs = x.clone().requires_grad_(True)
    leaves = [xs, *(p for n, p in blk.named_parameters() if n.startswith(("W_all", "alpha")))]
    got = blk(xs)
    gg = torch.autograd.grad(got, leaves, g)
    torch._dynamo.reset()
    want = torch.compile(blk, fullgraph=True, backend="aot_eager")(xs)
    same(got, want)
    for a, b in zip(gg, torch.autograd.grad(want, leaves, g)):
        same(a, b)
