"""Autograd around the 8-bit activation and layer norm operators, on the CPU with stand-ins for the launchers
(pack8_cpu_kernels) and on the GPU with the kernels."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import flash_mhc
import pack8_cpu_kernels as cpu

BF16, F32 = torch.bfloat16, torch.float32
OPS = torch.ops.flash_mhc


def rnd(shape, seed, scale=1.0, dtype=F32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _grad(t):
    return t.requires_grad_(True)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    """The eager Functions: on the CPU with stand-ins, on the GPU with the kernels."""
    if request.param == "cpu":
        cpu.eager(monkeypatch)
    return request.param


# ---------------------------------------------------------------------------
# Differentiable once: what a gradient's gradient would need is not computed, so
# asking for it raises, whatever the incoming gradient depends on.


def _twice(loss, leaf, match="once_differentiable"):
    """The gradient of loss + |grad loss|^2, through all nodes and through those that lead to the leaf."""
    (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
    total = loss + g.float().square().sum()
    with pytest.raises(RuntimeError, match=match):
        total.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match=match):
        torch.autograd.grad(total, leaf, retain_graph=True)


def _weights(y):
    return rnd(y.shape, 9, dtype=y.dtype).to(y.device)


SCORES = {
    "square": lambda y: y.square().sum(),
    "linear": lambda y: (y * _weights(y)).sum(),
    "sum": lambda y: y.sum(),
}


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("bits", [16, 8])
def test_layer_norm_once(dev, bits, score):
    x, w = _grad(rnd((5, 48), 1).to(dev)), rnd((48,), 2).to(dev)
    for weight in (w, _grad(w.clone()), None):
        _twice(SCORES[score](flash_mhc.layer_norm(x, weight, activation_bits=bits)), x)
        # With respect to what is no leaf, and is not kept either.
        u = x * 1.5
        _twice(SCORES[score](flash_mhc.layer_norm(u * 1, weight, activation_bits=bits)), u)
        # Kept as a copy.
        u = x.t().contiguous() * 1.5
        _twice(SCORES[score](flash_mhc.layer_norm(u.t(), weight, activation_bits=bits)), u)
    wide = _grad(rnd((48, 2), 2).to(dev))
    _twice(SCORES[score](flash_mhc.layer_norm(x, wide[:, 0], activation_bits=bits)), wide)
    # A parameter's gradient too.
    weight = _grad(w.clone())
    _twice(SCORES[score](flash_mhc.layer_norm(x, weight, activation_bits=bits)), weight)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("use", ["norm", "residual", "both"])
def test_norm_with_residual_once(dev, use, score):
    norm = flash_mhc.LayerNorm(48).to(dev)
    x = _grad(rnd((5, 48), 1).to(dev))
    if score == "linear":
        y, r = norm.with_residual((x * 1.5).t().contiguous().t())
    else:
        y, r = norm.with_residual(x * 1.5)
    used = {"norm": [y], "residual": [r], "both": [y, r]}[use]
    loss = sum(SCORES[score](t) for t in used)
    if use == "residual":  # the identity, which has all its derivatives
        plain = lambda t: (lambda s: s + torch.autograd.grad(s, x, create_graph=True)[0].square().sum())(SCORES[score](t))
        got, want = (torch.autograd.grad(plain(t), x)[0] for t in (r, x * 1.5))
        assert torch.equal(got, want)
    else:
        _twice(loss, x)


def _mixed(out, leaves):
    """grad_H with respect to x, and grad_h_post with respect to the layer output."""
    x, lo, H, hp = leaves
    gH, ghp = torch.autograd.grad(out.float().sum(), [H, hp], create_graph=True)
    for g, t in ((gH, x), (ghp, lo)):
        with pytest.raises(RuntimeError, match="once_differentiable"):
            torch.autograd.grad(g.sum(), t, retain_graph=True)


@pytest.mark.parametrize("score", SCORES)
def test_post_res_once(dev, score):
    T, C = 6, 40
    x, lo, H, hp = rnd((T, 4, C), 1, dtype=BF16), rnd((T, C), 2, dtype=BF16), rnd((T, 4, 4), 3), rnd((T, 4), 4)
    leaves = [_grad(t.to(dev)) for t in (x, lo, H, hp)]
    op = OPS.fused_post_res_pack8 if dev == "cuda" else lambda *a: flash_mhc.activation8._FusedPostResEager.apply(*a)
    for leaf in leaves:
        _twice(SCORES[score](op(*leaves)[0].float()), leaf)
    inner = [t * 1.5 for t in leaves]
    for t in inner:
        _twice(SCORES[score](op(*(t * 1 for t in inner))[0].float()), t)
    # grad_H depends on x and grad_h_post on the layer output.
    _mixed(op(*leaves)[0], leaves)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("kw", [{}, {"pre_norm": True}])
def test_block_once(dev, kw, score):
    blk = cpu.make_block(64, **kw).to(dev)
    x = _grad(rnd((6, 4, 64), 3, dtype=BF16).to(dev))
    for leaf in (x, blk.W_all.weight, blk.layer.weight):
        _twice(SCORES[score](blk._forward_triton(x).float()), leaf)
    u = x * 1.5
    _twice(SCORES[score](blk._forward_triton(u * 1).float()), u)
    # The gradient of a coefficient's bias depends on the layer's output.
    (gb,) = torch.autograd.grad(SCORES[score](blk._forward_triton(x).float()), blk.W_all.bias, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(gb.float().sum(), blk.layer.weight)


def test_gradients_with_a_graph_have_the_same_values(dev):
    """create_graph alone changes no gradient, and a graph that does not go through them is free."""
    x, w, b = rnd((5, 48), 1).to(dev), rnd((48,), 2).to(dev), rnd((48,), 3).to(dev)
    results = []
    for graph in (False, True):
        leaves = [_grad(t.clone()) for t in (x, w, b)]
        y = flash_mhc.layer_norm(*leaves, activation_bits=8)
        results.append(torch.autograd.grad(y, leaves, rnd((5, 48), 4).to(dev), create_graph=graph))
    for a, c in zip(*results):
        assert torch.equal(a, c) and not a.requires_grad and c.requires_grad
    p = _grad(torch.ones(48, device=dev))
    y = flash_mhc.layer_norm(x, _grad(w.clone())) * p
    (gp,) = torch.autograd.grad(y.square().sum(), p, create_graph=True)  # 2 p sum y^2, not through the norm's backward
    torch.autograd.grad(gp.sum(), p)


def test_once_under_checkpoint(dev):
    """Recomputed tensors can be unpacked once: a graph of the gradients has the same values there."""
    from torch.utils.checkpoint import checkpoint

    blk = cpu.make_block(64, pre_norm=True).to(dev)
    x, g = rnd((6, 4, 64), 3, dtype=BF16).to(dev), rnd((6, 4, 64), 4, dtype=BF16).to(dev)
    results = []
    for graph in (False, True):
        xs = _grad(x.clone())
        out = checkpoint(blk._forward_triton, xs, use_reentrant=False)
        results.append(torch.autograd.grad(out, [xs, *blk.parameters()], g, create_graph=graph))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        results[1][0].float().sum().backward()


# The same through the registered ops: called by name, under a dispatch mode, with
# tensor subclasses.


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def opdev(request):
    """The registered ops: on the CPU with stand-ins, on the GPU with the kernels."""
    if request.param == "cpu":
        with cpu.registered():
            yield request.param
    else:
        yield request.param


def premap_args(dev, C=32, T=6):
    x, W = rnd((T, 4, C), 1, dtype=BF16), rnd((32, 4 * C), 2, 0.1, BF16)
    alphas = [torch.tensor([a]) for a in (0.25, 0.375, 0.5)]
    perm = flash_mhc.build_permutation_matrices(4)[0]
    return [t.to(dev) for t in (x, W, *alphas, rnd((32,), 3, 0.1), perm)]


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("op", [OPS.layer_norm, OPS.layer_norm_pack8])
def test_layer_norm_ops_once(opdev, op, score):
    x, w = _grad(rnd((5, 48), 1).to(opdev)), rnd((48,), 2).to(opdev)
    for weight in (w, _grad(w.clone()), None):
        _twice(SCORES[score](op(x, weight, None, 1e-5)[0]), x)
        u = x * 1.5
        _twice(SCORES[score](op(u * 1, weight, None, 1e-5)[0]), u)


@pytest.mark.parametrize("score", SCORES)
def test_post_res_ops_once(opdev, score):
    T, C = 6, 40
    x, lo, H, hp = rnd((T, 4, C), 1, dtype=BF16), rnd((T, C), 2, dtype=BF16), rnd((T, 4, 4), 3), rnd((T, 4), 4)
    leaves = [_grad(t.to(opdev)) for t in (x, lo, H, hp)]
    op = OPS.fused_post_res_pack8_traced
    for leaf in leaves:
        _twice(SCORES[score](op(*leaves)[0].float()), leaf)
    inner = [t * 1.5 for t in leaves]
    for t in inner:
        _twice(SCORES[score](op(*(t * 1 for t in inner))[0].float()), t)
    _mixed(op(*leaves)[0], leaves)


@pytest.mark.parametrize("score", SCORES)
def test_block_ops_once(opdev, score):
    x, *params, perm = premap_args(opdev)
    leaves = [_grad(t) for t in (x, *params)]
    li, H, hq, _hpre, _proj, _inv, sink, codes, scales = OPS.mhc_pre_map_pack8(*leaves, perm)
    out = OPS.mhc_post_res_pack8(x, sink, codes, scales, li, H, hq)[0].float()
    for leaf in leaves[:2]:
        _twice(SCORES[score](out), leaf)


def test_backward_ops_have_no_derivative(opdev):
    """The backward ops themselves: called with inputs that require grad."""
    T, C = 6, 32
    x, W, ap, apo, ar, b, perm = premap_args(opdev)
    g, w = _grad(rnd((T, C), 5, dtype=BF16).to(opdev)), rnd((C,), 6).to(opdev)
    _y, mean, rstd, q, s = OPS.layer_norm_pack8(x[:, 0].contiguous(), w, None, 1e-5)
    outs = [OPS.layer_norm_backward(g, None, q, s, mean, rstd, w, F32, True, True)]
    li, H, hq, hpre, proj, inv, _sink, xq, xs = OPS.mhc_pre_map_pack8(x, W, ap, apo, ar, b, perm)
    lq, ls = OPS.pack8(li)
    outs.append(OPS.fused_post_res_backward_pack8(_grad(rnd((T, 4, C), 7, dtype=BF16).to(opdev)), xq, xs, lq, ls, H, hq))
    outs.append(OPS.fused_rmsnorm_project_bwd_pack8(_grad(proj.clone()), xq, xs, W, proj, inv))
    outs.append(OPS.mhc_pre_map_backward_pack8(g, None, None, None, None, None, xq, xs, W, ap, apo, ar, b, perm, hpre,
                                               proj, inv))
    for out in outs:
        for t in out:
            with pytest.raises(RuntimeError, match="once_differentiable"):
                t.float().sum().backward(retain_graph=True)


# ---------------------------------------------------------------------------
# Forward mode: there is no derivative in it, and a tangent is not dropped.


def _dual(t):
    return fwAD.make_dual(t, torch.ones_like(t))


def _refuses(call):
    with pytest.raises(NotImplementedError, match="forward.mode"):
        call()


@pytest.mark.parametrize("bits", [16, 8])
def test_layer_norm_refuses_dual_tensors(dev, bits):
    x, w, b = (rnd(s, i).to(dev) for i, s in enumerate(((5, 48), (48,), (48,))))
    norm = lambda *a: flash_mhc.layer_norm(*a, activation_bits=bits)
    with fwAD.dual_level():
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                for k in range(3):
                    args = [x, w, b]
                    args[k] = _dual(args[k])
                    _refuses(lambda: norm(*args))
                    _refuses(lambda: norm(x.clone().requires_grad_(True), args[1], _dual(b)))
                assert torch.equal(norm(x, w, b), norm(x, w, b))  # ordinary tensors within a level
        y = norm(_grad(x.clone()), w, b)
        _refuses(lambda: y.backward(_dual(torch.ones_like(y))))
    with pytest.raises(NotImplementedError, match="forward.mode"):
        torch.func.jvp(lambda t: norm(t, w, b), (x,), (x,))


def test_block_refuses_dual_tensors(dev):
    blk = cpu.make_block(32, pre_norm=True).to(dev).requires_grad_(False)
    x = rnd((6, 4, 32), 1, dtype=BF16).to(dev)
    with fwAD.dual_level():
        _refuses(lambda: blk._forward_triton(_dual(x)))


def test_ops_refuse_dual_tensors(opdev):
    T, C = 6, 32
    x, W, ap, apo, ar, b, perm = premap_args(opdev)
    params = (W, ap, apo, ar, b, perm)
    w = rnd((C,), 6).to(opdev)
    lo = x[:, 0].contiguous()
    _y, mean, rstd, q, s = OPS.layer_norm_pack8(lo, w, None, 1e-5)
    li, H, hq, hpre, proj, inv, sink, xq, xs = OPS.mhc_pre_map_pack8(x, *params)
    post_res = OPS.fused_post_res_pack8 if opdev == "cuda" else OPS.fused_post_res_pack8_traced
    with fwAD.dual_level():
        for call in (
            lambda: OPS.layer_norm(lo, _dual(w), None, 1e-5),
            lambda: OPS.layer_norm_pack8(_dual(lo), w, None, 1e-5),
            lambda: OPS.layer_norm_backward(_dual(lo), None, q, s, mean, rstd, w, F32, True, True),
            lambda: OPS.mhc_pre_map_pack8(_dual(x), *params),
            lambda: OPS.mhc_pre_map_backward_pack8(_dual(li), None, None, None, None, None, xq, xs, *params, hpre, proj, inv),
            lambda: OPS.mhc_post_res_pack8(x, sink, xq, xs, li, _dual(H), hq),
            lambda: post_res(x, _dual(li), H, hq),
            lambda: OPS.fused_post_res_backward_pack8(_dual(x), xq, xs, q, s, H, hq),
            lambda: OPS.fused_rmsnorm_project_bwd_pack8(_dual(proj), xq, xs, W, proj, inv),
        ):
            _refuses(call)
    blk = cpu.make_block(C).to(opdev).requires_grad_(False)
    with fwAD.dual_level():
        _refuses(lambda: blk._mhc_pre_map_triton(_dual(x)))
    with pytest.raises(NotImplementedError, match="forward.mode"):
        torch.func.jvp(lambda t: blk._mhc_pre_map_triton(t)[0], (x,), (x,))


# ---------------------------------------------------------------------------
# The streams changed in place between the pre-map, which packs them, and post-res,
# which mixes them: refused on the op path as in eager mode.


class Changing(torch.nn.Module):
    """A layer that is also given the streams."""

    def __init__(self, C, how=None, breaks=False):
        super().__init__()
        self.lin, self.how, self.breaks = torch.nn.Linear(C, C), how, breaks

    def forward(self, u, x=None):
        if self.how == "whole":
            x.mul_(2)
        elif self.how == "part":
            x[1:].add_(3)
        elif self.how == "item":
            x[0, 0, 0] = 3
        elif self.how == "view":
            x.view(-1).relu_()
        elif self.how == "detached":
            x.detach().zero_()
        if self.breaks:
            torch._dynamo.graph_break()
        return self.lin(u)


def _forward(blk, route):
    if route == "ops":
        return blk._forward_triton
    torch._dynamo.reset()
    return torch.compile(blk._forward_triton, backend=route, fullgraph=not blk.layer.breaks)


ROUTES = ["ops", "eager", "aot_eager", "inductor"]


@pytest.fixture(params=["1", "0"])
def op_route(request, opdev, monkeypatch):
    """The block on the ops, with the x-gradient's sink or without it."""
    monkeypatch.setattr(flash_mhc.block, "_plain_eager", lambda x: False)
    monkeypatch.setenv("FLASH_MHC_FUSED_XGRAD", request.param)
    return opdev


@pytest.mark.parametrize("route,how", [(r, "whole") for r in ROUTES] + [
    (r, how) for r in ROUTES[:3] for how in ("part", "item", "view", "detached")])
def test_block_ops_refuse_changed_streams(op_route, route, how):
    C = 32
    blk = cpu.make_block(C, layer=Changing(C, how)).to(op_route)
    x = _grad(rnd((6, 4, C), 1, dtype=BF16).to(op_route)) * 1
    with pytest.raises(Exception, match="inplace"):
        blk_out = _forward(blk, route)(x, x=x)
        torch.autograd.grad(blk_out.sum(), blk.W_all.weight)


def test_post_res_op_takes_copies_of_the_streams(opdev):
    """By name: the codes with an equal tensor that has a history of its own."""
    x, *params, perm = premap_args(opdev)
    x.add_(1)
    li, H, hq, *_o, sink, codes, scales = OPS.mhc_pre_map_pack8(_grad(x), *params, perm)
    want = OPS.mhc_post_res_pack8(x, sink, codes, scales, li, H, hq)[0]
    got = OPS.mhc_post_res_pack8(x.detach().clone(), sink, codes, scales, li, H, hq)[0]
    assert torch.equal(got, want)
    for a, b in zip(*(torch.autograd.grad(t.float().sum(), [x, H], retain_graph=True) for t in (got, want))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("breaks", [False, True])
@pytest.mark.parametrize("route", ROUTES)
def test_block_ops_take_streams_changed_before(op_route, route, breaks):
    """No version but the one between pre-map and post-res counts: buffers filled
    anew for every step, stacks of blocks, layers that break the graph.  (Inductor
    rounds the layer's bf16 intermediates at other places, 2^-8 each, and a
    weight's gradient is a sum of such terms, within 2^-6 of its largest.)"""
    C, T = 32, 6
    blks = [cpu.make_block(C, s, layer=Changing(C, breaks=breaks)).to(op_route) for s in (1, 2)]
    fns = [_forward(b, route) for b in blks]
    buf = torch.zeros(T, 4, C, dtype=BF16, device=op_route)
    for step in range(3):
        buf.copy_(rnd((T, 4, C), step, dtype=BF16))
        y = fns[0](buf)
        y = fns[1](y + 0)
        got = torch.autograd.grad(y.float().square().sum(), [p for b in blks for p in b.parameters()])
        want = blks[1]._forward_triton(blks[0]._forward_triton(buf.clone()))
        want = torch.autograd.grad(want.float().square().sum(), [p for b in blks for p in b.parameters()])
        for a, b in zip(got, want):
            assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=2 ** -6 * float(b.abs().max()))
        buf.add_(1)


# ---------------------------------------------------------------------------
# What a block with pre_norm calls is its norm, whatever was put around it.


class _CallsTwice(flash_mhc.LayerNorm):
    def __call__(self, x):
        return super().__call__(x) * 2


class _Wrapper(torch.nn.Module):
    """Attributes are those of the wrapped module, as offloading and sharding wrappers have it."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            return getattr(super().__getattr__("inner"), name)

    def forward(self, x):
        return self.inner(x) * 2


def _instance_forward(norm):
    plain = norm.forward
    norm.forward = lambda x: plain(x) * 2
    return norm


def _instance_call(norm):
    plain = norm._call_impl
    norm._call_impl = lambda x: plain(x) * 2
    return norm


def _subclass(norm):
    norm.__class__ = _CallsTwice
    return norm


def _hook(norm):
    norm.register_forward_hook(lambda m, a, out: out * 2)
    return norm


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("change", [_instance_forward, _instance_call, _subclass, _hook, _Wrapper])
def test_block_calls_its_norm(dev, change, bits):
    """A norm that gives twice its output: the same as a layer that takes twice its input, in training too."""
    C = 32
    layer = torch.nn.Linear(C, C, bias=False)
    blk = cpu.make_block(C, layer=layer, pre_norm=True).to(dev)
    blk.activation_bits = blk.norm.activation_bits = bits
    if dev == "cpu" and bits == 16:
        pytest.skip("the 16-bit block has no stand-ins")
    x, g = rnd((6, 4, C), 1, dtype=BF16).to(dev), rnd((6, 4, C), 2, dtype=BF16).to(dev)

    def step():
        xs = _grad(x.clone())
        out = blk._forward_triton(xs)
        return out.detach(), torch.autograd.grad(out, xs, g)[0]

    once = step()
    blk.norm = change(blk.norm)
    changed = step()
    with torch.no_grad():
        layer.weight.mul_(0.5)  # exact
    again = step()
    for a, b in zip(again, once):
        assert torch.equal(a, b)
    assert not torch.equal(changed[0], once[0]) and not torch.equal(changed[1], once[1])


def test_hooked():
    norm = flash_mhc.LayerNorm(8)
    assert not norm._hooked()
    norm.compile(backend="eager")
    assert norm._hooked()


# ---------------------------------------------------------------------------
# The streams' codes go from post-res to the pre-map's backward.


def _li_loss(blk, seen):
    blk.layer.register_forward_hook(lambda m, i, o: seen.__setitem__("li", i[0]))


@pytest.mark.parametrize("way", ["whole", "input alone"])
def test_codes_on_another_stream(monkeypatch, way):
    """The codes are made on post-res's stream and read on the pre-map's: with stand-ins that count where they are."""
    cpu.eager(monkeypatch)
    a8 = flash_mhc.activation8
    now, borrowed = [1], []
    monkeypatch.setattr(a8, "_stream_of", lambda t: now[0])
    monkeypatch.setattr(a8, "_borrow", lambda tensors, stream: borrowed.append((len(tensors), stream)))
    blk, seen = cpu.make_block(32), {}
    _li_loss(blk, seen)
    x = _grad(rnd((6, 4, 32), 1, dtype=BF16))
    for during, expect in ((1, []), (2, [(2, 2)])):
        handle = blk.layer.register_forward_hook(lambda m, i, o: now.__setitem__(0, during))
        now[0] = 1
        out = blk._forward_triton(x)
        handle.remove()
        now[0] = 1
        (out if way == "whole" else seen["li"]).float().sum().backward()
        assert borrowed == expect


class _Leaves(torch.nn.Module):
    """A layer that leaves another stream current."""

    def __init__(self, C, stream):
        super().__init__()
        self.lin, self.stream = torch.nn.Linear(C, C), stream

    def forward(self, u):
        if self.stream is not None:
            self.stream.wait_stream(torch.cuda.current_stream())
            torch.cuda.set_stream(self.stream)
        return self.lin(u)


@pytest.mark.gpu
def test_layer_that_leaves_another_stream_current():
    """The same gradients, and the allocator is told of the codes' second stream."""
    C, T = 256, 2048
    x, g = (rnd((T, 4, C), i, dtype=BF16).cuda() for i in (1, 2))
    home = torch.cuda.current_stream()

    def step(stream, alone):
        seen = {}
        torch.manual_seed(0)  # the layer's weights
        blk = cpu.make_block(C, layer=_Leaves(C, stream)).cuda()
        _li_loss(blk, seen)
        xs = _grad(x.clone())
        home.synchronize()
        try:
            out = blk(xs)
            torch.cuda.current_stream().synchronize()
        finally:
            torch.cuda.set_stream(home)
        loss, up = (seen["li"], g[:, 0].contiguous()) if alone else (out, g)
        leaves = [xs, blk.W_all.weight]
        got = torch.autograd.grad(loss, leaves, up)
        del out, loss, seen
        torch.cuda.synchronize()
        return got

    marked = []
    with pytest.MonkeyPatch.context() as m:
        record = torch.Tensor.record_stream
        m.setattr(torch.Tensor, "record_stream", lambda t, s: (marked.append(s), record(t, s))[1])
        for alone in (False, True):
            want = step(None, alone)
            assert not marked
            got = step(torch.cuda.Stream(), alone)
            assert marked == [home, home]
            marked.clear()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_frozen_block_frees_its_codes(dev):
    """A trained layer in a block whose streams and coefficients are frozen: once its
    backward is over no codes are left, whoever still holds the output."""
    C, T = 256, 512
    blk = cpu.make_block(C).to(dev).requires_grad_(False)
    blk.layer.requires_grad_(True)
    x, g = (rnd((T, 4, C), i, dtype=BF16).to(dev) for i in (1, 2))
    kept = []
    with pytest.MonkeyPatch.context() as m:
        init = flash_mhc.activation8._Kept.__init__
        m.setattr(flash_mhc.activation8._Kept, "__init__", lambda self, v: (kept.append(self), init(self, v))[1])
        out = blk._forward_triton(x)
    before = torch.cuda.memory_allocated() if dev == "cuda" else 0
    out.backward(g)
    assert blk.layer.weight.grad is not None and len(kept) == 1 and kept[0].codes is None
    if dev == "cuda":
        freed = before - torch.cuda.memory_allocated() + 2 * sum(p.numel() for p in blk.layer.parameters())
        assert freed >= T * 5 * C  # the codes of x and of the layer's output
    # Where a later backward may take them they stay.
    blk.requires_grad_(True)
    xs = _grad(x.clone())
    with pytest.MonkeyPatch.context() as m:
        m.setattr(flash_mhc.activation8._Kept, "__init__", lambda self, v: (kept.append(self), init(self, v))[1])
        out = blk._forward_triton(xs)
    torch.autograd.grad(out, blk.layer.weight, g)
    assert kept[1].codes is not None


# ---------------------------------------------------------------------------
# Parameters that are wrappers (sharded, quantised) have no memory of their own.


class _Held(torch.Tensor):
    """A wrapper subclass: ops run on what it holds."""

    seen: list = []

    @staticmethod
    def __new__(cls, held):
        return torch.Tensor._make_wrapper_subclass(cls, held.shape, dtype=held.dtype, device=held.device)

    def __init__(self, held):
        self.held = held

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(func)
        return func(*(a.held if isinstance(a, _Held) else a for a in args), **(kwargs or {}))


@pytest.mark.parametrize("bits", [16, 8])
def test_wrapped_parameters(opdev, monkeypatch, bits):
    if opdev == "cpu":
        cpu.eager(monkeypatch)
    x, w, b = (rnd(s, i).to(opdev) for i, s in enumerate(((5, 48), (48,), (48,))))
    want = flash_mhc.layer_norm(x, w, b)
    norm = flash_mhc.LayerNorm(48, activation_bits=bits).to(opdev)
    for args in ((x, _Held(w), b), (x, w, _Held(b))):
        _Held.seen.clear()
        assert torch.equal(flash_mhc.layer_norm(*args, activation_bits=bits), want)
        del norm.weight, norm.bias
        norm.weight, norm.bias = args[1:]
        y, _r = norm.with_residual(_grad(x.clone()))
        assert torch.equal(y, want)
        assert OPS.layer_norm.default in _Held.seen or OPS.layer_norm_pack8.default in _Held.seen


def test_launchers_refuse_parameters_without_memory(monkeypatch):
    from flash_mhc import _abi
    from flash_mhc import kernels as K

    monkeypatch.setattr(K, "_device_of", lambda t: t.device)
    monkeypatch.setattr(_abi, "stream_of", lambda t: None)
    monkeypatch.setattr(K, "_launch", lambda *args: pytest.fail("launched"))
    x, w, stat = rnd((5, 48), 1), rnd((48,), 2), torch.ones(5)
    for weight, bias in ((_Held(w), None), (w, _Held(w))):
        with pytest.raises(TypeError, match="wrapper"):
            K.layer_norm_fwd(x, weight, bias, 1e-5)
    with pytest.raises(TypeError, match="wrapper"):
        K.layer_norm_bwd(x, x, None, None, stat, stat, _Held(w), F32)


# ---------------------------------------------------------------------------
# The module's width.


@pytest.mark.parametrize("affine", [True, False])
def test_module_refuses_another_width(dev, affine):
    norm = flash_mhc.LayerNorm(48, elementwise_affine=affine).to(dev)
    assert norm(rnd((2, 3, 48), 1).to(dev)).shape == (2, 3, 48)
    for shape in ((5, 40), (48, 5), *([()] if dev == "cuda" or not affine else [])):
        x = rnd(shape, 1).to(dev)
        for call in (norm, norm.with_residual):
            for leaf in (x, _grad(x.clone())):
                with pytest.raises((ValueError, RuntimeError)):
                    call(leaf)
