"""Autograd around the 8-bit activation and layer norm operators, on the CPU with stand-ins for the launchers
(pack8_cpu_kernels) and on the GPU with the kernels."""

from __future__ import annotations

import pytest
import torch

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
    """loss + |grad loss|^2 differentiated; the first gradient is right to take."""
    (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match=match):
        (loss + g.float().square().sum()).backward()


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
    # A parameter's gradient too.
    weight = _grad(w.clone())
    _twice(SCORES[score](flash_mhc.layer_norm(x, weight, activation_bits=bits)), weight)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("use", ["norm", "residual", "both"])
def test_norm_with_residual_once(dev, use, score):
    norm = flash_mhc.LayerNorm(48).to(dev)
    x = _grad(rnd((5, 48), 1).to(dev))
    y, r = norm.with_residual(x * 1.5)
    used = {"norm": [y], "residual": [r], "both": [y, r]}[use]
    loss = sum(SCORES[score](t) for t in used)
    if use == "residual":  # the identity, which has all its derivatives
        plain = lambda t: (lambda s: s + torch.autograd.grad(s, x, create_graph=True)[0].square().sum())(SCORES[score](t))
        got, want = (torch.autograd.grad(plain(t), x)[0] for t in (r, x * 1.5))
        assert torch.equal(got, want)
    else:
        _twice(loss, x)


@pytest.mark.parametrize("score", SCORES)
def test_post_res_once(dev, score):
    T, C = 6, 40
    x, lo, H, hp = rnd((T, 4, C), 1, dtype=BF16), rnd((T, C), 2, dtype=BF16), rnd((T, 4, 4), 3), rnd((T, 4), 4)
    leaves = [_grad(t.to(dev)) for t in (x, lo, H, hp)]
    op = OPS.fused_post_res_pack8 if dev == "cuda" else lambda *a: flash_mhc.activation8._FusedPostResEager.apply(*a)
    for leaf in leaves:
        _twice(SCORES[score](op(*leaves)[0].float()), leaf)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("kw", [{}, {"pre_norm": True}])
def test_block_once(dev, kw, score):
    blk = cpu.make_block(64, **kw).to(dev)
    x = _grad(rnd((6, 4, 64), 3, dtype=BF16).to(dev))
    for leaf in (x, blk.W_all.weight, blk.layer.weight):
        _twice(SCORES[score](blk._forward_triton(x).float()), leaf)


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
