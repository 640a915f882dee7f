"""GPU tests of RMS norm, forward and backward, with and without the residual's addition.

Values are compared with 64-bit ones; how far they may be off is derived in
oracle/rows8_oracle.py."""

from __future__ import annotations

import pytest
import torch

import flash_mhc
from flash_mhc import _abi
from oracle import rows8_oracle as R
from oracle.act8_oracle import check

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"
EPS = 1e-6


def rnd(shape, seed, scale=1.0, mean=0.0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + mean).to(dtype)


def inputs(T, C, dtype=BF16, pdt=BF16, seed=0, residual=True):
    """x, residual, weight, the gradients of y and of the sum."""
    x = rnd((T, C), seed, 1.0, 0.25, dtype)
    x[::5] *= 50
    r = rnd((T, C), seed + 4, 2.0, 0.0, dtype).to(DEV) if residual else None
    gs = rnd((T, C), seed + 5, dtype=dtype).to(DEV) if residual else None
    return x.to(DEV), r, rnd((C,), seed + 1, 0.2, 1.0, pdt).to(DEV), rnd((T, C), seed + 3, dtype=dtype).to(DEV), gs


def run(x, r, w, gy, gs, eps=EPS):
    """[y, sum, grad_x, grad_residual, grad_w] (None for what there is not)."""
    x, r, w = (None if t is None else t.detach().clone().requires_grad_(True) for t in (x, r, w))
    out = flash_mhc.rms_norm(x, w, eps, residual=r)
    outs, grads = ([out], [gy]) if r is None else (list(out), [gy, gs])
    have = [t for t in (x, r, w) if t is not None]
    gr = iter(torch.autograd.grad(outs, have, grads))
    return [outs[0].detach(), None if r is None else outs[1].detach(),
            *[None if t is None else next(gr) for t in (x, r, w)]]


def verify(x, r, w, gy, gs, eps=EPS):
    y, total, gx, gr, gw = run(x, r, w, gy, gs, eps)
    s = x
    if r is not None:
        s = total
        assert torch.equal(total.cpu(), R.add(x, r)) and total.dtype is x.dtype
        assert torch.equal(gx, gr)
    assert y.dtype is x.dtype and gx.dtype is x.dtype and gx.shape == x.shape
    check("y", y, *R.rms_fwd(s, w, eps))
    want = R.rms_bwd(gy, s, w, eps, gs)
    check("grad_x", gx.reshape(-1, x.shape[-1]), *want["x"])
    if w is not None:
        assert gw.dtype is w.dtype
        check("grad_w", gw, *want["w"])


TYPES = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)]
SIZES = [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (40, 65), (33, 100), (70, 128), (31, 256), (17, 300), (9, 512),
         (20, 777), (6, 1000), (5, 1024), (9, 1535), (7, 2048), (3, 2560), (5, 4096), (2, 4099), (2, 6000), (2, 8192),
         (3, 12000), (2, 16384), (3, 16385), (2, 20000)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("T,C", SIZES)
def test_sizes(T, C, residual):
    verify(*inputs(T, C, residual=residual))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,pdt", TYPES)
@pytest.mark.parametrize("T,C", [(1, 40), (37, 100), (600, 264), (130, 1024), (65, 1001), (3, 4096), (2, 17000)])
def test_types(T, C, dtype, pdt, residual):
    verify(*inputs(T, C, dtype, pdt, residual=residual))


@pytest.mark.parametrize("T,C", [(5000, 32), (4097, 520), (3000, 2000), (9000, 1024), (1100, 4096), (8200, 2560)])
def test_many_rows(T, C):
    verify(*inputs(T, C, BF16, F32))


@pytest.mark.parametrize("dtype,pdt", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("T,C", [(511, 12), (512, 1032), (513, 1025), (1024, 9), (1024, 1024), (1025, 777), (1100, 8),
                                 (600, 2048), (700, 4099), (530, 16384), (515, 16390)])
def test_weight_gradient(T, C, dtype, pdt):
    """Sums of the weight's gradient on both sides of where they take a second launch."""
    verify(*inputs(T, C, dtype, pdt, residual=bool(C % 2)))


@pytest.mark.parametrize("C", [3, 24, 520, 20000])
def test_without_weight(C):
    for residual in (False, True):
        x, r, _w, gy, gs = inputs(7, C, residual=residual)
        verify(x, r, None, gy, gs)


def test_zero_and_constant_rows():
    x, r, w, gy, gs = inputs(4, 96, F32, F32)
    x[0], r[0] = 0.0, 0.0
    x[1], r[1] = 3.0, -3.0
    y = run(x, r, w, gy, gs)[0]
    assert float(y[:2].abs().sum()) == 0.0
    verify(x, r, w, gy, gs)


def test_inf_and_nan_stay_in_their_row():
    x, r, w, gy, gs = inputs(6, 300)
    clean = run(x, r, w, gy, gs)
    x[2, 17], r[4, 299] = float("inf"), float("nan")
    y, _s, gx, _gr, _gw = run(x, r, w, gy, gs)
    ok = [0, 1, 3, 5]
    assert torch.equal(y[ok], clean[0][ok]) and torch.isnan(y[[2, 4]]).any(1).all()
    assert torch.equal(gx[ok], clean[2][ok])


def test_zero_gradient_rows():
    """Padded rows without a gradient get none and give none."""
    x, r, w, gy, gs = inputs(50, 200, BF16, F32)
    gy[30:], gs[30:] = 0, 0
    _y, s, gx, _gr, gw = run(x, r, w, gy, gs)
    assert float(gx[30:].float().abs().sum()) == 0
    check("grad_w", gw, *R.rms_bwd(gy[:30], s[:30], w, EPS)["w"])


def test_against_differences():
    """Central differences of the 64-bit forward: a step of 1e-4 gives an error of its
    square, far below fp32's; 2e-3 of the gradient's norm bounds what fp32 is off by."""
    x, r, w, gy, gs = inputs(3, 24, F32, F32)
    x[::5] /= 50
    _y, _s, gx, gr, gw = run(x, r, w, gy, gs)
    X, RR, W, G, GS = (t.double().cpu() for t in (x, r, w, gy, gs))

    def f(X, RR, W):
        return float((R.rms_fwd(X + RR, W, EPS)[0] * G).sum() + ((X + RR) * GS).sum())

    for name, t, grad in (("x", X, gx), ("residual", RR, gr), ("w", W, gw)):
        num = torch.zeros_like(t)
        for i in range(t.numel()):
            e = torch.zeros(t.numel(), dtype=t.dtype)
            e[i] = 1e-4
            e = e.view_as(t)
            num.view(-1)[i] = (f(*[u + e if u is t else u for u in (X, RR, W)])
                               - f(*[u - e if u is t else u for u in (X, RR, W)])) / 2e-4
        assert float((num - grad.double().cpu()).norm()) <= 2e-3 * float(num.norm()), name


def test_eval_and_ops_agree():
    for T, C in ((1, 4096), (9, 100)):
        x, r, w, gy, gs = inputs(T, C)
        want, alone = run(x, r, w, gy, gs), run(x, None, w, gy, None)
        with torch.no_grad():
            y, s = flash_mhc.rms_norm(x, w, EPS, residual=r)
            assert torch.equal(y, want[0]) and torch.equal(s, want[1])
            assert torch.equal(flash_mhc.rms_norm(x, w, EPS), alone[0])
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
        y, s, _rstd = torch.ops.flash_mhc.add_rms_norm(*leaves, EPS)
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])
        for a, b in zip(torch.autograd.grad([y, s], leaves, [gy, gs]), want[2:]):
            assert torch.equal(a, b)
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        y, _rstd = torch.ops.flash_mhc.rms_norm(*leaves, EPS)
        for a, b in zip(torch.autograd.grad(y, leaves, gy), (alone[2], alone[4])):
            assert torch.equal(a, b)


def test_some_gradients_only():
    x, r, w, gy, gs = inputs(9, 72)
    for ins in ((x, r, w), (x, None, w)):
        want = run(ins[0], ins[1], w, gy, gs)[2:]
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
            leaves = [None if t is None else t.clone().requires_grad_(bool(n)) for t, n in zip(ins, need)]
            if not any(t is not None and t.requires_grad for t in leaves):
                continue
            out = flash_mhc.rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
            torch.autograd.backward([out] if leaves[1] is None else list(out), [gy] if leaves[1] is None else [gy, gs])
            for t, n, g in zip(leaves, need, want):
                if t is not None:
                    assert (t.grad is not None) == bool(n)
                    if n:
                        assert torch.equal(t.grad, g)


def test_one_output_only():
    """A loss of y alone, and of the sum alone."""
    x, r, w, gy, gs = inputs(11, 136)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = flash_mhc.rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
    gx, gr, gw = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    alone = run(s, None, w, gy, None)
    assert torch.equal(gx, alone[2]) and torch.equal(gr, gx) and torch.equal(gw, alone[4])
    gx, gr, gw = torch.autograd.grad(s, leaves, gs, allow_unused=True)
    assert torch.equal(gx, gs) and torch.equal(gr, gs) and gw is None


def test_the_same_tensor_twice():
    """x as its own residual: its gradient is the sum of the two."""
    x, _r, w, gy, gs = inputs(6, 200)
    leaf = x.clone().requires_grad_(True)
    y, s = flash_mhc.rms_norm(leaf, w, EPS, residual=leaf)
    g, = torch.autograd.grad([y, s], leaf, [gy, gs])
    want = run(x, x, w, gy, gs)
    assert torch.equal(y, want[0]) and torch.equal(g, want[2] + want[3])


def test_strided_unaligned_and_leading_dims():
    x, r, w, gy, gs = inputs(24, 104)
    want = run(x, r, w, gy, gs)
    wide = torch.empty(24, 208, device=DEV, dtype=BF16)
    wide[:, ::2] = x
    xt, rt = wide[:, ::2].requires_grad_(True), r.t().contiguous().t().requires_grad_(True)
    gt = torch.empty(104, 24, device=DEV, dtype=BF16).copy_(gy.t()).t()
    y, s = flash_mhc.rms_norm(xt, w, EPS, residual=rt)
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    for a, b in zip(torch.autograd.grad([y, s], [xt, rt], [gt, gs]), want[2:4]):
        assert torch.equal(a, b)

    def off(t):  # 2 bytes off a 16-byte address
        return torch.empty(1 + t.numel(), device=DEV, dtype=BF16)[1:].view_as(t).copy_(t)

    verify(off(x), off(r), w, off(gy), off(gs))
    shape = (2, 3, 4, 104)
    for a, b in zip(run(x.view(shape), r.view(shape), w, gy.view(shape), gs.view(shape)), want):
        assert torch.equal(a.reshape(b.shape), b)
    # A residual that is one row for all tokens, and a gradient broadcast from one value.
    row = r[:1].clone().requires_grad_(True)
    xs = x.clone().requires_grad_(True)
    y, s = flash_mhc.rms_norm(xs, w, EPS, residual=row.expand_as(x))
    (y.sum() + s.sum()).backward()
    one = torch.ones_like(gy)
    ref = run(x, row.detach().expand_as(x).contiguous(), w, one, one)
    assert torch.equal(xs.grad, ref[2])
    check("grad_row", row.grad, ref[2].double().cpu().sum(0, keepdim=True),
          24 * 2.0 ** -8 * ref[2].double().cpu().abs().sum(0, keepdim=True))  # torch adds in bf16


def test_empty():
    x = torch.empty(0, 40, device=DEV, dtype=BF16).requires_grad_(True)
    w = torch.ones(40, device=DEV).requires_grad_(True)
    y, s = flash_mhc.rms_norm(x, w, EPS, residual=torch.empty_like(x))
    gx, gw = torch.autograd.grad([y, s], [x, w], [torch.empty_like(y), torch.empty_like(y)])
    assert gx.shape == (0, 40) and float(gw.abs().sum()) == 0
    with torch.no_grad():
        assert flash_mhc.rms_norm(x, w).shape == (0, 40)


def test_deterministic_on_two_streams():
    args = inputs(3000, 520)
    want = run(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(*args))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        assert all(torch.equal(a, c) for a, c in zip(g, want))


def test_captured():
    x, r, w, gy, gs = inputs(700, 1024)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]

    def step():
        y, s = flash_mhc.rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
        return (y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [gy, gs]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for k in range(3):
        with torch.no_grad():
            x.copy_(rnd((700, 1024), 50 + k))
            gs.copy_(rnd((700, 1024), 60 + k))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want)), k


def test_many_elements():
    """More than 2^32 elements: offsets past 32 bits.  The last rows and a middle one."""
    C = 4096
    T = (1 << 32) // C + 7
    x = torch.zeros(T, C, device=DEV, dtype=BF16)
    part = rnd((9, C), 1).to(DEV)
    rows = [0, T // 2, *range(T - 7, T)]
    x[rows] = part
    w = rnd((C,), 2, 0.2, 1.0).to(DEV)
    with torch.no_grad():
        y, s = flash_mhc.rms_norm(x, w, EPS, residual=x)
    two = (part.float() * 2).to(BF16)
    assert torch.equal(s[rows], two)
    check("y", y[rows], *R.rms_fwd(two, w, EPS))
    del y
    leaf = s.requires_grad_(True)
    out = flash_mhc.rms_norm(leaf, w, EPS)
    g = out.detach()
    gx, = torch.autograd.grad(out, leaf, g)
    check("grad_x", gx[rows], *R.rms_bwd(g[rows], two, w, EPS)["x"])


def test_nothing_beside_the_outputs():
    """Sentinels around y, the sum, rstd and the gradients stay."""
    lib = _abi.load()
    for T, C in ((3, 5), (5, 100), (4, 777), (2, 17001)):
        x, r, w, gy, gs = inputs(T, C)
        s0 = _abi.stream_of(x)

        def guarded(n, dtype):
            buf = torch.full((n + 64,), 7.0, device=DEV, dtype=dtype)
            return buf, buf[32:32 + n]

        bufs = [guarded(T * C, BF16), guarded(T * C, BF16), guarded(T, F32), guarded(T * C, BF16), guarded(C, BF16)]
        (_, y), (_, s), (_, rstd), (_, gx), (_, gw) = bufs
        assert lib.fmhc_rms_norm_fwd(x.data_ptr(), r.data_ptr(), w.data_ptr(), y.data_ptr(), s.data_ptr(),
                                     rstd.data_ptr(), 1, 1, T, C, EPS, s0) == 0
        n = lib.fmhc_rms_norm_bwd_workspace_bytes(T, C)
        ws = torch.full((n + 64,), 77, device=DEV, dtype=torch.uint8)
        assert lib.fmhc_rms_norm_bwd(gy.data_ptr(), s.data_ptr(), rstd.data_ptr(), w.data_ptr(), gs.data_ptr(),
                                     gx.data_ptr(), gw.data_ptr(), ws.data_ptr(), n, 1, 1, T, C, s0) == 0
        want = run(x, r, w, gy, gs)
        for got, ref in zip((y, s, gx, gw), (want[0], want[1], want[2], want[4])):
            assert torch.equal(got.view_as(ref), ref)
        for buf, part in bufs:
            assert float((buf[:32] - 7).abs().sum() + (buf[32 + part.numel():] - 7).abs().sum()) == 0
        assert bool((ws[n:] == 77).all())


@pytest.mark.parametrize("T,C", [(513, 2048), (600, 16384), (515, 16390), (1025, 1024), (2000, 5), (5000, 32),
                                 (9000, 64), (4097, 520), (1100, 4096)])
def test_partial_sums_stay_in_the_workspace(T, C):
    """The workspace that the query names is enough, with a second gradient and without: what follows it stays."""
    lib = _abi.load()
    x, r, w, gy, gs = inputs(T, C, BF16, F32)
    n = lib.fmhc_rms_norm_bwd_workspace_bytes(T, C)
    assert n > 0
    rstd = (x.float().square().mean(-1) + EPS).rsqrt()
    for gi in (None, gs):
        ws = torch.full((n + 4096,), 77, device=DEV, dtype=torch.uint8)
        gx, gw = torch.empty_like(x), torch.empty_like(w)
        assert lib.fmhc_rms_norm_bwd(gy.data_ptr(), x.data_ptr(), rstd.data_ptr(), w.data_ptr(),
                                     None if gi is None else gi.data_ptr(), gx.data_ptr(), gw.data_ptr(), ws.data_ptr(),
                                     n, 1, 0, T, C, _abi.stream_of(x)) == 0
        assert bool((ws[n:] == 77).all())
        want = R.rms_bwd(gy, x, w, EPS, gi)
        check("grad_x", gx, *want["x"])
        check("grad_w", gw, *want["w"])


def test_hooks_for_saved_tensors():
    """Saved tensors that went through the host, lie elsewhere or have other strides."""
    x, r, w, gy, gs = inputs(20, 264, pdt=F32)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    norm = lambda: flash_mhc.rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
    want = torch.autograd.grad(norm(), leaves, [gy, gs])
    for unpack in (lambda t: t.to(DEV), lambda t: torch.stack([t, t], -1)[..., 0].to(DEV)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
            out = norm()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, [gy, gs]), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):  # left on the host
        out = norm()
    with pytest.raises(ValueError, match="expected cuda"):
        torch.autograd.grad(out, leaves, [gy, gs])


def test_compiled():
    """Traced and compiled, forward and backward: the eager call's bits."""
    x, r, w, gy, gs = inputs(33, 520)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]

    def both(x, r, w):
        y, s = flash_mhc.rms_norm(x, w, EPS, residual=r)
        return y, s, flash_mhc.rms_norm(s, None, EPS)

    fast = torch.compile(both, fullgraph=True)
    want, got = both(*leaves), fast(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    want, got = (torch.autograd.grad(list(out), leaves, [gy, gs, gy]) for out in (want, got))
    # The sum's two gradients are added by autograd, in bf16 or in the compiler's kernels: one rounding apart.
    for a, b in zip(want, got):
        assert float((a.float() - b.float()).norm()) <= 2.0 ** -8 * float(a.float().norm())
    strided = [t.t().contiguous().t() for t in (x, r)]
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(both(*strided, w), fast(*strided, w)))
