"""GPU tests of layer norm, forward and backward, with its input kept as it is and in 8 bits.

Values are compared with 64-bit ones; how far they may be off is derived in
oracle/act8_oracle.py."""

from __future__ import annotations

import pytest
import torch

import flash_mhc
from oracle import act8_oracle as A

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"
EPS = 1e-5


def rnd(shape, seed, scale=1.0, mean=0.0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + mean).to(dtype)


def inputs(T, C, dtype, pdt, seed=0):
    x = rnd((T, C), seed, 1.0, 0.25, dtype)
    x[::5] *= 50
    w, b = rnd((C,), seed + 1, 0.2, 1.0, pdt), rnd((C,), seed + 2, 0.2, 0.0, pdt)
    return x.to(DEV), w.to(DEV), b.to(DEV), rnd((T, C), seed + 3, dtype=dtype).to(DEV)


def run(x, w, b, g, bits, eps=EPS):
    leaves = [None if t is None else t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    y = flash_mhc.layer_norm(leaves[0], leaves[1], leaves[2], eps, activation_bits=bits)
    have = [t for t in leaves if t is not None]
    gr = iter(torch.autograd.grad(y, have, g))
    return y.detach(), *[None if t is None else next(gr) for t in leaves]


def verify(x, w, b, g, bits, eps=EPS):
    y, gx, gw, gb = run(x, w, b, g, bits, eps)
    A.check("y", y, *A.ln_fwd(x, w, b, eps))
    kept = A.unpack8(*A.pack8(x)) if bits == 8 else x
    r = A.ln_bwd(g, x, kept, w, eps)
    A.check("grad_x", gx.reshape(-1, x.shape[-1]), *r["x"])
    assert gx.dtype is x.dtype and y.dtype is x.dtype
    if w is not None:
        A.check("grad_w", gw, *r["w"])
        assert gw.dtype is w.dtype
    if b is not None:
        A.check("grad_b", gb, *r["b"])


TYPES = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)]
# One lane group to rows past the registers; whole, ragged and single columns.
SIZES = [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (40, 65), (33, 100), (70, 128), (31, 256), (17, 300), (9, 512),
         (20, 777), (6, 1000), (5, 1024), (9, 1535), (7, 2048), (3, 2560), (5, 4096), (2, 4099), (2, 6000), (2, 8192),
         (3, 12000), (2, 16384), (3, 16385), (2, 20000)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,C", SIZES)
def test_sizes(T, C, bits):
    verify(*inputs(T, C, BF16, BF16), bits)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype,pdt", TYPES)
@pytest.mark.parametrize("T,C", [(1, 40), (37, 100), (600, 264), (130, 1024), (65, 1001), (3, 4096), (2, 17000)])
def test_types(T, C, dtype, pdt, bits):
    verify(*inputs(T, C, dtype, pdt), bits)


@pytest.mark.parametrize("T,C", [(5000, 32), (4097, 520), (3000, 2000)])
def test_many_rows(T, C):
    for bits in (16, 8):
        verify(*inputs(T, C, BF16, F32), bits)


@pytest.mark.parametrize("C", [24, 520, 20000])
def test_without_parameters(C):
    x, w, b, g = inputs(7, C, BF16, BF16)
    for bits in (16, 8):
        verify(x, None, None, g, bits)
        verify(x, w, None, g, bits)
        verify(x, None, b, g, bits)


def test_far_mean():
    """A mean far from the spread: the variance is around the mean.  bf16 values
    near 256 are multiples of 2, exact in fp32, so the tolerance is the usual one."""
    x = (rnd((9, 512), 1, 8.0, 256.0)).to(DEV)
    _x, w, b, g = inputs(9, 512, BF16, BF16)
    verify(x, w, b, g, 16)
    xf = rnd((9, 512), 1, 1.0, 100.0, F32).to(DEV)
    verify(xf, w.float(), b.float(), g.float(), 16)


def test_constant_and_zero_rows():
    x, w, b, g = inputs(4, 96, F32, F32)
    x[0], x[1] = 0.0, 4.0  # sums and means of 4.0 are exact
    y, gx, gw, gb = run(x, w, b, g, 16)
    assert torch.equal(y[:2], b.expand(2, -1))
    verify(x, w, b, g, 16)


def test_inf_and_nan_stay_in_their_row():
    x, w, b, g = inputs(6, 300, BF16, BF16)
    clean = run(x, w, b, g, 8)
    x[2, 17], x[4, 299] = float("inf"), float("nan")
    for bits in (16, 8):
        y, gx, _gw, _gb = run(x, w, b, g, bits)
        ok = [0, 1, 3, 5]
        assert torch.equal(y[ok], clean[0][ok]) and torch.isnan(y[[2, 4]]).any(1).all()
        assert torch.isfinite(gx[ok]).all()
        if bits == 8:
            assert torch.equal(gx[ok], clean[1][ok])


def test_zero_gradient_rows():
    """Padded rows with no gradient: they get none and give none."""
    x, w, b, g = inputs(50, 200, BF16, F32)
    g[30:] = 0
    _y, gx, gw, gb = run(x, w, b, g, 16)
    assert float(gx[30:].float().abs().sum()) == 0
    r = A.ln_bwd(g[:30], x[:30], x[:30], w, EPS)
    A.check("grad_w", gw, *r["w"])
    A.check("grad_b", gb, *r["b"])


def test_against_differences():
    """grad_x, grad_w, grad_b against central differences of the 64-bit forward.
    f = sum(y g) is smooth; step s gives an error of order s^2, with s = 1e-4
    1e-8 of the values, far below fp32's; 2e-3 of the gradient's norm bounds
    what the fp32 gradients may be off by a wide margin."""
    x, w, b, g = inputs(3, 24, F32, F32)
    x[::5] /= 50
    _y, gx, gw, gb = run(x, w, b, g, 16)
    X, W, B, Gr = (t.double().cpu() for t in (x, w, b, g))
    f = lambda X, W, B: float((A.ln_fwd(X, W, B, EPS)[0] * Gr).sum())
    for name, t, grad in (("x", X, gx), ("w", W, gw), ("b", B, gb)):
        num = torch.zeros_like(t)
        for i in range(t.numel()):
            e = torch.zeros_like(t).view(-1)
            e[i] = 1e-4
            e = e.view_as(t)
            hi = f(*[u + e if u is t else u for u in (X, W, B)])
            lo = f(*[u - e if u is t else u for u in (X, W, B)])
            num.view(-1)[i] = (hi - lo) / 2e-4
        assert float((num - grad.double().cpu()).norm()) <= 2e-3 * float(num.norm()), name


def test_eval_and_ops_agree():
    for T, C in ((1, 4096), (9, 100)):
        x, w, b, g = inputs(T, C, BF16, BF16)
        y = run(x, w, b, g, 16)[0]
        with torch.no_grad():
            assert torch.equal(flash_mhc.layer_norm(x, w, b, EPS), y)
            assert torch.equal(flash_mhc.layer_norm(x, w, b, EPS, activation_bits=8), y)
        for op in (torch.ops.flash_mhc.layer_norm, torch.ops.flash_mhc.layer_norm_pack8):
            leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
            out = op(*leaves, EPS)
            assert torch.equal(out[0], y)
            if len(out) == 5:
                assert all(torch.equal(a.cpu(), r) for a, r in zip(out[3:], A.pack8(x)))
            bits = 16 if len(out) == 3 else 8
            for a, r in zip(torch.autograd.grad(out[0], leaves, g), run(x, w, b, g, bits)[1:]):
                assert torch.equal(a, r)


def test_some_gradients_only():
    x, w, b, g = inputs(9, 72, BF16, BF16)
    want = run(x, w, b, g, 16)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        leaves = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        y = flash_mhc.layer_norm(*leaves, EPS)
        y.backward(g)
        for t, n, r in zip(leaves, need, want[1:]):
            assert (t.grad is not None) == bool(n)
            if n:
                assert torch.equal(t.grad, r)


def test_strided_unaligned_and_leading_dims():
    x, w, b, g = inputs(24, 104, BF16, BF16)
    want = run(x, w, b, g, 8)
    wide = torch.empty(24, 208, device=DEV, dtype=BF16)
    wide[:, ::2] = x
    xt = wide[:, ::2].requires_grad_(True)
    gt = torch.empty(104, 24, device=DEV, dtype=BF16).copy_(g.t()).t()
    y = flash_mhc.layer_norm(xt, w, b, EPS, activation_bits=8)
    assert torch.equal(y, want[0])
    assert torch.equal(torch.autograd.grad(y, xt, gt)[0], want[1])
    off = torch.empty(1 + x.numel(), device=DEV, dtype=BF16)[1:].view_as(x).copy_(x)  # 2 bytes off
    for a, r in zip(run(off, w, b, g, 8), want):
        assert a.shape == r.shape
        assert float((a.double() - r.double()).norm()) <= 2.0 ** -8 * float(r.double().norm())
    for a, r in zip(run(x.view(2, 3, 4, 104), w, b, g.view(2, 3, 4, 104), 8), want):
        assert torch.equal(a.reshape(r.shape), r)
    # A gradient broadcast from one value.
    xs = x.clone().requires_grad_(True)
    flash_mhc.layer_norm(xs, w, b, EPS).sum().backward()
    assert torch.equal(xs.grad, run(x, w, b, torch.ones_like(g), 16)[1])


def test_empty():
    x = torch.empty(0, 40, device=DEV, dtype=BF16).requires_grad_(True)
    w = torch.ones(40, device=DEV).requires_grad_(True)
    b = torch.ones(40, device=DEV).requires_grad_(True)
    y = flash_mhc.layer_norm(x, w, b, EPS, activation_bits=8)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert gx.shape == (0, 40) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0


def test_deterministic_on_two_streams():
    x, w, b, g = inputs(3000, 520, BF16, BF16)
    want = run(x, w, b, g, 8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(x, w, b, g, 8))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for r in got:
        assert all(torch.equal(a, c) for a, c in zip(r, want))


def test_captured():
    x, w, b, g = inputs(700, 1024, BF16, BF16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = flash_mhc.layer_norm(*leaves, EPS, activation_bits=8)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

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
            x.copy_(inputs(700, 1024, BF16, BF16, seed=20 + k)[0])
        for graph in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_module():
    m = flash_mhc.LayerNorm(96, activation_bits=8).to(DEV)
    ref = torch.nn.LayerNorm(96).to(DEV)
    assert list(m.state_dict()) == list(ref.state_dict())
    m.load_state_dict(ref.state_dict())
    x = rnd((5, 96), 1, dtype=F32).to(DEV)
    A.check("y", m(x), *A.ln_fwd(x, m.weight, m.bias, m.eps))
    y = m.double()(x.double())  # a dtype that the kernels do not take
    assert y.dtype is torch.float64
    comp = torch.compile(flash_mhc.LayerNorm(96).to(DEV), fullgraph=True, backend="aot_eager")
    xs = x.clone().requires_grad_(True)
    comp(xs).square().sum().backward()
    xe = x.clone().requires_grad_(True)
    flash_mhc.LayerNorm(96).to(DEV)(xe).square().sum().backward()
    assert torch.equal(xs.grad, xe.grad)


# Every way to lay rows over lanes: the lanes per row depend on the columns and
# the rows.  Memory that held NaN shows a row that is not written.
@pytest.mark.parametrize("T,C", [(4, 8193), (4, 10240), (520, 4100), (520, 8192), (520, 8200), (520, 10240), (520, 10250),
                                 (520, 16384), (1030, 1030), (1030, 1544), (1030, 2560), (1030, 2568), (8200, 1540),
                                 (8200, 2564), (8200, 4104)])
def test_layouts(T, C):
    x, w, b, g = inputs(T, C, BF16, F32)
    held = [torch.full((T, C), float("nan"), dtype=BF16, device=DEV) for _ in range(8)]
    del held
    verify(x, w, b, g, 16 if T > 8000 else 8)


@pytest.mark.parametrize("T", [3, 530, 1030])
def test_layouts_fp32(T):
    for C in (1536, 1544, 6000, 8200) if T < 1000 else (1544,):
        verify(*inputs(T, C, F32, F32), 16)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,C,dtype", [(1, 5, BF16), (3, 40, F16), (70, 300, BF16), (33, 1024, F32), (1100, 2048, BF16),
                                       (9, 1001, BF16), (40, 4096, F16), (3, 8200, BF16), (2, 16384, BF16),
                                       (2, 17001, BF16), (2, 17000, F32)])
def test_with_residual(T, C, dtype, bits):
    """The bits of two gradients that are added."""
    x, w, b, g = inputs(T, C, dtype, F32)
    g2 = rnd((T, C), 9, 0.5, dtype=dtype).to(DEV)
    norm = flash_mhc.LayerNorm(C, activation_bits=bits).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(w)
        norm.bias.copy_(b)
    for other in (lambda r: r, lambda r: r.t().contiguous().t()):  # a strided gradient too
        results = []
        for fused in (True, False):
            xs = x.clone().requires_grad_(True)
            y, r = norm.with_residual(xs) if fused else (norm(xs), xs)
            assert torch.equal(r, x)
            results.append((y, *torch.autograd.grad([y, r], [xs, norm.weight, norm.bias], [g, other(g2)])))
        for a, c in zip(*results):
            assert torch.equal(a, c)
    # One of the two only.
    xs = x.clone().requires_grad_(True)
    y, r = norm.with_residual(xs)
    assert torch.equal(torch.autograd.grad(r, xs, g2, retain_graph=True)[0], g2)
    only = torch.autograd.grad(y, xs, g)[0]
    xs = x.clone().requires_grad_(True)
    assert torch.equal(only, torch.autograd.grad(norm(xs), xs, g)[0])


def test_with_residual_in_a_block():
    """Hooks are called, in-place layers work, other norms and frozen inputs too."""
    torch.manual_seed(0)
    C = 96
    layer = torch.nn.Sequential(torch.nn.ReLU(inplace=True), torch.nn.Linear(C, C))
    blk = flash_mhc.MHCLiteBlock(4, C, layer, pre_norm=True).to(DEV).to(BF16)
    x = rnd((17, 4, C), 1).to(DEV)

    def step():
        xs = x.clone().requires_grad_(True)
        out = blk(xs)
        return out, *torch.autograd.grad(out.float().square().sum(), [xs, *blk.parameters()])

    want = step()
    seen = []
    handle = blk.norm.register_forward_hook(lambda m, a, out: seen.append(out.shape))
    got = step()
    handle.remove()
    assert seen == [(17, C)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: seen.append(type(m).__name__))
    got = step()
    handle.remove()
    assert "LayerNorm" in seen
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    blk.norm.requires_grad_(False)
    out = blk(x.clone().requires_grad_(True))
    assert torch.equal(out, want[0])
    out.float().sum().backward()
    blk.norm = torch.nn.RMSNorm(C, device=DEV, dtype=BF16)
    assert torch.isfinite(step()[1]).all()


def test_opcheck():
    x, w, b, g = inputs(7, 72, BF16, F32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y, mean, rstd, q, s = torch.ops.flash_mhc.layer_norm_pack8(x, w, b, EPS)
    check = torch.library.opcheck
    check(torch.ops.flash_mhc.layer_norm, (*leaves, EPS))
    check(torch.ops.flash_mhc.layer_norm, (leaves[0], None, None, EPS))
    check(torch.ops.flash_mhc.layer_norm_pack8, (*leaves, EPS))
    check(torch.ops.flash_mhc.layer_norm_backward, (g, x, None, None, mean, rstd, w, F32, True, True))
    check(torch.ops.flash_mhc.layer_norm_backward, (g, None, q, s, mean, rstd, w, F32, True, False))


@pytest.mark.parametrize("bits", [16, 8])
def test_differentiable_once(bits):
    x, w, b, _g = inputs(5, 48, F32, F32)
    x.requires_grad_(True)
    (gx,) = torch.autograd.grad(flash_mhc.layer_norm(x, w, b, activation_bits=bits).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.square().sum().backward()


@pytest.mark.parametrize("C", [2048, 2051])
def test_past_32_bits(C):
    """Over 2^32 elements: 2100 copies of the same rows have the same results.  (One
    copy alone is summed in another order: fewer rows take more lanes each.)"""
    n, reps = 1000, 2100
    T = n * reps
    assert T * C > 1 << 32
    x, w, b, g = inputs(n, C, BF16, BF16)
    t, d = x.repeat(reps, 1), g.repeat(reps, 1)
    y, mean, rstd, q, s = torch.ops.flash_mhc.layer_norm_pack8(t, w, b, EPS)
    bwd = torch.ops.flash_mhc.layer_norm_backward
    gx = bwd(d, t, None, None, mean, rstd, w, BF16, True, True)[0]
    gx8 = bwd(d, None, q, s, mean, rstd, w, BF16, False, False)[0]
    for o in (y, mean, rstd, q, s, gx, gx8):
        for k in (reps // 2, reps - 1):
            assert torch.equal(o[k * n:(k + 1) * n], o[:n])
    A.check("y", y[:n], *A.ln_fwd(x, w, b, EPS))
    A.check("grad_x", gx[:n], *A.ln_bwd(g, x, x, w, EPS)["x"])
    A.check("grad_x of 8 bits", gx8[:n], *A.ln_bwd(g, x, A.unpack8(*A.pack8(x)), w, EPS)["x"])
    del t, d, y, mean, rstd, q, s, gx, gx8, o
    torch.cuda.empty_cache()


def test_one_row_without_leading_dims_and_two_streams_at_once():
    x, w, b, g = inputs(1, 1000, BF16, F32)
    verify(x[0], w, b, g[0], 16)
    verify(x[0], w, b, g[0], 8)
    # Two forwards and backwards that overlap on two streams, workspaces of their own.
    many = [inputs(3000, 520, BF16, F32, seed) for seed in (1, 2)]
    want = [run(*m, 8) for m in many]
    streams = [torch.cuda.Stream() for _ in many]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s, m in zip(streams, many):
        with torch.cuda.stream(s):
            got.append(run(*m, 8))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, c in zip(got, want):
        for u, v in zip(a, c):
            assert torch.equal(u, v)


class Fenced:
    """Outputs inside larger buffers whose other bytes have to stay as they were."""

    def __init__(self):
        self.held = []

    def __call__(self, shape, dtype):
        n = torch.empty(shape, dtype=dtype, device="meta").numel() * dtype.itemsize
        buf = torch.full((n + 1024,), 0xA5, dtype=torch.uint8, device=DEV)
        self.held.append((buf, n))
        return buf[512:512 + n].view(dtype).view(shape)

    def check(self):
        for buf, n in self.held:
            assert bool((buf[:512] == 0xA5).all()) and bool((buf[512 + n:] == 0xA5).all())


@pytest.mark.parametrize("T,C", [(1, 1), (3, 7), (5, 8), (2, 33), (7, 100), (130, 300), (33, 1001), (1030, 1544), (5, 2560),
                                 (3, 4099), (2, 8200), (2, 16384), (3, 17003)])
@pytest.mark.parametrize("dtype,code", [(BF16, 1), (F32, 0)])
def test_writes_stay_inside(T, C, dtype, code):
    """Every output of layer norm, pack8 and unpack8 is written whole and nothing beside it."""
    from flash_mhc import _abi

    lib, st = _abi.load(), torch.cuda.current_stream().cuda_stream
    x, w, b, g = inputs(T, C, dtype, F32)
    out, G = Fenced(), (C + 31) // 32
    y, mean, rstd = out((T, C), dtype), out((T,), F32), out((T,), F32)
    q, s = out((T, C), torch.int8), out((T, G), torch.uint8)
    P = lambda *ts: [None if t is None else t.data_ptr() for t in ts]
    _abi.check(lib.fmhc_layer_norm_fwd(*P(x, w, b, y, mean, rstd, q, s), code, 0, T, C, EPS, st), "forward")
    nbytes = lib.fmhc_layer_norm_bwd_workspace_bytes(T, C)
    for kept in ((x, None, None), (None, q, s)):
        for extra in (None, g):
            gx, gw, gb = out((T, C), dtype), out((C,), F32), out((C,), F32)
            ws = out((nbytes,), torch.uint8)
            _abi.check(lib.fmhc_layer_norm_bwd(*P(g, *kept, mean, rstd, w, extra, gx, gw, gb, ws), nbytes, code, 0, T, C,
                                               st), "backward")
            a = torch.ops.flash_mhc.layer_norm_backward(g, *kept, mean, rstd, w, F32, True, True)
            assert torch.equal(gw, a[1]) and torch.equal(gb, a[2])
            assert torch.equal(gx, a[0] if extra is None else a[0] + g)
    q2, s2, back = out((T, C), torch.int8), out((T, G), torch.uint8), out((T, C), dtype)
    _abi.check(lib.fmhc_pack8(*P(x), code, *P(q2, s2), T, C, st), "pack8")
    _abi.check(lib.fmhc_unpack8(*P(q2, s2, back), code, T, C, st), "unpack8")
    out.check()
    want = torch.ops.flash_mhc.layer_norm_pack8(x, w, b, EPS)
    for a, v in zip((y, mean, rstd, q, s), want):
        assert torch.equal(a, v)
    assert torch.equal(q2, q) and torch.equal(s2, s)
    assert torch.equal(back, flash_mhc.unpack8(q, s, dtype))
