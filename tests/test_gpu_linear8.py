"""GPU tests of rows in 8 bits and of their product.

pack8_rows is tested for the bits that the format's fp32 operations give on the CPU; the
others against 64-bit values (oracle/rows8_oracle.py derives how far they may be off)."""

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


def rows(T, C, dtype=BF16, seed=0):
    x = rnd((T, C), seed, 1.0, 0.25, dtype)
    x[::5] *= 50
    return x.to(DEV)


ROWS = [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (40, 65), (33, 100), (70, 128), (31, 256), (17, 300), (9, 512),
        (20, 777), (6, 1000), (5, 1024), (9, 1535), (7, 2048), (3, 2560), (5, 4096), (2, 4099), (2, 8192), (3, 12000),
        (2, 16384), (3, 16385), (2, 20000), (5000, 32), (1100, 4096)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,C", ROWS)
def test_pack_rows(T, C, dtype):
    x = rows(T, C, dtype)
    codes, scales = flash_mhc.pack8_rows(x)
    want = R.pack_rows(x)
    assert codes.shape == (T, C) and codes.dtype is torch.int8 and scales.dtype is F32
    assert codes.stride() == (-(-C // 16) * 16, 1)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])


def test_pack_rows_edges():
    """Zero rows, tiny and huge ones, ties, Inf and NaN."""
    x = torch.zeros(9, 40)
    x[1] = 1e-38
    x[2] = 1e-42
    x[3] = 3e38
    x[4, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])  # unit 1: half to even
    x[5] = rnd((40,), 1, dtype=F32)
    x[5, 3] = float("inf")
    x[6] = rnd((40,), 2, dtype=F32)
    x[6, 39] = float("nan")
    x[7] = -0.0
    x[8, 0] = 2.0 ** -100
    codes, scales = flash_mhc.pack8_rows(x.to(DEV))
    want = R.pack_rows(x)
    assert torch.equal(codes.cpu(), want[0])
    assert torch.equal(torch.isnan(scales).cpu(), torch.isnan(want[1])) and bool(torch.isnan(scales[5:7]).all())
    assert torch.equal(scales.cpu().nan_to_num(0), want[1].nan_to_num(0))
    assert want[0][4, :4].tolist() == [127, 0, 2, -2] and int(want[0][8, 0]) == 127
    out = flash_mhc.linear8(codes, scales, torch.ones(3, 40, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV))
    assert bool(torch.isnan(out[5:7]).all()) and bool(torch.isfinite(out[[0, 1, 2, 4, 7, 8]]).all())
    assert bool(torch.isinf(out[3]).all())  # 40 times 3e38 is past the largest bf16 (3.39e38)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,pdt", [(BF16, BF16), (BF16, F32), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("T,C", [(1, 1), (2, 6), (3, 8), (9, 100), (31, 256), (20, 777), (5, 1024), (7, 2048),
                                 (3, 2560), (5, 4096), (2, 8192), (3, 16385), (600, 264), (1100, 4096)])
def test_norm_rows(T, C, dtype, pdt, residual):
    x, w = rows(T, C, dtype), rnd((C,), 1, 0.2, 1.0, pdt).to(DEV)
    r = rnd((T, C), 4, 2.0, 0.0, dtype).to(DEV) if residual else None
    out = flash_mhc.rms_norm_pack8_rows(x, w, EPS, residual=r)
    s = x
    if residual:
        s = out[2]
        assert torch.equal(s.cpu(), R.add(x, r))
    else:
        assert len(out) == 2
    R.check_rows(out[0], out[1], *R.rms_fwd(s, w, EPS))
    op = (torch.ops.flash_mhc.rms_norm_pack8_rows(x, w, EPS) if r is None
          else torch.ops.flash_mhc.add_rms_norm_pack8_rows(x, r, w, EPS))
    assert all(torch.equal(a, b) for a, b in zip(op, out))


def test_norm_rows_without_weight_and_with_bad_rows():
    x = rows(6, 300)
    clean = flash_mhc.rms_norm_pack8_rows(x, None, EPS)
    R.check_rows(*clean, *R.rms_fwd(x, None, EPS))
    x[2, 17], x[4, 299] = float("inf"), float("nan")
    x[5] = 0
    codes, scales = flash_mhc.rms_norm_pack8_rows(x, None, EPS)
    ok = [0, 1, 3]
    assert torch.equal(codes[ok], clean[0][ok]) and torch.equal(scales[ok], clean[1][ok])
    assert bool(torch.isnan(scales[[2, 4]]).all()) and int(codes[[2, 4, 5]].abs().max()) == 0
    assert float(scales[5]) == float(torch.tensor(2.0 ** -100) / 127)


@pytest.mark.parametrize("C", [5, 40, 1024, 20000])
def test_norm_rows_at_the_ends_of_fp32(C):
    """Products with the weight past fp32's range and below its normal numbers, at eps = 0."""
    x = torch.ones(4, C, device=DEV) * torch.tensor([2.0 ** 60, 2.0 ** -63, 1.0, 0.0], device=DEV)[:, None]
    for e, bad in ((70, [0, 3]), (-70, [3])):  # 2^130 and 2^-133 (0 / 0 in the last row)
        codes, scales = flash_mhc.rms_norm_pack8_rows(x, torch.full((C,), 2.0 ** e, device=DEV), 0.0)
        assert bool(torch.isnan(scales[bad]).all()) and int(codes[bad].abs().max()) == 0
        # (The scale is off by the statistic's roundings: C / C, rsqrt, and its own two.)
        # From C = 256 on the first row's sum of squares is 2^120 C >= 2^128, past fp32: rstd and the norm are 0.
        zero = C >= 256
        for row in ([2] if e > 0 or zero else [0, 2]):
            assert abs(float(scales[row]) * 127 / 2.0 ** e - 1) <= 2.0 ** -21 and int(codes[row].min()) == 127
        for row in ([] if e > 0 else [0, 1] if zero else [1]):
            assert float(scales[row]) == float(torch.tensor(2.0 ** -100) / 127) and int(codes[row].abs().max()) == 0


def test_norm_rows_in_fp32_are_the_norms_rows():
    """fp32 rows are packed from the values that rms_norm returns: the same codes but for the
    scale's last bits."""
    x, w = rows(40, 520, F32), rnd((520,), 1, 0.2, 1.0, F32).to(DEV)
    codes, scales = flash_mhc.rms_norm_pack8_rows(x, w, EPS)
    q, s = flash_mhc.pack8_rows(flash_mhc.rms_norm(x, w, EPS))
    assert float((s - scales).abs().max() / s.max()) <= 2.0 ** -21
    assert int((q.int() - codes.int()).abs().max()) <= 1 and float((q != codes).float().mean()) < 1e-3


def test_strided_and_leading_dims():
    x, w = rows(24, 104), rnd((104,), 1, 0.2, 1.0).to(DEV)
    want, packed = flash_mhc.rms_norm_pack8_rows(x, w, EPS, residual=x), flash_mhc.pack8_rows(x)
    wide = torch.empty(24, 208, device=DEV, dtype=BF16)
    wide[:, ::2] = x
    off = torch.empty(1 + x.numel(), device=DEV, dtype=BF16)[1:].view_as(x).copy_(x)
    for t in (wide[:, ::2], x.t().contiguous().t(), off):
        for a, b in zip(flash_mhc.rms_norm_pack8_rows(t, w, EPS, residual=t), want):
            assert torch.equal(a, b)
        for a, b in zip(flash_mhc.pack8_rows(t), packed):
            assert torch.equal(a, b)
    codes, scales = flash_mhc.pack8_rows(x.view(2, 3, 4, 104))
    assert codes.shape == (2, 3, 4, 104) and scales.shape == (2, 3, 4)
    assert torch.equal(codes.reshape(24, 104), packed[0]) and torch.equal(scales.reshape(24), packed[1])


def test_one_row_without_a_batch():
    x, w = rows(1, 100)[0], rnd((7, 100), 3, dtype=F32).to(DEV)
    q, s = flash_mhc.pack8_rows(x)
    wq, ws = flash_mhc.pack8_rows(w)
    assert q.shape == (100,) and s.shape == ()
    out = flash_mhc.linear8(q, s, wq, ws, residual=x[:7].contiguous())
    assert out.shape == (7,)
    check("row", out, *R.linear8(q[None], s[None], wq, ws, None, x[None, :7]))
    n, sn = flash_mhc.rms_norm_pack8_rows(x)
    R.check_rows(n[None], sn[None], *R.rms_fwd(x[None], None, EPS))
    y, total = flash_mhc.rms_norm(x, residual=x)
    assert torch.equal(total, x + x)
    check("norm", y, *(t[0] for t in R.rms_fwd(total[None], None, EPS)))
    with torch.no_grad():
        layer = flash_mhc.Linear8.from_linear(torch.nn.Linear(100, 7).to(DEV))
        assert layer(x).shape == (7,) and layer(x.expand(2, 3, 100)).shape == (2, 3, 7)


def test_rows_leave_what_is_between():
    """The bytes between rows, and before and behind the codes, stay as they were."""
    lib = _abi.load()
    for C, ld in ((5, 16), (33, 48), (100, 131), (1001, 1008), (17001, 17008)):
        T = 6
        x = rows(T, C)
        want = R.pack_rows(x)
        for norm in (False, True):
            buf = torch.full((64 + T * ld,), 99, device=DEV, dtype=torch.int8)
            sc = torch.full((T + 8,), 99.0, device=DEV)
            q = buf[32:32 + T * ld].view(T, ld)
            st = _abi.stream_of(x)
            if norm:
                rc = lib.fmhc_rms_norm_pack8_rows(x.data_ptr(), None, None, q.data_ptr(), sc[4:].data_ptr(), None, 1, 0,
                                                  T, C, ld, EPS, st)
            else:
                rc = lib.fmhc_pack8_rows(x.data_ptr(), 1, q.data_ptr(), sc[4:].data_ptr(), T, C, ld, st)
                assert torch.equal(q[:, :C].cpu(), want[0])
            assert rc == 0
            assert bool((buf[:32] == 99).all()) and bool((buf[32 + T * ld:] == 99).all())
            assert bool((q[:, C:] == 99).all())
            assert bool((sc[:4] == 99).all()) and bool((sc[4 + T:] == 99).all())


# ---------------------------------------------------------------------------
# The product


def codes(shape, seed, lo=-127, hi=127):
    """Codes in rows at a 16-byte pitch whose gaps hold anything."""
    g = torch.Generator().manual_seed(seed)
    K = shape[-1]
    full = torch.randint(-128, 128, (*shape[:-1], -(-K // 16) * 16), generator=g, dtype=torch.int8)
    full[..., :K] = torch.randint(lo, hi + 1, shape, generator=g, dtype=torch.int8)
    return full.to(DEV)[..., :K]


def operands(T, N, K, seed=0):
    xs, ws = rnd((T,), seed + 2, dtype=F32).abs().to(DEV) * 0.02, rnd((N,), seed + 3, dtype=F32).abs().to(DEV) * 0.01
    return codes((T, K), seed), xs, codes((N, K), seed + 1), ws


def verify(T, N, K, dtype=BF16, bias=None, residual=False, seed=0):
    x, xs, w, ws = operands(T, N, K, seed)
    b = None if bias is None else rnd((N,), seed + 4, 0.1, dtype=bias).to(DEV)
    r = rnd((T, N), seed + 5, dtype=dtype).to(DEV) if residual else None
    out = flash_mhc.linear8(x, xs, w, ws, b, residual=r, dtype=dtype)
    assert out.shape == (T, N) and out.dtype is dtype and out.is_contiguous()
    check(f"{T} {N} {K}", out, *R.linear8(x, xs, w, ws, b, r))
    return out


TOKENS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 257, 300, 513]
WIDTHS = [(1, 1), (3, 5), (16, 16), (17, 63), (40, 64), (64, 65), (100, 127), (128, 128), (129, 129), (250, 200),
          (256, 256), (257, 300), (512, 520), (777, 1001), (1024, 1024), (300, 2560), (1000, 4096)]


@pytest.mark.parametrize("N,K", WIDTHS)
@pytest.mark.parametrize("T", TOKENS)
def test_sizes(T, N, K):
    verify(T, N, K, bias=F32 if T % 2 else None, residual=bool(N % 2))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,N,K", [(1, 100, 72), (5, 4096, 4096), (33, 520, 1000), (200, 300, 700), (1030, 512, 256)])
def test_types(T, N, K, dtype):
    for bias in (None, F32, dtype):
        for residual in (False, True):
            verify(T, N, K, dtype, bias, residual)


@pytest.mark.parametrize("T,N,K", [(5000, 40, 64), (4099, 520, 264), (2003, 777, 1001), (16400, 1024, 128),
                                   (2500, 4096, 96), (1300, 2560, 2560), (3, 9000, 40), (70, 12345, 33)])
def test_many(T, N, K):
    verify(T, N, K, bias=F32, residual=True)


# Sizes at which each of the product's kernels is taken: rows in lines, rows off them, and edges.
KINDS = [(8, 8000), (40, 2000), (192, 2560), (201, 2561), (1024, 2560), (1030, 2603), (1030, 2600), (2048, 4096),
         (2049, 4097), (8192, 2048), (8190, 2041), (8190, 2040)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,N", KINDS)
def test_kinds(T, N, dtype):
    for residual in (False, True):
        verify(T, N, 200, dtype, F32, residual)


@pytest.mark.parametrize("K", [1, 64, 127, 128, 129, 256, 257, 500, 512, 513, 640, 769, 1024, 1300])
def test_lengths(K):
    """Ends inside and at a step, and numbers of steps on both sides of what lies in LDS."""
    for T, N in ((8, 8000), (40, 2000), (192, 1111), (1030, 2600), (2049, 4097), (8190, 2048)):
        x, xs, w, ws = operands(T, N, K)
        out = flash_mhc.linear8(x, xs, w, ws, dtype=F32)
        pick = torch.tensor([0, 1, T // 2, T - 7, T - 2, T - 1], device=DEV)
        check(f"{T} {N} {K}", out[pick], *R.linear8(x[pick], xs[pick], w, ws))
        # All of it against the same rows in another order, which lie in other tiles.
        turned = flash_mhc.linear8(x.flip(0), xs.flip(0), w, ws, dtype=F32)
        assert torch.equal(turned.flip(0), out)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_exact_sums(T):
    """The largest codes over the longest rows: the integer sum stays exact."""
    K = (1 << 17) - 1
    x = torch.full((T, K + 1), -128, dtype=torch.int8, device=DEV)[:, :K]
    w = torch.full((18, K + 1), -128, dtype=torch.int8, device=DEV)[:, :K]
    w[1] = 127
    w[2, 1:] = 0
    out = flash_mhc.linear8(x, torch.ones(T, device=DEV), w, torch.ones(18, device=DEV), dtype=F32)
    for n, v in ((0, K << 14), (1, -K * 128 * 127), (2, 1 << 14)):
        assert bool((out[:, n].double() == float(torch.tensor(v).to(F32))).all())


def check_range(name, out, value, error):
    """check, where a value that rounds past the type's largest is Inf: from half a step above it on, which is
    65504 + 16 in fp16 (steps of 32 from 2^15 on), max + max eps / (2 - eps) / 2 in general."""
    info = torch.finfo(out.dtype)
    half = info.max * info.eps / (2 - info.eps) / 2
    past = value.abs() >= info.max + half + error
    o = out.detach().to("cpu", torch.float64)
    assert torch.equal(o[past], torch.sign(value[past]) * float("inf"))
    assert not bool(((value.abs() - info.max - half).abs() < error).any())  # none that may be either
    check(name, out.cpu().masked_fill(past, 0), value.masked_fill(past, 0), error)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,N", [(1, 4096), (8, 8000), (40, 2000), (192, 2560), (201, 2561), (1030, 2600), (2048, 4096),
                                 (2049, 4097), (8192, 2048), (8190, 2041)])
def test_scales_at_the_ends_of_fp32(T, N, dtype):
    """A sum times its larger scale is past fp32's range, times both it is not; in all, some or one of the rows."""
    x, xs, w, ws = operands(T, N, 200)
    w[N // 2] = 0
    small, large = 1e-35, 1e36 / 0.02
    for mine, other, n in ((xs, ws, T), (ws, xs, N)):
        for which in (slice(None), slice(None, None, 3), slice(n - 1, n)):
            a, b = mine.clone(), other * small
            a[which] *= large
            pair = (a, b) if mine is xs else (b, a)
            for residual in (None, rnd((T, N), 5, 100.0, dtype=dtype).to(DEV)):
                out = flash_mhc.linear8(x, pair[0], w, pair[1], residual=residual, dtype=dtype)
                check_range(f"{T} {N}", out, *R.linear8(x, pair[0], w, pair[1], None, residual))
    # On both sides of where the order changes, and rows that are NaN.
    a = xs * 0 + 2.0 ** 96
    a[::2] = 2.0 ** 96 * (1 + 2.0 ** -23)
    a[T // 2] = float("nan")
    out = flash_mhc.linear8(x, a, w, ws * 1e-30, dtype=dtype)
    ok = [t for t in range(T) if t != T // 2]
    check_range("threshold", out[ok], *R.linear8(x[ok], a[ok], w, ws * 1e-30))
    assert bool(torch.isnan(out[T // 2]).all())


def test_large_scales_among_many_tiles():
    """Workgroups with several tiles, of which some hold tokens with large scales: before, between and behind others."""
    T, N, K = 66000, 1024, 264
    x, xs, w, ws = operands(T, N, K)
    ws = ws * 1e-35
    want = flash_mhc.linear8(x, xs, w, ws, dtype=F32)
    large = torch.tensor([3, 255, 256, 9000, 30000, 30001, 65535, 65999], device=DEV)
    xs[large] *= 1e36 / 0.02
    out = flash_mhc.linear8(x, xs, w, ws, dtype=F32)
    check("large", out[large], *R.linear8(x[large], xs[large], w, ws))
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[large] = False
    assert torch.equal(out[rest], want[rest])


@pytest.mark.parametrize("T", [2, 40, 700])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_of_huge_rows(T, dtype):
    lin = torch.nn.Linear(4096, 300, bias=False)
    torch.nn.init.constant_(lin.weight, 0.01)
    layer = flash_mhc.Linear8.from_linear(lin).to(DEV)
    x = torch.full((T, 4096), 1e33, device=DEV, dtype=dtype)
    with torch.no_grad():
        y = layer(x)
    check("layer", y, *R.linear8(*R.pack_rows(x), *R.pack_rows(lin.weight.detach())))
    assert bool(torch.isfinite(y).all())


def test_strides():
    """Codes at any strides: rows off 16 bytes, transposed, broadcast, spread, at a buffer's end."""
    T, N, K = 37, 50, 100
    x, xs, w, ws = operands(T, N, K)
    want = flash_mhc.linear8(x, xs, w, ws)

    def spread(t):
        full = torch.zeros(t.shape[0], 2 * t.shape[1], dtype=torch.int8, device=DEV)
        full[:, ::2] = t
        return full[:, ::2]

    def at_end(t):  # the last row ends where the storage does
        n = (t.shape[0] - 1) * 112 + t.shape[1]
        return torch.empty(n, dtype=torch.int8, device=DEV).as_strided(t.shape, (112, 1)).copy_(t)

    def padded(t):
        full = torch.full((t.shape[0], 1024), 55, dtype=torch.int8, device=DEV)
        full[:, 16:16 + t.shape[1]] = t
        return full[:, 16:16 + t.shape[1]]

    for form in (torch.Tensor.contiguous, lambda t: t.t().contiguous().t(), spread, at_end, padded):
        assert torch.equal(flash_mhc.linear8(form(x), xs, form(w), ws), want)
    one = x[:1].expand(T, K)
    assert torch.equal(flash_mhc.linear8(one, xs[:1].expand(T), w, ws), want[:1].expand(T, N))
    lead = flash_mhc.linear8(x[:36].unflatten(0, (2, 3, 6)), xs[:36].view(2, 3, 6), w, ws)
    assert lead.shape == (2, 3, 6, N) and torch.equal(lead.reshape(36, N), want[:36])
    spaced = torch.zeros(2 * N, device=DEV)
    spaced[::2] = ws
    assert torch.equal(flash_mhc.linear8(x, xs, w, spaced[::2]), want)


def test_empty():
    w, ws = codes((5, 40), 1), torch.ones(5, device=DEV)
    assert flash_mhc.linear8(codes((0, 40), 0), torch.empty(0, device=DEV), w, ws).shape == (0, 5)
    q, s = flash_mhc.pack8_rows(torch.empty(0, 3, 40, device=DEV))
    assert q.shape == (0, 3, 40) and s.shape == (0, 3)
    assert flash_mhc.rms_norm_pack8_rows(torch.empty(0, 40, device=DEV))[0].shape == (0, 40)


def test_nothing_beside_the_output():
    lib = _abi.load()
    for T, N, K in ((1, 3, 5), (5, 17, 33), (70, 129, 40), (130, 300, 100), (300, 1025, 64)):
        x, xs, w, ws = operands(T, N, K)
        buf = torch.full((T * N + 512,), 7.0, device=DEV, dtype=BF16)
        assert lib.fmhc_linear8(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(), None,
                                None, buf[256:].data_ptr(), 1, 0, T, N, K, _abi.stream_of(x)) == 0
        assert torch.equal(buf[256:256 + T * N].view(T, N), flash_mhc.linear8(x, xs, w, ws))
        assert bool((buf[:256] == 7).all()) and bool((buf[256 + T * N:] == 7).all())


def test_large_offsets():
    """Outputs and codes past 2^32 bytes and 2^31 elements."""
    T, N, K = 70000, 33000, 16  # 2.3e9 outputs
    x, xs, w, ws = operands(T, N, K)
    out = flash_mhc.linear8(x, xs, w, ws)
    pick = torch.tensor([0, 1, 40000, 65535, 69998, 69999], device=DEV)
    check("rows", out[pick], *R.linear8(x[pick], xs[pick], w, ws))
    del out
    T, K = 1 << 20, 4352  # 4.6e9 codes
    x = torch.zeros(T, K, dtype=torch.int8, device=DEV)
    xs = torch.ones(T, device=DEV)
    last = codes((3, K), 9)
    x[-3:] = last
    w, ws = codes((20, K), 10), torch.ones(20, device=DEV) * 0.01
    out = flash_mhc.linear8(x, xs, w, ws)
    check("last", out[-3:], *R.linear8(last, xs[-3:], w, ws))
    assert float(out[:-3].abs().max()) == 0


def test_deterministic_on_two_streams():
    for T, N, K in ((3, 1024, 4096), (700, 520, 1024)):
        x, xs, w, ws = operands(T, N, K)
        want = flash_mhc.linear8(x, xs, w, ws)
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got += [flash_mhc.linear8(x, xs, w, ws) for _ in range(3)]
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(g, want) for g in got)


# ---------------------------------------------------------------------------
# The layer


def test_layer_is_the_product_of_its_rows():
    lin = torch.nn.Linear(1001, 300).to(DEV).to(BF16)
    layer = flash_mhc.Linear8.from_linear(lin)
    wq, ws = R.pack_rows(lin.weight.detach())
    assert torch.equal(layer.weight_codes[:, :1001].cpu(), wq) and torch.equal(layer.weight_scales.cpu(), ws)
    assert layer.weight_codes.shape == (300, 1008) and int(layer.weight_codes[:, 1001:].abs().max()) == 0
    for x in (rows(50, 1001), rows(6, 1001).view(2, 3, 1001)):
        q, s = R.pack_rows(x)
        with torch.no_grad():
            y = layer(x)
        assert y.shape == (*x.shape[:-1], 300) and y.dtype is BF16
        check("layer", y, *R.linear8(q, s, wq, ws, lin.bias.detach()))


def test_layer_in_64_bits_packs_the_same_rows():
    """Off the kernels the layer packs its rows as they do."""
    for dtype in (BF16, F16, F32):
        x = rows(200, 1000, dtype)
        q, s = flash_mhc.rows8._plain_rows(x.double())
        want = flash_mhc.pack8_rows(x)
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])


def test_layer_in_64_bits_has_no_gradient():
    layer = flash_mhc.Linear8.from_linear(torch.nn.Linear(100, 7)).to(DEV)
    x = rows(5, 100, F32)
    for leaf in (x.double().requires_grad_(True), x.clone().requires_grad_(True)):
        out = layer(leaf)
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="has no gradient"):
            out.sum().backward()


@pytest.mark.parametrize("T", [3, 40, 700])
@pytest.mark.parametrize("dtype,kept", [(F16, BF16), (BF16, F16), (BF16, torch.float64), (F32, BF16)])
def test_bias_of_another_type(T, dtype, kept):
    """A bias is added in its own bits, before the one rounding: 99840 in bf16 is past fp16's range, and the sum is not."""
    x = rnd((T, 500), 1, dtype=dtype).to(DEV)
    x[:, 0] = 50
    w = rnd((300, 500), 2, 0.04, dtype=F32)
    w[:, 0] = -1000
    lin = torch.nn.Linear(500, 300).to(kept)
    with torch.no_grad():
        lin.weight.copy_(w)
        lin.bias.copy_(rnd((300,), 3, 1.0, 1000.0, F32))
        if kept is BF16:
            lin.bias[::3] = 99840
        layer = flash_mhc.Linear8.from_linear(lin).to(DEV)
        assert layer.bias.dtype is kept
        y = layer(x)
    wq, ws = R.pack_rows(lin.weight.detach().float())
    check("layer", y, *R.linear8(*R.pack_rows(x), wq, ws, lin.bias.detach().float()))
    assert bool(torch.isfinite(y).all())


def _block(C, norm="rms", bias=True, seed=0):
    torch.manual_seed(seed)
    lin = torch.nn.Linear(C, C, bias=bias)
    blk = flash_mhc.MHCLiteBlock(4, C, flash_mhc.Linear8.from_linear(lin.to(DEV).to(BF16)), pre_norm=norm)
    blk = blk.to(DEV).to(BF16).eval()
    with torch.no_grad():
        blk.alpha_pre.fill_(0.8)
        blk.alpha_post.fill_(1.2)
        blk.norm.weight.copy_(rnd((C,), 3, 0.2, 1.0))
    return blk


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("T,C", [(1, 256), (40, 1024), (300, 520), (70, 300)])
def test_block(T, C, norm):
    """The block's layer is u + F(norm(u)): the norm's rows in 8 bits, the product with u."""
    blk = _block(C, norm)
    x = rnd((T, 4, C), 5).to(DEV)
    with torch.no_grad():
        out = blk(x)
        li, H, hq, *_ = torch.ops.flash_mhc.mhc_pre_map(x, blk.W_all.weight, blk.alpha_pre, blk.alpha_post,
                                                        blk.alpha_res, blk.W_all.bias, blk.perm_mat)
        if norm == "rms":
            q, s = flash_mhc.rms_norm_pack8_rows(li, blk.norm.weight, blk.norm.eps)
        else:
            q, s = flash_mhc.pack8_rows(flash_mhc.layer_norm(li, blk.norm.weight, blk.norm.bias, blk.norm.eps))
        layer = blk.layer
        lo = flash_mhc.linear8(q, s, layer.weight_codes[:, :C], layer.weight_scales, layer.bias, residual=li)
        check("lo", lo, *R.linear8(q, s, layer.weight_codes[:, :C], layer.weight_scales, layer.bias, li))
        assert torch.equal(out, torch.ops.flash_mhc.fused_post_res(x, lo, H, hq))


@pytest.mark.parametrize("kw", [{"activation_bits": 8}, {"activation_checkpointing": True}, {"triton_fused": False}])
def test_block_with_its_options(kw):
    """What concerns the backward changes no inference; the plain formulation rounds the layer's input elsewhere."""
    blk, x = _block(256), rnd((30, 4, 256), 5).to(DEV)
    other = flash_mhc.MHCLiteBlock(4, 256, blk.layer, pre_norm="rms", **kw).to(DEV).to(BF16).eval()
    other.load_state_dict(blk.state_dict())
    with torch.no_grad():
        want, got = blk(x), other(x)
    if kw.get("triton_fused", True):
        assert torch.equal(got, want)
    else:
        assert float((got.float() - want.float()).norm()) <= 2.0 ** -6 * float(want.float().norm())


@pytest.mark.parametrize("dtype", [F16, F32])
def test_block_in_other_types(dtype):
    """Where the streams take the plain formulation, the layer is the same two calls."""
    blk = _block(264).to(dtype)
    u = rnd((21, 264), 5, dtype=dtype).to(DEV)
    with torch.no_grad():
        q, s = flash_mhc.rms_norm_pack8_rows(u, blk.norm.weight, blk.norm.eps)
        layer = blk.layer
        want = flash_mhc.linear8(q, s, layer.weight_codes[:, :264], layer.weight_scales, layer.bias, residual=u, dtype=dtype)
        assert layer.weight_scales.dtype is F32 and want.dtype is dtype
        assert torch.equal(blk._apply_layer(u, {}), want)
        assert bool(torch.isfinite(blk(rnd((21, 4, 264), 6, dtype=dtype).to(DEV))).all())


def test_strided_rows_compiled():
    x = rows(40, 264).t().contiguous().t()
    f = lambda x: flash_mhc.linear8(*flash_mhc.pack8_rows(x), *flash_mhc.rms_norm_pack8_rows(x), dtype=F32)
    assert torch.equal(torch.compile(f, fullgraph=True)(x), f(x))


def test_block_with_hooks():
    """A hooked layer or norm is called: the same up to the rounding of what passes between."""
    blk = _block(256)
    x = rnd((30, 4, 256), 5).to(DEV)
    with torch.no_grad():
        want = blk(x)
        for module in (blk.layer, blk.norm):
            calls = []
            handle = module.register_forward_hook(lambda *a: calls.append(1))
            out = blk(x)
            handle.remove()
            assert calls == [1]
            assert float((out.float() - want.float()).norm()) <= 2.0 ** -6 * float(want.float().norm())
        assert torch.equal(blk(x), want)


def test_block_against_its_16_bit_layer():
    """8 bits beside the layer in bf16: each of the two operands is off by at most half a
    scale (uniformly: scale / sqrt(12)), a scale being a 127th of the row's maximum, 3 to 4.5
    times its spread: 4.5 / 127 / sqrt(12) = 1.0% each, 1.5% of the layer's output in all,
    which the block adds to its residual."""
    C = 1024
    blk = _block(C, bias=False)
    ref = _block(C, bias=False)
    ref.layer = torch.nn.Linear(C, C, bias=False, device=DEV, dtype=BF16)
    with torch.no_grad():
        ref.layer.weight.copy_(blk.layer.weight_codes.float() * blk.layer.weight_scales.unsqueeze(-1))
        x = rnd((200, 4, C), 5).to(DEV)
        a, b = blk(x).float(), ref(x).float()
    assert float((a - b).norm()) <= 0.015 * float(b.norm())


def test_captured_block():
    blk = _block(1024)
    xs = [rnd((48, 4, 1024), 50).to(DEV), rnd((1, 4, 1024), 51).to(DEV)]
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for x in xs:
                blk(x)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for x in xs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(blk(x))
            graphs.append(graph)
        for k in range(3):
            for x in xs:
                x.copy_(rnd(tuple(x.shape), 60 + k))
            want = [blk(x).clone() for x in xs]
            torch.cuda.synchronize()
            for graph, out, w in zip(graphs, outs, want):
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, w), k


def test_compiled_block():
    blk = _block(256)
    x = rnd((30, 4, 256), 5).to(DEV)
    torch._dynamo.reset()
    with torch.no_grad():
        want = blk(x)
        out = torch.compile(blk, fullgraph=True)(x)
    assert torch.equal(out, want)


def test_rms_block_trains():
    """pre_norm="rms" with a 16-bit layer, eager and through the ops: the same bits."""
    torch.manual_seed(0)
    blk = flash_mhc.MHCLiteBlock(4, 256, torch.nn.Linear(256, 256), pre_norm="rms").to(DEV).to(BF16)
    x = rnd((70, 4, 256), 5).to(DEV)
    g = rnd((70, 4, 256), 6).to(DEV)

    def step(f):
        leaf = x.clone().requires_grad_(True)
        out = f(leaf)
        return [out.detach(), *torch.autograd.grad(out, [leaf, *blk.parameters()], g)]

    eager = step(blk)
    # norm(u) + u as two uses of u in the graph: x's gradients there are rounded once more.
    handle = blk.norm.register_forward_hook(lambda *a: None)
    hooked = step(blk)
    handle.remove()
    assert torch.equal(eager[0], hooked[0])
    for a, b in zip(eager[1:], hooked[1:]):
        assert float((a.float() - b.float()).norm()) <= 2.0 ** -6 * float(b.float().norm())
