"""Layer norm of more rows than one launch has threads for (2^31 rows of 8 columns and more)."""

from __future__ import annotations

import pytest
import torch

import flash_mhc

pytestmark = pytest.mark.gpu

BF16, DEV = torch.bfloat16, "cuda"


@pytest.mark.parametrize("bits", [16, 8])
def test_rows_past_2_31(bits):
    """Copies of the same rows have the same results, the last ones too."""
    C, n, reps = 8, 1 << 21, 1025
    assert n * reps > 1 << 31
    if torch.cuda.mem_get_info()[1] < 250 << 30:
        pytest.skip("needs 250 GiB")
    g = torch.Generator().manual_seed(1)
    part, up = (torch.randn(n, C, generator=g).to(BF16).to(DEV) for _ in range(2))
    w, b = (torch.randn(C, generator=g).to(DEV) for _ in range(2))
    want = flash_mhc.layer_norm(part, w, b)

    def check(got, want):
        assert got.shape == (n * reps, C)
        for piece in got.view(reps, n, C):
            assert torch.equal(piece, want)

    x = part.repeat(reps, 1)
    with torch.no_grad():
        y = flash_mhc.layer_norm(x, w, b)
    check(y, want)
    del y
    ref = part.clone().requires_grad_(True)
    (ref_grad,) = torch.autograd.grad(flash_mhc.layer_norm(ref, w, b, activation_bits=bits), ref, up)
    y = flash_mhc.layer_norm(x.requires_grad_(True), w, b, activation_bits=bits)
    check(y.detach(), want)
    (gx,) = torch.autograd.grad(y, x, up.repeat(reps, 1))
    del y, x
    check(gx, ref_grad)
    del gx
    torch.cuda.empty_cache()
