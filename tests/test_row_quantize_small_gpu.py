"""Rows behind the norm whose values are tiny but whose normalised values are not."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
TOP = {E4M3: 448.0, torch.int8: 127.0}
TINY = torch.finfo(torch.float32).tiny


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


@pytest.mark.parametrize("out_dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("with_residual", [True, False], ids=["residual", "plain"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,n", [(40, 136), (40, 77), (40, 40003), (8192, 4096), (2048, 8192)])
def test_tiny_rows_behind_the_norm(hb, m, n, dtype, with_residual, out_dtype):
    """s of 2**-72 down to 2**-112 with eps 2**-100 or 2**-120 gives y between 2**-22 and 2**-62 (the squares underflow or vanish
    next to eps): none is a row of zeros.  s and w are bf16 numbers of few bits, so s w is exact and normal in fp32.  As for any
    other row the scale is within 2**-19 and a code within half a step and 2**-18 relative."""
    g = torch.Generator(device="cuda").manual_seed(n)
    for power, eps in ((-75, 2.0**-100), (-101, 2.0**-100), (-115, 2.0**-100), (-115, 2.0**-120)):
        s = torch.randint(-8, 9, (m, n), generator=g, device="cuda").double() * 2.0**power
        s[:, 3] = 8 * 2.0**power
        w = (torch.randint(4, 8, (n,), generator=g, device="cuda").double() / 4).to(dtype)
        x = (s / 2).to(dtype) if with_residual else s.to(dtype)
        codes, scales = hb.rms_norm_quantize(x, w, residual=x if with_residual else None, eps=eps, out_dtype=out_dtype)[:2]
        y = s / (s.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
        top = y.abs().amax(1, keepdim=True)
        torch.testing.assert_close(scales.double(), top / TOP[out_dtype], rtol=2.0**-19, atol=0)
        exact = y / top * TOP[out_dtype]
        half = torch.full_like(exact, 0.5) if out_dtype == torch.int8 else (exact.abs() * 2.0**-4).clamp_min(2.0**-10)
        assert ((codes.double() - exact).abs() <= half + exact.abs() * 2.0**-18).all()


def test_rows_of_zeros_are_told_by_their_normalised_values(hb):
    """A row whose largest |y| is below 2**-100 counts as a row of zeros: zero codes and the smallest normal scale."""
    x = torch.zeros(3, 40, device="cuda")
    x[1, 5], x[2, 5] = 2.0**-120, 2.0**-120
    w = torch.ones(40, device="cuda")
    for out_dtype in (E4M3, torch.int8):
        codes, scales = hb.rms_norm_quantize(x, w, eps=2.0**-30, out_dtype=out_dtype)  # |y| = 2**-105
        assert (codes.double() == 0).all() and (scales == TINY).all()
        codes, scales = hb.rms_norm_quantize(x, w, eps=2.0**-50, out_dtype=out_dtype)  # |y| = 2**-95
        assert codes[1:, 5].double().tolist() == [TOP[out_dtype]] * 2 and (codes.double() != 0).sum().item() == 2
        assert scales[0].item() == pytest.approx(TINY)
        torch.testing.assert_close(scales[1:].double(), torch.full((2, 1), 2.0**-95 / TOP[out_dtype], device="cuda", dtype=torch.float64), rtol=2.0**-19, atol=0)
