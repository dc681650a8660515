"""The codes of exact ties, code for code.

A code is round_to_nearest_even(x Q / max|x|), behind the norm round_to_nearest_even(s w Q / max|s w|) (1 / sqrt of the mean
square is common to both).  The values here are such that x Q and s w Q are exact in 64 bits.  A quotient that is not a tie is
at least 2**-21 (relative) away from one: x Q - tie max is a whole multiple of the last place of a product of at most 11 + 11
bits.  So one division in 64 bits, which is exact for a tie, decides every code, and every code has to be that one."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
TOP = {E4M3: 448.0, torch.int8: 127.0}


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def exact_codes(y, out_dtype):
    """Codes of rows whose products with Q are exact in 64 bits, as numbers."""
    q = y * TOP[out_dtype] / y.abs().amax(-1, keepdim=True)
    return q.round() if out_dtype == torch.int8 else q.float().to(E4M3).double()


def rows_of_maxima(g, m, n, dtype):
    """Rows whose largest magnitudes run through a binade's significands (times a few powers of two), among values of
    `dtype` spread over the binades below it, and among the values nearest to the row's tie points (many are ties); the
    first values are +-max/2 and max."""
    bits = 10 if dtype == torch.float16 else 7  # significands of bf16 for fp32 rows too
    steps = 2**bits
    top = 1.0 + torch.arange(m, device="cuda").remainder(steps).double().reshape(m, 1) / steps
    sig = 1.0 + torch.randint(0, steps, (m, n), generator=g, device="cuda").double() / steps
    x = sig * torch.exp2(-torch.randint(1, 7, (m, n), generator=g, device="cuda").double())
    x = torch.where(torch.rand(m, n, generator=g, device="cuda") < 0.5, -x, x)
    x = torch.where(x.abs() <= top, x, x / 2)
    # the tie points themselves: (k + 0.5) / 127 of the maximum for int8, odd multiples of half a step for e4m3
    tie8 = (torch.randint(0, 127, (m, n), generator=g, device="cuda").double() + 0.5) / 127.0 * top
    tie4 = (torch.randint(8, 15, (m, n), generator=g, device="cuda").double() * 2 + 1) * torch.exp2(torch.randint(0, 5, (m, n), generator=g, device="cuda").double()) / 448.0 * top
    pick = torch.randint(0, 3, (m, n), generator=g, device="cuda")
    x = torch.where(pick == 1, tie8, torch.where(pick == 2, tie4, x))
    x[:, 0], x[:, 1], x[:, 2:3] = top[:, 0] / 2, -top[:, 0] / 2, top
    scale = torch.exp2(torch.randint(-12, 9, (m, 1), generator=g, device="cuda").double()) if dtype != torch.float16 else 1.0
    x = (x * scale).to(torch.float16 if dtype == torch.float16 else torch.bfloat16).to(dtype)
    return torch.where(x.abs() <= x[:, 2:3], x, x[:, 2:3])  # rounding to dtype may have passed the maximum


@pytest.mark.parametrize("out_dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n", [(1024, 520), (1024, 1031), (130, 8192), (128, 40003), (8192, 4096)])
def test_codes_of_ties(hb, m, n, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = rows_of_maxima(g, m, n, dtype)
    codes, scales = hb.quantize_rows(x, out_dtype=out_dtype)
    wrong = (codes.double() != exact_codes(x.double(), out_dtype)).sum().item()
    assert wrong == 0, f"{wrong} of {x.numel()} codes"
    torch.testing.assert_close(scales.double(), x.double().abs().amax(1, keepdim=True) / TOP[out_dtype], rtol=2.0**-23, atol=0)


def test_a_pair_of_ties_by_hand(hb):
    """2.734375 * 448 / 3.0625 = 400, between the codes 384 and 416 (even: 384); 1.1875 * 127 / 2.375 = 63.5 (even: 64)."""
    x = torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16)
    x[0, :2] = torch.tensor([3.0625, 2.734375])
    x[1, :2] = torch.tensor([2.375, 1.1875])
    assert hb.quantize_rows(x)[0][0, :2].tolist() == [448, 384]
    assert hb.quantize_rows(x, out_dtype=torch.int8)[0][1, :2].tolist() == [127, 64]


@pytest.mark.parametrize("out_dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("with_residual", [True, False], ids=["residual", "plain"])
@pytest.mark.parametrize("m,n", [(1024, 520), (1024, 1031), (8192, 4096)])
def test_codes_of_ties_behind_the_norm(hb, m, n, with_residual, out_dtype):
    """Weights of +-1 keep s w exact, and halves as x and residual the sum."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    s = rows_of_maxima(g, m, n, torch.bfloat16)
    w = torch.randint(0, 2, (n,), generator=g, device="cuda").bfloat16() * 2 - 1
    x, r = (s / 2, s / 2) if with_residual else (s, None)
    codes = hb.rms_norm_quantize(x, w, residual=r, out_dtype=out_dtype)[0]
    wrong = (codes.double() != exact_codes(s.double() * w.double(), out_dtype)).sum().item()
    assert wrong == 0, f"{wrong} of {s.numel()} codes"
