"""Row-wise quantisation, alone and behind the RMS norm with the residual's addition, against the definition in 64 bits.

Tolerances, from the formulas.  The scale is max|s w| * rstd / Q in fp32: the sum s, the product s w, the sum of
squares (relative error below 2**-20 for any order of up to 2**15 positive terms a thread-and-tree sum adds here), the
root, two products and a division, each 2**-24: 2**-19 in all.  A code is round((s w) * (Q / max|s w|)) with five fp32
roundings in front of it, so before its own rounding it is within 5 * 2**-24 of the exact quotient (relative), and the
code is an 8-bit neighbour of the exact code only where the quotient lies that close to a tie: with one more half step
(e4m3 2**-4 relative above the subnormals, 2**-10 absolute below; int8 0.5) codes * scale is within
half a step + 2**-18 of y / scale."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

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


def check_codes(codes, scales, y):
    """codes * scales against y in 64 bits."""
    top = TOP[codes.dtype]
    want = y.abs().amax(-1, keepdim=True) / top
    assert scales.dtype == torch.float32 and scales.shape == want.shape
    torch.testing.assert_close(scales.double(), want.clamp_min(TINY), rtol=2.0**-19, atol=0)
    q, exact = codes.double(), y / want.clamp_min(TINY)
    half = torch.full_like(exact, 0.5) if codes.dtype == torch.int8 else (exact.abs() * 2.0**-4).clamp_min(2.0**-10)
    off = (q - exact).abs() - half - exact.abs() * 2.0**-18
    assert off.max().item() <= 0, f"a code is {off.max().item()} beyond half a step"


def norm64(x, weight, residual, eps):
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


@pytest.mark.parametrize("out_dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (1, 8), (5, 64), (2, 4096), (3, 4099), (33, 5003), (2, 8200), (2, 14336), (2, 32768), (2, 32761), (3, 40000), (2, 50001),
                                 (592, 1024), (1700, 1031), (900, 4096), (601, 5003), (777, 9000), (650, 14336), (593, 16377), (600, 16384), (2401, 14336), (8200, 4096)])
def test_quantize_rows(hb, m, n, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(m * 100003 + n)
    x = (torch.randn(m, n, generator=g, device="cuda") * 3.0).to(dtype)
    codes, scales = hb.quantize_rows(x, out_dtype=out_dtype)
    assert codes.dtype == out_dtype and codes.shape == x.shape and codes.is_contiguous()
    check_codes(codes, scales, x.double())
    again = hb.quantize_rows(x, out_dtype=out_dtype)
    assert torch.equal(codes.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scales, again[1])


@pytest.mark.parametrize("with_residual", [True, False], ids=["residual", "plain"])
@pytest.mark.parametrize("out_dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("m,n", [(1, 1), (2, 9), (1, 4096), (7, 5003), (2, 14336), (2, 24576), (2, 40001), (1190, 1031), (900, 4096), (601, 5003), (601, 8192), (650, 14336), (593, 16377), (600, 16384), (4099, 4096)])
def test_rms_norm_quantize(hb, m, n, dtype, w_dtype, out_dtype, with_residual):
    g = torch.Generator(device="cuda").manual_seed(m * 100003 + n + 1)
    x = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    r = (torch.randn(m, n, generator=g, device="cuda") * 5.0).to(dtype) if with_residual else None
    w = (1.0 + 0.3 * torch.randn(n, generator=g, device="cuda")).to(w_dtype)
    got = hb.rms_norm_quantize(x, w, residual=r, eps=1e-5, out_dtype=out_dtype)
    s, y = norm64(x, w, r, 1e-5)
    check_codes(got[0], got[1], y)
    if with_residual:
        assert torch.equal(got[2], (x.float() + r.float()).to(dtype))  # one fp32 sum, rounded once
    else:
        assert len(got) == 2


def test_leading_dimensions_and_given_buffers(hb):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 3, 136, generator=g, device="cuda").bfloat16()
    r = torch.randn(2, 3, 136, generator=g, device="cuda").bfloat16()
    w = torch.rand(136, generator=g, device="cuda").bfloat16()
    want = hb.rms_norm_quantize(x.reshape(6, 136), w, residual=r.reshape(6, 136))
    got = hb.rms_norm_quantize(x, w, residual=r)
    assert [tuple(t.shape) for t in got] == [(2, 3, 136), (2, 3, 1), (2, 3, 136)]
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))
    one = hb.quantize_rows(x[0, 0])
    assert one[0].shape == (136,) and one[1].shape == (1,)
    # in place on the residual, then on x, with every result in the caller's buffers
    for target in ("residual", "x"):
        x2, r2 = x.clone(), r.clone()
        bufs = torch.empty_like(x, dtype=E4M3), torch.empty(2, 3, 1, device="cuda")
        back = hb.rms_norm_quantize(x2, w, residual=r2, out=bufs[0], scale_out=bufs[1], residual_out=r2 if target == "residual" else x2)
        assert back[0] is bufs[0] and back[1] is bufs[1] and back[2] is (r2 if target == "residual" else x2)
        for a, b in zip(back, got):
            assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("m,n", [(3, 40003), (3, 520), (3, 77), (1500, 1031), (1500, 4096), (700, 8200)])
def test_in_place_on_rows_of_every_kind(hb, m, n):
    """Rows read twice (n > 32768), whole and odd, few and many: the sum overwrites an input that is still being read."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x, r = (torch.randn(m, n, generator=g, device="cuda").half() for _ in range(2))
    w = torch.rand(n, generator=g, device="cuda").half()
    want = hb.rms_norm_quantize(x, w, residual=r)
    got = hb.rms_norm_quantize(x, w, residual=r, residual_out=r)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_strided_and_offset_rows(hb):
    """Rows with a stride, rows that start off every vector boundary, tensors that start apart from one another,
    overlapping (expanded) rows and columns with a stride give what contiguous copies give."""
    g = torch.Generator(device="cuda").manual_seed(6)
    wide = torch.randn(9, 1000, generator=g, device="cuda").bfloat16()
    res = torch.randn(9, 1001, generator=g, device="cuda").bfloat16()
    w = torch.rand(1000, generator=g, device="cuda").bfloat16()
    views = [(wide[:, 0:512], res[:, 0:512], w[0:512]), (wide[:, 3:603], res[:, 3:603], w[5:605]), (wide[:, 8:208], res[:, 1:201], w[1:201]),
             (wide[:, ::2], res[:, 1::2], w[::2]), (wide[:1].expand(4, 1000), res[:4, :1000], w), (wide.t()[:9, :9], res.t()[:9, :9], w[:9])]
    for x, r, wt in views:
        got = hb.rms_norm_quantize(x, wt, residual=r)
        want = hb.rms_norm_quantize(x.contiguous(), wt.contiguous(), residual=r.contiguous())
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))
        check_codes(*got[:2], norm64(x, wt, r, 1e-6)[1])
        check_codes(*hb.quantize_rows(x, out_dtype=torch.int8), x.double())
    # many rows with strides and offsets
    big = torch.randn(700, 2100, generator=g, device="cuda").bfloat16()
    w = torch.rand(2100, generator=g, device="cuda")
    for x, r, wt in ((big.view(175, -1)[:, 8:8200].repeat(4, 1)[:, :8192], big.view(175, -1)[:, :8192].repeat(4, 1), torch.rand(8192, generator=g, device="cuda")),
                     (big[:, 8:2056], big[:, 0:2048], w[:2048]), (big[:, 3:2052], big[:, 11:2060], w[:2049]), (big[:, 3:2052], big[:, 4:2053], w[:2049])):
        got = hb.rms_norm_quantize(x, wt, residual=r)
        check_codes(*got[:2], norm64(x, wt, r, 1e-6)[1])  # the order of a row's sum goes by its layout: not the same bits
        assert torch.equal(got[2], (x.float() + r.float()).bfloat16())
        check_codes(*hb.quantize_rows(x, out_dtype=torch.int8), x.double())
    # a phased row next to guard values: nothing outside the row is written
    store = torch.full((4 * 77 + 32,), 7, dtype=torch.int8, device="cuda")
    out = store[16 : 16 + 4 * 77].view(4, 77)
    hb.quantize_rows(torch.randn(4, 77, generator=g, device="cuda").half(), out_dtype=torch.int8, out=out)
    assert (store[:16] == 7).all() and (store[16 + 4 * 77 :] == 7).all()


def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite(hb):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(6, 40, device="cuda")
    x[1, 3] = 2.0**-101
    x[2, 3] = -3.0
    x[3, 3] = nan
    x[4, 3] = inf
    x[5, :] = 3e38
    for out_dtype in (E4M3, torch.int8):
        codes, scales = hb.quantize_rows(x, out_dtype=out_dtype)
        c, s = codes.double(), scales.double()
        assert (c[:2] == 0).all() and (s[:2] == TINY).all()
        assert c[2, 3] == -TOP[out_dtype] and (c[2, 4:] == 0).all()
        assert s[3].isnan().all() and s[4].item() == inf
        torch.testing.assert_close((c[5] * s[5]), x[5].double(), rtol=2.0**-20, atol=0)
        # behind the norm: a row of zeros stays one
        w = torch.ones(40, device="cuda")
        codes, scales = hb.rms_norm_quantize(x, w, eps=1e-6, out_dtype=out_dtype)
        assert (codes[0].double() == 0).all() and scales[0].item() == pytest.approx(TINY)
        assert scales[3:].isnan().all()  # a NaN, an infinity, and a sum of squares beyond fp32
        # squares that underflow: the root is eps's
        small = torch.full((2, 40), 1e-25, device="cuda")
        codes, scales = hb.rms_norm_quantize(small, w, eps=1e-30, out_dtype=out_dtype)
        check_codes(codes, scales, norm64(small, w, None, 1e-30)[1])
    # one infinite or NaN row leaves the others as they were
    for m, n in ((3, 256), (1001, 1024)):
        y = torch.randn(m, n, device="cuda").bfloat16()
        want = hb.quantize_rows(y)
        y2 = y.clone()
        y2[1, 100] = nan
        got = hb.quantize_rows(y2)
        assert got[1][1].isnan().all()
        rest = [i for i in range(m) if i != 1]
        assert torch.equal(got[0].view(torch.uint8)[rest], want[0].view(torch.uint8)[rest]) and torch.equal(got[1][rest], want[1][rest])


def test_the_first_call_of_a_process_may_be_captured(hb):
    code = """
import torch, helion_b200 as hb
x = torch.randn(2, 1024, device="cuda")
w = torch.randint(-128, 128, (2, 256, 1024), device="cuda", dtype=torch.int8)
def calls():
    codes, scales = hb.quantize_rows(x, out_dtype=torch.int8)
    s = scales.new_ones(1, 256)
    few = hb.int8_gemm(codes, w[0].t(), scale_a=scales, scale_b=s, out_dtype=torch.float32)
    gated = hb.gated_gemm(codes, w[0].t(), w[1].t(), scale_x=scales, scale_gate=s, scale_up=s, out_dtype=torch.float32)
    many = hb.int8_gemm(w[0], w[1].t(), out_dtype=torch.float32)
    return codes, scales, few, gated, many
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(__file__).resolve().parent.parent, timeout=300)


def test_offsets_beyond_31_bits(hb):
    """The last rows of a matrix of 2.3e9 values are what they are on their own."""
    m, n = 70000, 32776
    x = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, n, device="cuda").bfloat16()
    x[70] = 5.0
    codes, scales = hb.quantize_rows(x)
    want = hb.quantize_rows(x[-3:].clone())
    assert torch.equal(codes[-3:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales[-3:], want[1])
    assert (codes[70].float() == 448).all() and scales[71].item() == pytest.approx(TINY)
    del codes, scales
    m, n = 140000, 16384  # many rows: through the ring
    x = x.view(-1)[: m * n].view(m, n)
    x[-1] = torch.randn(n, device="cuda").bfloat16()
    codes, scales = hb.quantize_rows(x)
    want = hb.quantize_rows(x[-1:].clone())
    assert torch.equal(codes[-1:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales[-1:], want[1])


def test_empty_inputs(hb):
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16)
    codes, scales = hb.quantize_rows(x)
    assert codes.shape == (0, 64) and scales.shape == (0, 1) and codes.dtype == E4M3
    got = hb.rms_norm_quantize(x, torch.ones(64, device="cuda", dtype=torch.bfloat16), residual=x)
    assert [tuple(t.shape) for t in got] == [(0, 64), (0, 1), (0, 64)]
    with pytest.raises(ValueError, match="at least one value"):
        hb.quantize_rows(torch.zeros(4, 0, device="cuda"))


def test_another_stream_and_a_captured_graph(hb):
    g = torch.Generator(device="cuda").manual_seed(8)
    x, r = (torch.randn(300, 4096, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.rand(4096, generator=g, device="cuda").bfloat16()
    want = hb.rms_norm_quantize(x, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hb.rms_norm_quantize(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    xs = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = hb.rms_norm_quantize(xs, w, residual=r)
    xs.copy_(x)
    graph.replay()
    for a, b, c in zip(got, want, held):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(c.view(torch.uint8), b.view(torch.uint8))
