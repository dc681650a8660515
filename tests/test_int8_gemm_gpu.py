"""int8 GEMM with token and channel scales against the definition in 64 bits.

The integer sums are exact.  One conversion to fp32 and two fp32 products (each 2**-24 relative) precede the output's
own rounding (half a step: bf16 2**-8, fp16 2**-11, fp32 2**-24), so a result is within half a step + 3 * 2**-24, and
unscaled fp32 results of sums below 2**24 are exact."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def check(out, x, y, sa=None, sb=None):
    want = x.double() @ y.double()
    if sa is not None:
        want = want * sa.double().reshape(-1, 1) * sb.double().reshape(1, -1)
    torch.testing.assert_close(out.double(), want, rtol=HALF_STEP[out.dtype] + 3 * 2.0**-24, atol=2.0**-25 if out.dtype == torch.float16 else 0)


@pytest.mark.parametrize("out_dtype", list(HALF_STEP), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 4096, 256), (16, 14336, 144), (17, 1000, 2048), (33, 24, 4096), (64, 19000, 128), (65, 520, 272),
                                   (128, 4224, 2048), (100, 4232, 2064), (7, 9472, 1024), (3, 72, 14336), (128, 9480, 528), (128, 128, 128), (129, 136, 144), (300, 1000, 1040), (1024, 2048, 512), (777, 5000, 2064)])
def test_scaled_products(hb, m, n, k, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, y = codes(g, m, k), codes(g, n, k).t()
    sa = torch.rand(m, 1, generator=g, device="cuda") * 1e-3
    sb = torch.rand(1, n, generator=g, device="cuda") * 1e-3 + 1e-4
    check(hb.int8_gemm(x, y, scale_a=sa, scale_b=sb, out_dtype=out_dtype), x, y, sa, sb)
    one = torch.full((1,), 3e-6, device="cuda")
    check(hb.int8_gemm(x, y, scale_a=one, scale_b=one * 2, out_dtype=out_dtype), x, y, one.expand(m), (one * 2).expand(n))
    if out_dtype != torch.float16:
        out = hb.int8_gemm(x, y, out_dtype=out_dtype)
        check(out, x, y)
        if out_dtype == torch.float32 and k * 128 * 128 < 1 << 24:
            assert torch.equal(out.double(), x.double() @ y.double())


@pytest.mark.parametrize("m,n,k", [(129, 1024, 4096), (130, 4096, 14336), (192, 9000, 16384), (256, 520, 8192), (257, 33, 8208), (513, 2048, 8200), (700, 1536, 12304), (1023, 512, 6160), (2049, 72, 4112)])
def test_more_rows_with_long_k_and_few_columns(hb, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, y = codes(g, m, k), codes(g, n, k).t()
    sa, sb = (torch.rand(c, generator=g, device="cuda") * 1e-3 + 1e-6 for c in (m, n))
    for out_dtype in (torch.bfloat16, torch.float32):
        store = torch.full((m + 3, n + 8), 5.0, device="cuda", dtype=out_dtype)
        check(hb.int8_gemm(x, y, scale_a=sa, scale_b=sb, out_dtype=out_dtype, out=store[:m, :n]), x, y, sa, sb)
        assert (store[m:] == 5).all() and (store[:, n:] == 5).all()
    check(hb.int8_gemm(x, y, out_dtype=torch.float32), x, y)
    assert torch.equal(hb.int8_gemm(x, y, scale_a=sa, scale_b=sb), hb.int8_gemm(x, y, scale_a=sa, scale_b=sb, config=1))


@pytest.mark.parametrize("row", [0, 1, 2, 3, 6, 7, 10, 14, 17, 18, 21])
def test_every_table_row_gives_the_same_bits(hb, row):
    g = torch.Generator(device="cuda").manual_seed(row)
    m = 100 if row == 18 else 700
    x, y = codes(g, m, 1552), codes(g, 1304, 1552).t()
    sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(1304, generator=g, device="cuda")
    want = (x.double() @ y.double()).float() * sa[:, None] * sb[None, :]  # sums below 2**24: exact in fp32
    assert torch.equal(hb.int8_gemm(x, y, scale_a=sa, scale_b=sb, out_dtype=torch.float32, config=row), want)


def test_largest_sums(hb):
    """-128 * -128 over the longest K there is: 2**31 - 2**18, still int32."""
    k = 131056
    for m in (3, 200):
        x = torch.full((m, k), -128, device="cuda", dtype=torch.int8)
        y = torch.full((8, k), -128, device="cuda", dtype=torch.int8).t()
        assert (hb.int8_gemm(x, y, out_dtype=torch.float32) == float(k * 128 * 128)).all()
        y = torch.full((8, k), 127, device="cuda", dtype=torch.int8).t()
        check(hb.int8_gemm(x, y, out_dtype=torch.float32), x, y)


@pytest.mark.parametrize("m", [1, 40, 130])
@pytest.mark.parametrize("n,k", [(33, 17), (1001, 250), (16, 16), (5, 1)])
def test_odd_sizes_layouts_and_given_outputs(hb, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m * n + k)
    x, y = codes(g, m, k), codes(g, k, n)
    sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    want = (x.double() @ y.double()).float() * sa[:, None] * sb[None, :]
    wide = codes(g, m, 2 * k + 3)
    wide[:, 1 : k + 1] = x
    for xx in (x, x.t().contiguous().t(), wide[:, 1 : k + 1]):
        for yy in (y, y.t().contiguous().t()):
            assert torch.equal(hb.int8_gemm(xx, yy, scale_a=sa, scale_b=sb, out_dtype=torch.float32), want)
    out = torch.empty(m, n, device="cuda")
    assert hb.int8_gemm(x, y, scale_a=sa, scale_b=sb, out_dtype=torch.float32, out=out) is out and torch.equal(out, want)


def test_rows_behind_the_last_are_left_alone(hb):
    g = torch.Generator(device="cuda").manual_seed(11)
    for m in (5, 140):
        store = torch.full((m + 8, 264), 9.0, device="cuda", dtype=torch.bfloat16)
        x, y = codes(g, m, 512), codes(g, 256, 512).t()
        hb.int8_gemm(x, y, out=store[:m, :256])
        check(store[:m, :256], x, y)
        assert (store[m:] == 9).all() and (store[:, 256:] == 9).all()


def test_offsets_beyond_31_bits(hb):
    g = torch.Generator(device="cuda").manual_seed(14)
    m, n = 70000, 32776
    x, y = codes(g, m, 16), codes(g, n, 16).t()
    out = hb.int8_gemm(x, y)
    check(out[-300:], x[-300:], y)
    check(out[:5], x[:5], y)


def test_empty_dimensions(hb):
    z = lambda *s: torch.zeros(s, device="cuda", dtype=torch.int8)  # noqa: E731
    assert hb.int8_gemm(z(0, 32), z(32, 8)).shape == (0, 8) and hb.int8_gemm(z(4, 32), z(32, 0)).shape == (4, 0)
    assert (hb.int8_gemm(z(4, 0), z(0, 8)) == 0).all()


def test_capture_another_stream_and_two_calls_at_once(hb):
    g = torch.Generator(device="cuda").manual_seed(12)
    y = codes(g, 4096, 2048).t()
    xs = [codes(g, m, 2048) for m in (4, 4, 500, 500)]
    want = [hb.int8_gemm(x, y, out_dtype=torch.float32) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(hb.int8_gemm(x, y, out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = torch.zeros_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hb.int8_gemm(held, y, out_dtype=torch.float32)
    for x, w in zip(xs[:2], want[:2]):
        held.copy_(x)
        graph.replay()
        assert torch.equal(out, w)


def test_norm_quantise_and_product_together(hb):
    """The 8-bit linear layer as it is used: norm with residual -> codes and scales -> product with token and channel scales."""
    g = torch.Generator(device="cuda").manual_seed(13)
    for m in (1, 200):
        x, r = (torch.randn(m, 1024, generator=g, device="cuda").bfloat16() for _ in range(2))
        w = 1 + 0.1 * torch.randn(1024, generator=g, device="cuda")
        y = codes(g, 512, 1024).t()
        sb = torch.rand(512, generator=g, device="cuda") * 1e-3
        q, s, h = hb.rms_norm_quantize(x, w, residual=r, out_dtype=torch.int8)
        check(hb.int8_gemm(q, y, scale_a=s, scale_b=sb), q, y, s, sb)
        q8, s8, _ = hb.rms_norm_quantize(x, w, residual=r)
        w8 = (torch.randn(512, 1024, generator=g, device="cuda")).to(torch.float8_e4m3fn).t()
        got = hb.fp8_gemm(q8, w8, scale_a=s8, scale_b=sb.reshape(1, -1), out_dtype=torch.float32)
        want = (q8.double() * s8.double()) @ (w8.double() * sb.double())
        # fp32 accumulation of 1024 products of either sign: each partial sum is within its rounding of the exact one
        scale = (q8.double().abs() * s8.double()) @ (w8.double().abs() * sb.double())
        assert ((got.double() - want).abs() <= scale * 1024 * 2.0**-24).all()
