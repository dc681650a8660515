"""The gated projection and its gradients against the formulas in 64 bits.

Tolerances.  A product's fp32 sum of K terms is within (K + 1) * 2**-24 of the exact one relative to the sum of the terms'
magnitudes; call that S for a result.  The activations and their derivatives are 1.13-Lipschitz and at most 1.13 + |g|
and 1.13 large, so h = act(g) u is within 1.13 (|u| eg + (1 + |g|) eu) of the formula, plus 2**-20 relative for the
activation's own arithmetic, plus half a step of the output.  The gradients' operands dG and dU are rounded once (half a
step h of the dtype) and carry the forward pass's errors: |dh| (1.13 eu + |u| eg) (no activation's second derivative is
above 1) and |dh| 1.13 eg.  A gradient is within h of its own value, plus (h + 2**-20 + (n + 4) 2**-24) of the sum of its n
terms' magnitudes, plus what the errors of dG and dU sum to."""
from __future__ import annotations

import math

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINIEST = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def act64(g, kind):
    """The activation and its derivative in 64 bits."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * torch.sigmoid(-g))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    z2 = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
    p = torch.sigmoid(z2)
    return g * p, p + g * p * torch.sigmoid(-z2) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


def check_forward(out, x, wg, wu, kind, sums_exact=False):
    """x, wg, wu in 64 bits, scales already applied."""
    g, u = x @ wg, x @ wu
    k = 0 if sums_exact else x.shape[1]
    eg, eu = ((k + 4) * 2.0**-24 * (x.abs() @ w.abs()) for w in (wg, wu))
    want = act64(g, kind)[0] * u
    bound = 1.13 * (u.abs() * eg + (1 + g.abs()) * eu) + (HALF_STEP[out.dtype] + 2.0**-20) * want.abs() + TINIEST[out.dtype]
    off = (out.double() - want).abs() - bound
    assert off.max().item() <= 0, f"{off.max().item()} beyond the bound"


def eight_bit(g, rows, cols, dtype):
    if dtype == torch.int8:
        return torch.randint(-128, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)
    return (torch.randn(rows, cols, generator=g, device="cuda") * 60).clamp(-448, 448).to(E4M3)


SIZES = [(1, 16, 8), (1, 4096, 264), (8, 2064, 14336), (17, 144, 19000), (33, 512, 1000), (64, 256, 136), (65, 1040, 520), (128, 2048, 4224), (96, 4112, 4232), (20, 1024, 9480), (128, 272, 128), (129, 128, 72), (257, 2048, 1000), (1000, 512, 5000)]


@pytest.mark.parametrize("out_dtype", list(HALF_STEP), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_eight_bit(hb, m, k, f, dtype, kind, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(m + k + f)
    x, wg, wu = eight_bit(g, m, k, dtype), eight_bit(g, f, k, dtype).t(), eight_bit(g, f, k, dtype).t()
    sx = (torch.rand(m, 1, generator=g, device="cuda") + 0.5) / 60
    sg, su = ((torch.rand(1, f, generator=g, device="cuda") + 0.5) / (60 * math.sqrt(k)) for _ in range(2))
    out = hb.gated_gemm(x, wg, wu, scale_x=sx, scale_gate=sg, scale_up=su, activation=kind, out_dtype=out_dtype)
    assert out.dtype == out_dtype and out.shape == (m, f)
    check_forward(out, x.double() * sx, wg.double() * sg, wu.double() * su, kind, dtype == torch.int8)
    assert torch.equal(out, hb.gated_gemm(x, wg, wu, scale_x=sx.reshape(-1), scale_gate=sg.reshape(-1), scale_up=su, activation=kind, out_dtype=out_dtype))


def test_eight_bit_tensor_scales_and_none(hb):
    g = torch.Generator(device="cuda").manual_seed(3)
    for m in (5, 300):
        x, wg, wu = eight_bit(g, m, 512, E4M3), eight_bit(g, 256, 512, E4M3).t(), eight_bit(g, 256, 512, E4M3).t()
        s = [torch.full((1,), v, device="cuda") for v in (0.01, 0.002, 0.003)]
        out = hb.gated_gemm(x, wg, wu, scale_x=s[0], scale_gate=s[1], scale_up=s[2], out_dtype=torch.float32)
        check_forward(out, x.double() * s[0].double(), wg.double() * s[1].double(), wu.double() * s[2].double(), "silu")
        x = (x.float() / 256).to(E4M3)
        wg, wu = ((w.float() / 256).to(E4M3) for w in (wg, wu))
        check_forward(hb.gated_gemm(x, wg, wu, out_dtype=torch.float32), x.double(), wg.double(), wu.double(), "silu")


@pytest.mark.parametrize("layout", ["col", "row", "mixed"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k,f", [(1, 8, 8), (1, 1000, 264), (7, 33, 50), (64, 136, 2000), (128, 264, 128), (130, 72, 1000), (333, 1000, 728), (700, 520, 4104)])
def test_sixteen_bit_forward(hb, m, k, f, dtype, kind, layout):
    g = torch.Generator(device="cuda").manual_seed(m + k + f)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    wg, wu = ((torch.randn(f, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype).t() for _ in range(2))
    if layout != "col":
        wu = wu.contiguous()
    if layout == "row":
        wg = wg.contiguous()
    out = hb.gated_matmul(x, wg, wu, activation=kind)
    assert out.dtype == dtype and out.shape == (m, f)
    check_forward(out, x.double(), wg.double(), wu.double(), kind)


def grads64(x, wg, wu, dh, kind, tiniest=0.0):
    """Every gradient, the sum of its terms' magnitudes, and what the errors of dG and dU sum to."""
    g, u = x @ wg, x @ wu
    a, d = act64(g, kind)
    dg, du = dh * u * d, dh * a
    three = lambda x, wg, wu, dg, du: (dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du)  # noqa: E731
    mag = [t.abs() for t in (x, wg, wu)]
    eg, eu = ((x.shape[1] + 4) * 2.0**-24 * (mag[0] @ w) for w in mag[1:])
    off = dh.abs() * (1.13 * eu + u.abs() * eg) + tiniest, dh.abs() * 1.13 * eg + tiniest
    return three(x, wg, wu, dg, du), three(*mag, dg.abs(), du.abs()), three(*mag, *off)


def check_grads(got, x, wg, wu, dh, kind, dtype, terms):
    """Gradients against the formula for x, weights and dh in 64 bits; terms: how many each one sums."""
    for name, a, w, s, e, n in zip(("dx", "dw_gate", "dw_up"), got, *grads64(x, wg, wu, dh, kind, TINIEST[dtype]), terms):
        assert a.dtype == dtype and a.shape == w.shape
        bound = HALF_STEP[dtype] * w.abs() + (HALF_STEP[dtype] + 2.0**-20 + (n + 4) * 2.0**-24) * s + e + TINIEST[dtype]
        off = (a.double() - w).abs() - bound
        assert off.max().item() <= 0, f"{name}: {off.max().item()} beyond the bound"


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k,f", [(1, 8, 8), (3, 40, 24), (65, 33, 50), (130, 264, 1000), (333, 1000, 728), (512, 4096, 512), (1025, 264, 2056), (200, 520, 9000), (60, 2048, 1000), (1100, 4104, 264)])
def test_gradients(hb, m, k, f, dtype, kind, layout):
    g = torch.Generator(device="cuda").manual_seed(m * 7 + k + f)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype).requires_grad_()
    wg, wu = ((torch.randn(f, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype).t() for _ in range(2))
    if layout == "row":
        wg, wu = wg.contiguous(), wu.contiguous()
    wg.requires_grad_()
    wu.requires_grad_()
    dh = torch.randn(m, f, generator=g, device="cuda").to(dtype)
    h = hb.gated_matmul(x, wg, wu, activation=kind)
    args = [t.detach().double() for t in (x, wg, wu)]
    check_forward(h.detach(), *args, kind)
    got = torch.autograd.grad(h, (x, wg, wu), dh)
    check_grads(got, *args, dh.double(), kind, dtype, (2 * f, m, m))


def test_formula_against_differences():
    """The 64-bit gradients that the kernels are held to, against central differences."""
    torch.manual_seed(0)
    for kind in ("silu", "gelu", "gelu_tanh"):
        x, wg, wu, dh = (torch.randn(s, dtype=torch.float64) for s in ((3, 4), (4, 5), (4, 5), (3, 5)))
        want = grads64(x, wg, wu, dh, kind)[0]
        for t, w in zip((x, wg, wu), want):
            for i in range(t.numel()):
                keep, e, v = t.view(-1)[i].item(), 1e-5, []
                for s in (e, -e):
                    t.view(-1)[i] = keep + s
                    v.append((act64(x @ wg, kind)[0] * (x @ wu) * dh).sum().item())
                t.view(-1)[i] = keep
                assert abs((v[0] - v[1]) / (2 * e) - w.reshape(-1)[i].item()) < 1e-7


def test_only_the_wanted_gradients_and_shared_weights(hb):
    g = torch.Generator(device="cuda").manual_seed(4)
    base = [torch.randn(70, 64, generator=g, device="cuda").bfloat16()] + [(torch.randn(48, 64, generator=g, device="cuda") / 8).bfloat16().t() for _ in range(2)]
    full = [t.clone().requires_grad_() for t in base]
    hb.gated_matmul(*full).sum().backward()  # an expanded gradient: every row of it is the same memory
    for i in range(3):
        only = [t.clone().requires_grad_(i == j) for j, t in enumerate(base)]
        hb.gated_matmul(*only).sum().backward()
        assert [t.grad is not None for t in only] == [i == j for j in range(3)]
        assert torch.equal(only[i].grad, full[i].grad)
    # the same tensor as both weights, and accumulation over two calls
    w = base[1].clone().requires_grad_()
    x = base[0].clone().requires_grad_()
    hb.gated_matmul(x, w, w).sum().backward()
    once = w.grad.clone()
    two = [t.clone().requires_grad_() for t in (base[0], base[1], base[1])]
    hb.gated_matmul(*two).sum().backward()
    torch.testing.assert_close(once.double(), two[1].grad.double() + two[2].grad.double(), rtol=2.0**-7, atol=2.0**-7)
    hb.gated_matmul(x, w, w).sum().backward()
    torch.testing.assert_close(w.grad, 2 * once)
    h = hb.gated_matmul(x, w, w)
    (dx,) = torch.autograd.grad(h, x, torch.ones_like(h), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with torch.no_grad():
        assert not hb.gated_matmul(x, w, w).requires_grad


def test_extreme_pre_activations(hb):
    """Large pre-activations of either sign saturate the gate without a NaN; NaN and infinity stay in their rows."""
    for dtype in (torch.bfloat16, torch.float16):
        big = 200.0
        x = torch.zeros(200, 16, device="cuda", dtype=dtype)
        x[:, 0] = torch.linspace(-big, big, 200, device="cuda").to(dtype)
        x[:, 1] = 1
        wg = torch.zeros(16, 8, device="cuda", dtype=dtype)
        wg[0] = 1
        wu = torch.zeros(16, 8, device="cuda", dtype=dtype)
        wu[1] = 1
        for kind in ("silu", "gelu", "gelu_tanh"):
            leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
            h = hb.gated_matmul(*leaves, activation=kind)
            check_forward(h.detach(), x.double(), wg.double(), wu.double(), kind)
            grads = torch.autograd.grad(h, leaves, torch.ones_like(h))
            # finite wherever the formula's gradient is: dw_up[0] sums x0 act(x0) to 100 * 200**2 / 3 = 1.3e6, which is
            # infinite in fp16
            want = grads64(x.double(), wg.double(), wu.double(), torch.ones_like(h).double(), kind)[0]
            assert all(torch.equal(t.isfinite(), w.to(dtype).isfinite()) and not t.isnan().any() for t, w in zip(grads, want))
    clean = hb.gated_matmul(x, wg, wu)
    x2 = x.clone()
    x2[3, 0], x2[150, 1] = float("nan"), float("inf")
    got = hb.gated_matmul(x2, wg, wu)
    rest = [i for i in range(200) if i not in (3, 150)]
    assert got[3].isnan().all() and torch.equal(got[rest], clean[rest])
    huge = torch.full((2, 8), 3e38, device="cuda", dtype=torch.bfloat16)
    eye = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    for kind in ("silu", "gelu", "gelu_tanh"):
        for sign in (1, -1):
            leaves = [(huge * sign).requires_grad_(), eye.clone().requires_grad_(), (eye * 2.0**-20).requires_grad_()]
            h = hb.gated_matmul(*leaves, activation=kind)
            assert not h.isnan().any()
            dx = torch.autograd.grad(h, leaves[0], torch.full_like(h, 2.0**-120))[0]
            assert not dx.isnan().any()


def test_offsets_beyond_31_bits(hb):
    g = torch.Generator(device="cuda").manual_seed(14)
    m, f = 70000, 32776
    x, wg, wu = eight_bit(g, m, 16, torch.int8), eight_bit(g, f, 16, torch.int8).t(), eight_bit(g, f, 16, torch.int8).t()
    s = torch.full((1,), 0.004, device="cuda")
    out = hb.gated_gemm(x, wg, wu, scale_x=s, scale_gate=s, scale_up=s)
    s64 = s.double()
    for rows in (slice(0, 5), slice(m - 300, m)):
        check_forward(out[rows], x[rows].double() * s64, wg.double() * s64, wu.double() * s64, "silu", True)
    del out
    xb = torch.zeros(m, 8, device="cuda", dtype=torch.bfloat16)
    xb[-2:] = torch.randn(2, 8, generator=g, device="cuda").bfloat16()
    wb = [torch.randn(f, 8, generator=g, device="cuda").bfloat16().t() for _ in range(2)]
    leaves = [xb.requires_grad_(), *(w.requires_grad_() for w in wb)]
    h = hb.gated_matmul(*leaves)
    dh = torch.zeros_like(h)
    dh[-2:] = 1
    got = torch.autograd.grad(h, leaves, dh)
    assert (got[0][:-2] == 0).all()
    last = [xb.detach()[-2:].double(), *(w.detach().double() for w in wb), dh[-2:].double()]
    check_grads((got[0][-2:], *got[1:]), *last, "silu", torch.bfloat16, (2 * f, 2, 2))


def test_empty_dimensions(hb):
    for m, k, f in ((0, 16, 8), (4, 16, 0), (4, 0, 8)):
        leaves = [torch.zeros(s, device="cuda", dtype=torch.bfloat16, requires_grad=True) for s in ((m, k), (k, f), (k, f))]
        h = hb.gated_matmul(*leaves)
        assert h.shape == (m, f) and (h == 0).all()
        h.sum().backward()
        assert all((t.grad == 0).all() and t.grad.shape == t.shape for t in leaves)
        z = [torch.zeros(s, device="cuda", dtype=torch.int8) for s in ((m, k), (k, f), (k, f))]
        out = hb.gated_gemm(*z)
        assert out.shape == (m, f) and (out == 0).all()


def test_layouts_odd_sizes_and_given_outputs(hb):
    g = torch.Generator(device="cuda").manual_seed(9)
    for m in (3, 150):
        for k, f in ((17, 33), (48, 40)):
            x, wg, wu = eight_bit(g, m, k, torch.int8), eight_bit(g, f, k, torch.int8), eight_bit(g, f, k, torch.int8)
            sx, sg, su = torch.rand(m, generator=g, device="cuda") / 90, torch.rand(f, generator=g, device="cuda") / 90, torch.rand(f, generator=g, device="cuda") / 90
            kw = {"scale_x": sx, "scale_gate": sg, "scale_up": su, "out_dtype": torch.float32}
            want = hb.gated_gemm(x, wg.t(), wu.t(), **kw)
            check_forward(want, x.double() * sx[:, None], wg.t().double() * sg, wu.t().double() * su, "silu", True)
            wide = eight_bit(g, m, 3 * k + 1, torch.int8)
            wide[:, 5 : 5 + k] = x
            for xx in (wide[:, 5 : 5 + k], x.t().contiguous().t()):
                for ww in ((wg.t().contiguous(), wu.t()), (wg.t().contiguous(), wu.t().contiguous())):
                    assert torch.equal(hb.gated_gemm(xx, *ww, **kw), want)
            store = torch.full((m + 3, 48), 7.0, device="cuda")
            out = store[:m, :f]
            assert hb.gated_gemm(x, wg.t(), wu.t(), **kw, out=out) is out
            assert torch.equal(out, want) and (store[m:] == 7).all() and (store[:, f:] == 7).all()


def test_streams_devices_and_graphs(hb):
    g = torch.Generator(device="cuda").manual_seed(10)
    x = torch.randn(260, 512, generator=g, device="cuda").bfloat16()
    wg, wu = ((torch.randn(1024, 512, generator=g, device="cuda") / 22).bfloat16().t() for _ in range(2))
    dh = torch.randn(260, 1024, generator=g, device="cuda").bfloat16()

    def step(x, wg, wu):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        h = hb.gated_matmul(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    want = step(x, wg, wu)
    side = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in side:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(step(x, wg, wu))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    # forward and backward passes captured into two graphs
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    held = torch.zeros_like(x).requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(hb.gated_matmul(held, *leaves[1:]), (held, *leaves[1:]), dh)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            h = hb.gated_matmul(held, *leaves[1:])
            outs.append((h.detach(), *torch.autograd.grad(h, (held, *leaves[1:]), dh)))
    with torch.no_grad():
        held.copy_(x)
    for graph, out in zip(graphs, outs):
        graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("k", [64, 33])
def test_capture_next_to_a_living_eager_graph_is_refused(hb, k):
    """An eager graph on the default stream ties the leaves' accumulators to it: capturing a backward pass over them is
    refused before anything is recorded, and works once that graph is gone."""
    g = torch.Generator(device="cuda").manual_seed(11)
    leaves = [torch.randn(s, generator=g, device="cuda").bfloat16().requires_grad_() for s in ((140, k), (k, 48), (k, 48))]
    dh = torch.randn(140, 48, generator=g, device="cuda").bfloat16()
    eager = hb.gated_matmul(*leaves)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            hb.gated_matmul(*leaves)
    want = torch.autograd.grad(eager, leaves, dh)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(hb.gated_matmul(*leaves), leaves, dh)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("m", [1, 16, 200])
@pytest.mark.parametrize("dtype", [E4M3, torch.int8], ids=["e4m3", "int8"])
def test_a_feed_forward_block_in_eight_bits(hb, m, dtype):
    """norm with residual -> gated projection -> quantise -> down projection, each step against 64 bits of its inputs."""
    g = torch.Generator(device="cuda").manual_seed(m)
    k, f = 512, 1536
    x, r = (torch.randn(m, k, generator=g, device="cuda").bfloat16() for _ in range(2))
    wn = 1 + 0.1 * torch.randn(k, generator=g, device="cuda")
    wg, wu = ((eight_bit(g, f, k, dtype)).t() for _ in range(2))
    wd = eight_bit(g, k, f, dtype).t()
    sg, su, sd = (torch.rand(1, n, generator=g, device="cuda") / (60 * math.sqrt(k)) for n in (f, f, k))
    q, s, stream = hb.rms_norm_quantize(x, wn, residual=r, out_dtype=dtype)
    h = hb.gated_gemm(q, wg, wu, scale_x=s, scale_gate=sg, scale_up=su)
    check_forward(h, q.double() * s, wg.double() * sg, wu.double() * su, "silu", dtype == torch.int8)
    q2, s2 = hb.quantize_rows(h, out_dtype=dtype)
    gemm = hb.int8_gemm if dtype == torch.int8 else hb.fp8_gemm
    y = gemm(q2, wd, scale_a=s2, scale_b=sd, out_dtype=torch.float32)
    want = (q2.double() * s2) @ (wd.double() * sd)
    size = (q2.double().abs() * s2) @ (wd.double().abs() * sd)
    assert ((y.double() - want).abs() <= size * (f + 4) * 2.0**-24).all()
    # the whole block is near the unquantised one: each quantisation is within half a step of a row's values (e4m3
    # relative 2**-4, int8 max/254), which the products average out
    y64 = (x.double() + r.double())
    y64 = y64 / (y64.square().mean(1, keepdim=True) + 1e-6).sqrt() * wn.double()
    g64, u64 = y64 @ (wg.double() * sg), y64 @ (wu.double() * su)
    exact = (act64(g64, "silu")[0] * u64) @ (wd.double() * sd)
    assert (y.double() - exact).norm() <= 0.1 * exact.norm()
