"""fp16 gradients of the gated projection where dG = dh u act'(g) and dU = dh act(g) leave fp16's range but the gradients do not.

dG and dU are operands of the gradients' products and held in fp16, together multiplied by one power of two where their
largest magnitude asks for it, which the products' fp32 results are divided by.  The bounds are those of any other size: half a
step h of the operands (for what lies more than 2**-29 below the largest of dG and dU, half a step of fp16's subnormals there,
2**-40 of that largest one), the forward pass's errors as in the tests of the gradients, the sum's own, and half a step of the
output."""
from __future__ import annotations

import math

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

H = 2.0**-11
TINIEST = 2.0**-25


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def silu64(g):
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * torch.sigmoid(-g))


def check(got, x, wg, wu, dh):
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    g, u = x @ wg, x @ wu
    a, d = silu64(g)
    dg, du = dh * u * d, dh * a
    top = torch.maximum(dg.abs().max(), du.abs().max())
    mag = [t.abs() for t in (x, wg, wu)]
    eg, eu = ((x.shape[1] + 4) * 2.0**-24 * (mag[0] @ w) for w in mag[1:])
    # largest of dG and dU at 2**14 or more of fp16's range where it was moved: half a step of a subnormal is 2**-25 of 2**14
    floor = max(TINIEST if 2.0**-6 <= top <= 65000 else 0.0, 0.0) + top * 2.0**-39
    off = dh.abs() * (1.13 * eu + u.abs() * eg) + floor, dh.abs() * 1.13 * eg + floor
    three = lambda x, wg, wu, dg, du: (dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du)  # noqa: E731
    for name, t, want, size, more, n in zip(("dx", "dw_gate", "dw_up"), got, three(x, wg, wu, dg, du), three(*mag, dg.abs(), du.abs()), three(*mag, *off), (2 * wg.shape[1], x.shape[0], x.shape[0])):
        bound = H * want.abs() + (H + 2.0**-19 + (n + 4) * 2.0**-24) * size + more + TINIEST
        over = (t.double() - want).abs() - bound
        fits = want.abs() + bound < 65504
        assert t.isfinite()[fits].all(), f"{name}: not finite where the formula is"
        assert over[fits].max().item() <= 0, f"{name}: {over[fits].max().item()} beyond the bound"
        assert not t.isnan().any()
        assert fits.double().mean() > 0.9  # (the case is about gradients that fp16 holds)


def run(hb, x, wg, wu, dh):
    leaves = [t.half().requires_grad_() for t in (x, wg, wu)]
    dh = dh.half()
    h = hb.gated_matmul(*leaves)
    got = torch.autograd.grad(h, leaves, dh)
    check(got, *leaves, dh)
    return got


@pytest.mark.parametrize("m,k,f", [(64, 64, 64), (333, 200, 728), (300, 4104, 72), (1100, 2056, 136), (2048, 1024, 512)])
@pytest.mark.parametrize("layout", ["col", "row"])
def test_products_beyond_the_largest_number(hb, m, k, f, layout):
    """dG reaches several times 65504; the weights that it meets are small, and so is x."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda") * 2.0**-9
    wg = torch.randn(f, k, generator=g, device="cuda") / math.sqrt(f) * 2.0**-7
    wu = torch.randn(f, k, generator=g, device="cuda") * (200 * 2**9 / math.sqrt(k))
    x = torch.where(torch.rand(m, 1, generator=g, device="cuda") < 0.5, x, x * 2.0**-6)
    wg, wu = wg.t(), wu.t().clamp(-60000, 60000)
    if layout == "row":
        wg, wu = wg.contiguous(), wu.contiguous()
    dh = torch.randn(m, f, generator=g, device="cuda") * 300
    top = (dh.double() * (x.double() @ wu.double()) * 0.5).abs().max()
    assert top > 65504
    run(hb, x, wg, wu, dh)


@pytest.mark.parametrize("m,k,f", [(64, 64, 64), (333, 200, 728), (2048, 1024, 512)])
def test_products_below_the_smallest_number(hb, m, k, f):
    """dG and dU below 2**-25, which fp16 holds as zero; the weights' gradients sum many of them times large values of x."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda").abs() * 2.0**7
    wg = torch.randn(f, k, generator=g, device="cuda").t() * (2.0**-8 / math.sqrt(k))
    wu = torch.randn(f, k, generator=g, device="cuda").t() * (2.0**-13 / math.sqrt(k))
    dh = torch.randint(1, 4, (m, f), generator=g, device="cuda") * 2.0**-22
    got = run(hb, x, wg, wu, dh)
    assert all((t != 0).double().mean() > 0.5 for t in got[1:])


def test_what_is_not_finite_stays_where_it_is(hb):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, dh = torch.randn(40, 64, generator=g, device="cuda").half(), torch.randn(40, 72, generator=g, device="cuda").half()
    wg, wu = (torch.randn(64, 72, generator=g, device="cuda").half() / 8 for _ in range(2))

    def grads(dh):
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
        return torch.autograd.grad(hb.gated_matmul(*leaves), leaves, dh)

    clean = grads(dh)
    for bad in (float("nan"), float("inf")):
        dirty = dh.clone()
        dirty[7, 9] = bad
        got = grads(dirty)
        rest = [i for i in range(40) if i != 7]
        assert torch.equal(got[0][rest], clean[0][rest]) and not got[0][7].isfinite().any()
        cols = [i for i in range(72) if i != 9]
        assert all(torch.equal(a[:, cols], b[:, cols]) and not a[:, 9].isfinite().any() for a, b in zip(got[1:], clean[1:]))
    zero = grads(torch.zeros_like(dh))
    assert all((t == 0).all() for t in zero)


def test_captured_with_other_magnitudes_than_replayed(hb):
    """The power of two is found anew in every pass: a graph captured with ordinary gradients is right for large ones."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x = (torch.randn(64, 64, generator=g, device="cuda") * 2.0**-9).half().requires_grad_()
    wg = (torch.randn(64, 64, generator=g, device="cuda") * 2.0**-10).half().requires_grad_()
    wu = (torch.randn(64, 64, generator=g, device="cuda") * 200 * 2**6).half().requires_grad_()
    dh = torch.randn(64, 64, generator=g, device="cuda").half()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(hb.gated_matmul(x, wg, wu), (x, wg, wu), dh)
    for factor in (1.0, 400.0, 2.0**-20):
        with torch.no_grad():
            dh.copy_((torch.randn(64, 64, generator=g, device="cuda") * factor).half())
        graph.replay()
        check(got, x, wg, wu, dh)
