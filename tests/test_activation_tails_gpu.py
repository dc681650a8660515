"""The gate's activations where they are small: relative errors out to where the values leave fp32's normal range.

x and the weights are int8 with one product each in g and u and scales that are powers of two, so g = a b / 2**s and u = 1 are
exact, and out = act(g) carries the activation's own errors alone.  In units of 2**-24 of the value:

fp32 output.  exp is within 2 ulp (4 units).  silu: 1 + e, the division, e / (1 + e) and g s add one each: 8.  gelu: the smooth
factor's fit is within 8.2e-8 (1.4 units), its argument within 3 and its sum within 4, two products, 1 + 1 for the
exponential's remainder and g p: 17, and 1 - q is no worse.  gelu_tanh: the argument 2 z has a constant, a square, a sum and
two products, each one unit of 2 z, which the exponential turns into 6 |2 z| of the value, and then as silu.
16-bit output.  The fast exponential is within 2 + 1.173 |v| ulp at v (CUDA's documentation), that is 4 + 2.4 |v| units, its argument
-g**2 / 2 has two roundings (2 |v| more, 6 |v| for 2 z as above) and the fast division 2 ulp; then half a step of the output.
Below 2**-126 the exponential (2 ulp) and its product with the division (half a step) are held in steps of 2**-149, which the
product with g multiplies; at the output's own smallest numbers half of their step is added."""
from __future__ import annotations

import math

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINIEST = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}
UNIT = 2.0**-24


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def act64(g, kind):
    """The activation, the exponential's argument v, and the derivative."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, g.abs(), s * (1 + g * torch.sigmoid(-g))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, g * g / 2, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    z2 = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
    p = torch.sigmoid(z2)
    return g * p, z2.abs(), p + g * p * torch.sigmoid(-z2) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


def units(kind, v, precise):
    if precise:
        return {"silu": 8.0, "gelu": 24.0, "gelu_tanh": 8.0 + 6.0 * v}[kind]  # (gelu: 17, and the last bits of its fit)
    return {"silu": 12 + 2.4 * v, "gelu": 24 + 4.4 * v, "gelu_tanh": 12 + 8.4 * v}[kind]


@pytest.mark.parametrize("out_dtype", list(HALF_STEP), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [120, 254])  # the kernel for few rows and the tiles
@pytest.mark.parametrize("divisor", [2**7, 2**9, 2**10, 2**12, 2**16])
def test_values_of_the_activations(hb, divisor, m, kind, out_dtype):
    x = torch.zeros(m, 16, device="cuda", dtype=torch.int8)
    x[:, 0] = torch.linspace(-127, 127, m, device="cuda").round().to(torch.int8)
    x[:, 1] = 1
    wg, wu = (torch.zeros(16, 128, device="cuda", dtype=torch.int8) for _ in range(2))
    wg[0] = torch.arange(128, device="cuda").to(torch.int8)
    wu[1] = 1
    one = torch.ones(1, device="cuda")
    wg, wu = (w.t().contiguous().t() for w in (wg, wu))
    got = hb.gated_gemm(x, wg, wu, scale_x=one, scale_gate=one / divisor, scale_up=one, activation=kind, out_dtype=out_dtype).double()
    g = x[:, :1].double() * wg[:1].double() / divisor
    want, v, _ = act64(g, kind)
    bound = (units(kind, v, out_dtype == torch.float32) * UNIT + HALF_STEP[out_dtype]) * want.abs() + (1 + 2 * g.abs()) * 2.0**-148 + TINIEST[out_dtype]
    worst = (got - want).abs() / bound
    at = worst.argmax()
    assert worst.max().item() <= 1, f"act({g.reshape(-1)[at].item()}) = {got.reshape(-1)[at].item()}, formula {want.reshape(-1)[at].item()}"


@pytest.mark.parametrize("out_dtype", list(HALF_STEP), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m", [4, 200])
def test_infinite_and_huge_arguments(hb, m, out_dtype):
    """g of +inf and 2**127 give themselves (fp16: infinity), -2**127 gives zero, and a NaN stays one, next to values that are none of these."""
    x = torch.zeros(m, 16, device="cuda", dtype=torch.int8)
    x[:, 0] = x[:, 1] = 1
    w = torch.zeros(8, 16, device="cuda", dtype=torch.int8)
    w[:, 0] = torch.tensor([1, 1, -1, 1, 1, 0, 0, 0])
    up = torch.zeros(8, 16, device="cuda", dtype=torch.int8)
    up[:, 1] = 1
    sx, su = torch.ones(m, device="cuda"), torch.ones(8, device="cuda")
    sg = torch.tensor([float("inf"), 2.0**127, 2.0**127, float("nan"), 1, 1, 1, 1], device="cuda")
    for kind in ("silu", "gelu", "gelu_tanh"):
        out = hb.gated_gemm(x, w.t(), up.t(), scale_x=sx, scale_gate=sg, scale_up=su, activation=kind, out_dtype=out_dtype).double()
        assert (out[:, 0] == float("inf")).all() and (out[:, 2] == 0).all() and out[:, 3].isnan().all() and (out[:, 5:] == 0).all()
        assert (out[:, 1] == (float("inf") if out_dtype == torch.float16 else 2.0**127)).all()
        assert (out[:, 4] - act64(torch.ones(1, dtype=torch.float64), kind)[0].item()).abs().max() < 2.0**-8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_gradients_far_out(hb, kind, dtype):
    """One row of x and one of each weight take part, so every gradient is one product: dg = dh act'(g) and du = dh act(g),
    rounded to the operands' type, times exact values, rounded once more.  dh lifts them out of fp16's subnormals."""
    n = 232
    x = torch.zeros(n, 16, device="cuda", dtype=dtype)
    x[:, 0] = (torch.arange(n, device="cuda") - 200).to(dtype) / 2  # g from -100 to 16
    x[:, 1] = 1
    wg, wu = (torch.zeros(16, 8, device="cuda", dtype=dtype) for _ in range(2))
    wg[0, 0] = 1
    wu[1, 0] = 1
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    h = hb.gated_matmul(*leaves, activation=kind)
    dh = torch.zeros_like(h)
    dh[:, 0] = 2.0**12 if dtype == torch.float16 else 2.0**20
    (dx,) = torch.autograd.grad(h, x, dh)
    g, scale = x.detach()[:, 0].double(), dh[0, 0].double()
    a, v, d = act64(g, kind)
    # the derivative is a sum p + g p' whose parts may cancel: relative to their magnitudes
    size = (d - a / torch.where(g == 0, 1.0, g)).abs() + (a / torch.where(g == 0, 1.0, g)).abs() + (g == 0) * 0.5
    for got, want, mag in ((dx[:, 0], d, size), (dx[:, 1], a, a.abs())):
        bound = (2.1 * HALF_STEP[dtype] * want.abs() + (units(kind, v, False) + 8) * UNIT * mag + (1 + g.abs()) * 2.0**-147) * scale + 3 * TINIEST[dtype]
        off = (got.double() - want * scale).abs() - bound
        assert off.max().item() <= 0, f"{off.max().item()} beyond the bound at g = {g[off.argmax()].item()}"
