"""Outputs that the caller gives are known to autograd as changed."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hb(built_library):
    import helion_b200

    _lib.reset_status(0)
    yield helion_b200
    torch.cuda.synchronize()
    _lib.check_status(0)


def test_an_update_in_place_of_what_a_graph_saved_is_seen(hb):
    for target in ("x", "residual"):
        t = {n: torch.randn(4, 64, device="cuda").bfloat16() for n in ("x", "residual")}
        w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = t[target] * w  # keeps t[target] for w's gradient
        hb.rms_norm_quantize(t["x"], w.detach(), residual=t["residual"], residual_out=t[target])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_every_given_output_counts_a_change_and_nothing_else_does(hb):
    x = torch.randn(4, 64, device="cuda").bfloat16()
    r = torch.randn(4, 64, device="cuda").bfloat16()
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    codes, scale, total = torch.empty(4, 64, device="cuda", dtype=torch.int8), torch.empty(4, 1, device="cuda"), torch.empty_like(x)
    wide = torch.empty(4, 16, device="cuda", dtype=torch.bfloat16)
    w8 = torch.ones(16, 64, device="cuda", dtype=torch.int8).t()
    odd = torch.empty(4, 13, device="cuda", dtype=torch.bfloat16)
    calls = [
        (lambda: hb.quantize_rows(x, out_dtype=torch.int8, out=codes, scale_out=scale), (codes, scale)),
        (lambda: hb.rms_norm_quantize(x, w, residual=r, out_dtype=torch.int8, out=codes, scale_out=scale, residual_out=total), (codes, scale, total)),
        (lambda: hb.int8_gemm(codes, w8, out=wide), (wide,)),
        (lambda: hb.int8_gemm(codes[:, :13].contiguous(), w8[:13, :13], out=odd), (odd,)),
        (lambda: hb.gated_gemm(codes, w8, w8, out=wide), (wide,)),
        (lambda: hb.gated_gemm(codes, w8[:, :13], w8[:, :13], out=odd), (odd,)),
    ]
    everything = (x, r, w, codes, scale, total, wide, w8, odd)
    for call, given in calls:
        before = [t._version for t in everything]
        call()
        assert [t._version - b > 0 for t, b in zip(everything, before)] == [any(t is o for o in given) for t in everything]


def test_outputs_made_in_inference_mode(hb):
    with torch.inference_mode():
        x = torch.randn(4, 64, device="cuda").bfloat16()
        codes, scale = hb.quantize_rows(x, out_dtype=torch.int8)
        again = hb.quantize_rows(x, out_dtype=torch.int8, out=torch.empty_like(codes), scale_out=torch.empty_like(scale))
        assert torch.equal(codes, again[0]) and torch.equal(scale, again[1])
