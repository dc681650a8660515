"""Refusals of the gated projection, in Python and at the C entry points: no GPU is touched."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib


def test_operators_refuse_what_they_do_not_take():
    import helion_b200 as hb

    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16)
    x8, w8 = x.to(torch.int8), w.to(torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.gated_matmul(x, w, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.gated_gemm(x8, w8, w8)
    with pytest.raises(TypeError, match="three float16 or three bfloat16"):
        hb.gated_matmul(x, w, w.half())
    with pytest.raises(TypeError, match="three float16 or three bfloat16"):
        hb.gated_matmul(x.float(), w.float(), w.float())
    with pytest.raises(TypeError, match="three int8"):
        hb.gated_gemm(x8, w8, w8.to(torch.float8_e4m3fn))
    with pytest.raises(TypeError, match="three int8"):
        hb.gated_gemm(x, w, w)
    for op, a, b in ((hb.gated_matmul, x, w), (hb.gated_gemm, x8, w8)):
        with pytest.raises(ValueError, match="2-D"):
            op(a[0], b, b)
        with pytest.raises(ValueError, match="differ in shape"):
            op(a, b, b[:, :4])
        with pytest.raises(ValueError, match="size mismatch"):
            op(a[:, :8], b, b)
        with pytest.raises(ValueError, match="activation must be one of"):
            op(a, b, b, activation="relu")
    with pytest.raises(TypeError, match="out_dtype"):
        hb.gated_gemm(x8, w8, w8, out_dtype=torch.int8)


def _forward(lib, M=64, F=64, K=64, x_rs=64, g=(1, 64), u=(1, 64), out_rs=64, i=_lib.DT_INT8, o=_lib.DT_BF16, act=0, x=256, wg=512, wu=768,
             out=1024, s=(4096, 8192, 12288), mode=2, p=None, a=None):
    return lib.hb200_gated_gemm(x, wg, wu, out, M, F, K, x_rs, *g, *u, out_rs, i, o, act, *s, mode, p, a, 0, None)


HALF = {"i": _lib.DT_BF16, "mode": 0}


@pytest.mark.parametrize("change,code", [
    ({"i": _lib.DT_FP32}, _lib.ERR_BAD_DTYPE), ({"o": _lib.DT_INT8}, _lib.ERR_BAD_DTYPE), ({**HALF, "o": _lib.DT_FP32}, _lib.ERR_BAD_DTYPE),
    ({"act": 3}, _lib.ERR_BAD_CONFIG), ({"mode": 5}, _lib.ERR_BAD_CONFIG), ({"i": _lib.DT_BF16}, _lib.ERR_BAD_CONFIG), ({"p": 256, "a": 512}, _lib.ERR_BAD_CONFIG),
    ({**HALF, "p": 256}, _lib.ERR_BAD_CONFIG), ({"M": 0}, _lib.ERR_BAD_SHAPE), ({"F": 60}, _lib.ERR_BAD_SHAPE), ({"K": 56}, _lib.ERR_BAD_SHAPE),
    ({"K": 131072, "x_rs": 131072, "g": (1, 131072), "u": (1, 131072)}, _lib.ERR_BAD_SHAPE), ({"x_rs": 48}, _lib.ERR_BAD_STRIDE), ({"x_rs": 72}, _lib.ERR_BAD_STRIDE),
    ({"g": (64, 1), "u": (64, 1)}, _lib.ERR_BAD_STRIDE), ({**HALF, "g": (64, 1)}, _lib.ERR_BAD_STRIDE), ({"g": (1, 72)}, _lib.ERR_BAD_STRIDE), ({"u": (1, 48)}, _lib.ERR_BAD_STRIDE),
    ({"out_rs": 56}, _lib.ERR_BAD_STRIDE), ({"x": None}, _lib.ERR_ALIGN), ({"wu": 776}, _lib.ERR_ALIGN), ({"s": (4096, None, 64)}, _lib.ERR_ALIGN), ({"s": (4096, 2, 64)}, _lib.ERR_ALIGN),
])
def test_forward_entry_point_checks_its_arguments(built_library, change, code):
    assert _forward(built_library, **change) == code
    assert "gated_gemm" in _lib.last_error()


def _backward(lib, M=64, F=64, K=64, dh_rs=64, x_rs=64, g=(1, 64), u=(1, 64), dt=_lib.DT_BF16, dh=256, x=512, wg=768, wu=1024, p=2048, a=4096, dx=8192, dg=16384, du=32768,
              ws=65536, ws_bytes=64 * 64 * 4):
    return lib.hb200_gated_gemm_backward(dh, x, wg, wu, p, a, dx, dg, du, M, F, K, dh_rs, x_rs, *g, *u, dt, ws, ws_bytes, 0, None)


@pytest.mark.parametrize("change,code", [
    ({"dt": _lib.DT_FP32}, _lib.ERR_BAD_DTYPE), ({"M": 0}, _lib.ERR_BAD_SHAPE), ({"K": 12}, _lib.ERR_BAD_SHAPE), ({"dh_rs": 56}, _lib.ERR_BAD_STRIDE),
    ({"dh_rs": 68}, _lib.ERR_BAD_STRIDE), ({"u": (64, 1)}, _lib.ERR_BAD_STRIDE), ({"p": None}, _lib.ERR_ALIGN), ({"dg": None}, _lib.ERR_ALIGN), ({"dx": 8}, _lib.ERR_ALIGN),
    ({"ws_bytes": 64 * 64 * 4 - 1}, _lib.ERR_WORKSPACE), ({"ws": None}, _lib.ERR_WORKSPACE), ({"ws": 8}, _lib.ERR_WORKSPACE),
])
def test_backward_entry_point_checks_its_arguments(built_library, change, code):
    assert _backward(built_library, **change) == code
    assert "gated_gemm_backward" in _lib.last_error()
