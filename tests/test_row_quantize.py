"""Refusals of the row-quantisation operators, in Python and at the C entry points: no GPU is touched."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib


def test_operators_refuse_what_they_do_not_take():
    import helion_b200 as hb

    x, w = torch.zeros(4, 32), torch.ones(32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.quantize_rows(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.rms_norm_quantize(x, w)
    with pytest.raises(TypeError, match="expects a float16"):
        hb.quantize_rows(x.double())
    with pytest.raises(TypeError, match="out_dtype"):
        hb.quantize_rows(x, out_dtype=torch.float8_e5m2)
    with pytest.raises(ValueError, match="at least one value"):
        hb.quantize_rows(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="vector of N=32"):
        hb.rms_norm_quantize(x, torch.ones(31))
    with pytest.raises(TypeError, match="weight must be"):
        hb.rms_norm_quantize(x, w.half())
    with pytest.raises(TypeError, match="residual must be"):
        hb.rms_norm_quantize(x, w, residual=x.half())
    with pytest.raises(ValueError, match="differ in shape"):
        hb.rms_norm_quantize(x, w, residual=torch.zeros(3, 32))
    for eps in (0.0, -1.0, 1e-40, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="positive normal"):
            hb.rms_norm_quantize(x, w, eps=eps)
    with pytest.raises(ValueError, match="needs a residual"):
        hb.rms_norm_quantize(x, w, residual_out=x)


def _call(lib, fn="norm", M=4, N=32, x_rs=32, res_rs=32, c_rs=32, so_rs=32, src=_lib.DT_BF16, wd=_lib.DT_BF16, od=_lib.DT_E4M3,
          x=256, res=512, w=1024, codes=2048, scales=4096, so=8192, eps=1e-6):
    if fn == "quantize":
        return lib.hb200_quantize_rows(x, codes, scales, M, N, x_rs, c_rs, src, od, 0, None)
    return lib.hb200_rms_norm_quantize(x, res, w, codes, scales, so, M, N, x_rs, res_rs, c_rs, so_rs, src, wd, od, eps, 0, None)


@pytest.mark.parametrize("change,code", [
    ({"src": _lib.DT_E4M3}, _lib.ERR_BAD_DTYPE), ({"od": _lib.DT_BF16}, _lib.ERR_BAD_DTYPE), ({"wd": _lib.DT_FP16}, _lib.ERR_BAD_DTYPE),
    ({"M": 0}, _lib.ERR_BAD_SHAPE), ({"N": 0}, _lib.ERR_BAD_SHAPE), ({"M": 1 << 31}, _lib.ERR_BAD_SHAPE), ({"N": (1 << 30) + 1}, _lib.ERR_BAD_SHAPE),
    ({"x_rs": 31}, _lib.ERR_BAD_STRIDE), ({"c_rs": 31}, _lib.ERR_BAD_STRIDE), ({"res_rs": 0}, _lib.ERR_BAD_STRIDE), ({"so_rs": 16}, _lib.ERR_BAD_STRIDE),
    ({"x": 257}, _lib.ERR_ALIGN), ({"res": 513}, _lib.ERR_ALIGN), ({"w": 1025}, _lib.ERR_ALIGN), ({"so": 8193}, _lib.ERR_ALIGN), ({"scales": 4098}, _lib.ERR_ALIGN),
    ({"x": None}, _lib.ERR_ALIGN), ({"w": None}, _lib.ERR_ALIGN), ({"codes": None}, _lib.ERR_ALIGN), ({"res": None}, _lib.ERR_ALIGN), ({"so": None}, _lib.ERR_ALIGN),
    ({"eps": -1.0}, _lib.ERR_BAD_CONFIG), ({"eps": 0.0}, _lib.ERR_BAD_CONFIG), ({"eps": float("inf")}, _lib.ERR_BAD_CONFIG), ({"eps": float("nan")}, _lib.ERR_BAD_CONFIG),
])
def test_entry_points_check_their_arguments(built_library, change, code):
    assert _call(built_library, **change) == code
    assert "rms_norm_quantize" in _lib.last_error()


def test_quantize_rows_entry_point_checks_its_arguments(built_library):
    assert _call(built_library, "quantize", od=_lib.DT_FP32) == _lib.ERR_BAD_DTYPE
    assert _call(built_library, "quantize", x_rs=8) == _lib.ERR_BAD_STRIDE
    assert _call(built_library, "quantize", scales=None) == _lib.ERR_ALIGN
    assert "quantize_rows" in _lib.last_error()
