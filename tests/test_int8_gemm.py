"""Refusals of the int8 GEMM, in Python and at the C entry point: no GPU is touched."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib


def test_operator_refuses_what_it_does_not_take():
    import helion_b200 as hb

    x = torch.zeros(16, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.int8_gemm(x, x)
    with pytest.raises(TypeError, match="expects int8"):
        hb.int8_gemm(x.float(), x)
    with pytest.raises(ValueError, match="2-D"):
        hb.int8_gemm(x[0], x)
    with pytest.raises(AssertionError, match="size mismatch 16 != 8"):
        hb.int8_gemm(x, x[:8])
    with pytest.raises(TypeError, match="out_dtype"):
        hb.int8_gemm(x, x, out_dtype=torch.int32)


def _call(lib, M=64, N=64, K=64, x_rs=64, x_cs=1, y_rs=1, y_cs=64, out_rs=64, dt=_lib.DT_BF16, x=256, y=512, out=1024, sa=4096, sb=8192, mode=2, cfg=-1):
    return lib.hb200_int8_gemm(x, y, out, M, N, K, x_rs, x_cs, y_rs, y_cs, out_rs, dt, sa, sb, mode, cfg, 0, None)


@pytest.mark.parametrize("change,code", [
    ({"K": 131072, "x_rs": 131072, "y_cs": 131072}, _lib.ERR_BAD_SHAPE), ({"K": 40}, _lib.ERR_BAD_SHAPE), ({"N": 60}, _lib.ERR_BAD_SHAPE), ({"M": 0}, _lib.ERR_BAD_SHAPE),
    ({"x_cs": 2}, _lib.ERR_BAD_STRIDE), ({"x_rs": 72}, _lib.ERR_BAD_STRIDE), ({"x_rs": 48}, _lib.ERR_BAD_STRIDE), ({"y_rs": 64, "y_cs": 1}, _lib.ERR_BAD_STRIDE),
    ({"y_cs": 48}, _lib.ERR_BAD_STRIDE), ({"out_rs": 32}, _lib.ERR_BAD_STRIDE), ({"dt": _lib.DT_INT8}, _lib.ERR_BAD_DTYPE), ({"x": 264}, _lib.ERR_ALIGN),
    ({"out": None}, _lib.ERR_ALIGN), ({"sa": None}, _lib.ERR_ALIGN), ({"sb": 8194}, _lib.ERR_ALIGN), ({"mode": 3}, _lib.ERR_BAD_CONFIG),
])
def test_entry_point_checks_its_arguments(built_library, change, code):
    assert _call(built_library, **change) == code
    assert "int8_gemm" in _lib.last_error()
