"""The largest sizes that the operators take: what lies beyond is refused before any work, in Python and at the C entry points."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib

BEYOND = 2**31 - 511  # a tile of up to 512 rows that starts below this may end past 2**31


def test_int8_operands_longer_than_their_sums_allow():
    """131056 = 131072 - 16 is the longest K: the sums are int32 and K is handled in pieces of 16."""
    import helion_b200 as hb

    for k in (131057, 131071, 131072):
        x, w = torch.zeros(1, k, dtype=torch.int8), torch.zeros(k, 1, dtype=torch.int8)
        with pytest.raises(ValueError, match="131056"):
            hb.int8_gemm(x, w)
        with pytest.raises(ValueError, match="131056"):
            hb.gated_gemm(x, w, w)
    x, w = torch.zeros(1, 131056, dtype=torch.int8), torch.zeros(131056, 1, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.int8_gemm(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.gated_gemm(x, w, w)
    x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    x, w = torch.cat([x.view(torch.uint8)] * 2, 1).view(torch.float8_e4m3fn), torch.cat([w.view(torch.uint8)] * 2).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hb.gated_gemm(x, w, w)


@pytest.mark.parametrize("m,n", [(BEYOND, 64), (2**31 - 1, 64), (64, (BEYOND + 7) // 8 * 8), (64, 2**31 - 8)])
def test_gemm_entry_points_refuse_tiles_past_31_bits(built_library, m, n):
    lib = built_library
    assert lib.hb200_int8_gemm(256, 512, 1024, m, n, 64, 64, 1, 1, 64, n, _lib.DT_BF16, None, None, 0, -1, 0, None) == _lib.ERR_BAD_SHAPE
    assert "int8_gemm" in _lib.last_error()
    assert lib.hb200_gemm_16bit(256, 512, 1024, m, n, 64, 64, 1, 1, 64, n, _lib.DT_BF16, _lib.DT_BF16, None, 0, -1, 0, None) == _lib.ERR_BAD_SHAPE
    assert lib.hb200_fp8_gemm(256, 512, 1024, m, n, 64, 64, 1, 1, 64, n, _lib.DT_BF16, -1, None, 0, 0, None) == _lib.ERR_BAD_SHAPE


@pytest.mark.parametrize("m,f", [(BEYOND, 64), (2**31 - 1, 64), (64, 2**30 - 504), (64, 2**30)])
def test_gated_entry_points_refuse_tiles_past_31_bits(built_library, m, f):
    lib = built_library
    assert lib.hb200_gated_gemm(256, 512, 768, 1024, m, f, 64, 64, 1, 64, 1, 64, f, _lib.DT_BF16, _lib.DT_BF16, 0, None, None, None, 0, None, None, 0, None) == _lib.ERR_BAD_SHAPE
    assert "gated_gemm" in _lib.last_error()
    got = lib.hb200_gated_gemm_backward(256, 512, 768, 1024, 2048, 4096, 8192, 16384, 32768, m, f, 64, f, 64, 1, 64, 1, 64, _lib.DT_BF16, 65536, 1 << 60, 0, None)
    assert got == _lib.ERR_BAD_SHAPE and "gated_gemm_backward" in _lib.last_error()
