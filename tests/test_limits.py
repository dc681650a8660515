"""The largest sizes that the operators take: what lies beyond is refused before any work."""
from __future__ import annotations

import pytest
import torch


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
