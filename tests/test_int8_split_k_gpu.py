"""More than 128 rows of x with K split: the kernel that is chosen is the one that runs, for every type of the result."""
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


@pytest.mark.parametrize("first", list(HALF_STEP), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(130, 4096, 14336), (512, 2048, 8192), (1024, 1024, 4096), (200, 72, 4112)])
def test_every_type_of_the_result(hb, m, n, k, first):
    """Whichever type comes first; sums exact, one conversion and two products (3 * 2**-24) and the result's half step."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x, y = (torch.randint(-128, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((m, k), (n, k)))
    sa, sb = torch.rand(m, 1, generator=g, device="cuda") * 1e-3 + 1e-4, torch.rand(1, n, generator=g, device="cuda") * 1e-2 + 1e-3
    want = (x.double() @ y.t().double()) * sa.double() * sb.double()
    for out_dtype in (first, *HALF_STEP):
        out = hb.int8_gemm(x, y.t(), scale_a=sa, scale_b=sb, out_dtype=out_dtype)
        torch.testing.assert_close(out.double(), want, rtol=HALF_STEP[out_dtype] + 3 * 2.0**-24, atol=2.0**-25 if out_dtype == torch.float16 else 0)
