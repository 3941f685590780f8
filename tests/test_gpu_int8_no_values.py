"""GPU: rows without values have the scale of rows of zeros."""
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (300,), (2, 3)])
def test_scales_of_rows_without_values(native, shape, dtype):
    x, q = torch.empty(*shape, 0, dtype=dtype, device=DEV), torch.empty(*shape, 0, dtype=torch.int8, device=DEV)
    want = ref.quant_rows(x)[1]
    for run in (lambda s: torch.ops._C.b200_quant_int8_rows(x, q, s), lambda s: torch.ops._C.b200_silu_and_mul_quant_int8_rows(q, x, s)):
        s = torch.full(shape, float("nan"), device=DEV)
        run(s)
        assert torch.equal(s.cpu(), want)
