"""GPU: operands of a grouped GEMM that are not on the device of its rows are refused before any launch."""
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16 = torch.bfloat16


def _refused(call, operands, names):
    want = call(**operands)
    for name in names:
        with pytest.raises(RuntimeError, match="device of ptr_A"):
            call(**{**operands, name: operands[name].cpu()})
    assert torch.equal(call(**operands), want)


@pytest.mark.parametrize("extended", [False, True])
def test_int8(native, extended):
    gen = torch.Generator().manual_seed(1)
    E, N, K, M = 3, 16, 32, 7
    q, qs = ref.weights(M, K, gen)
    w, ws = ref.weights(N, K, gen, E)
    op = torch.ops._xpu_C.b200_grouped_gemm if extended else torch.ops._xpu_C.cutlass_grouped_gemm_interface

    def call(a, s, b, t, bias, d, rows):
        return op(a, s, b, t, bias, d, rows, N, K, E).clone()
    _refused(call, dict(a=q, s=qs, b=w, t=ws, bias=torch.ones(E, N, dtype=B16, device=DEV), d=torch.empty(M, N, dtype=B16, device=DEV),
                        rows=torch.tensor([2, 0, 5], dtype=torch.int32, device=DEV)), ("s", "b", "t", "bias", "d", "rows"))


def test_16_bits(native):
    gen = torch.Generator().manual_seed(2)
    E, N, K, M = 2, 32, 64, 9
    a, b = torch.randn(M, K, generator=gen).to(B16).to(DEV), torch.randn(E, K, N, generator=gen).to(B16).to(DEV)

    def call(a, s, b, bias, d, rows):     # (scales of 16-bit rows are taken and not read)
        return torch.ops._xpu_C.cutlass_grouped_gemm_interface(a, s, b, None, bias, d, rows, N, K, E).clone()
    _refused(call, dict(a=a, s=torch.ones(3), b=b, bias=torch.ones(E, N, dtype=B16, device=DEV), d=torch.empty(M, N, dtype=B16, device=DEV),
                        rows=torch.tensor([4, 5], dtype=torch.int32, device=DEV)), ("b", "bias", "d", "rows"))
