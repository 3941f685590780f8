"""GPU: weights, scales and biases that are not on the device of a layer call's rows are refused before any launch."""
import pytest
import torch

from test_gpu_few_tokens import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("recipe,names", [("w16", ("w13", "w2", "w13_bias", "w2_bias")),
                                          ("fp8", ("w13", "w2", "gemm1_wei_scales", "gemm2_wei_scales", "w2_bias")),
                                          ("mxfp4", ("w13", "gemm1_wei_scales", "gemm2_wei_scales", "w13_bias")),
                                          ("int4", ("w2", "gemm1_wei_scales", "gemm2_wei_scales"))])
def test_tensors_of_another_device(native, recipe, names, few):
    c = Case(native, recipe, 3, 256, 256, 4, 2, bias=True, few=few)
    want = c.run()
    for name in names:
        kept = getattr(c.layer, name)
        setattr(c.layer, name, kept.cpu())
        with pytest.raises(RuntimeError, match="device of hidden_states"):
            c.run()
        setattr(c.layer, name, kept)
    assert torch.equal(c.run(), want)


def test_sorted_rows(native):
    c = Case(native, "w16", 4, 256, 256, 1, 1, bias=True, few=False)
    c.layer.w2_bias = c.layer.w2_bias.cpu()
    with pytest.raises(RuntimeError, match="device of hidden_states"):
        c.layer.apply_sorted(torch.empty_like(c.x), c.x, torch.tensor([4], dtype=torch.int32, device="cuda"))
