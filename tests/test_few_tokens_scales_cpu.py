"""CPU: what a layer for a few tokens does with the scales of 4-bit weights before its kernels run: nothing."""
import copy
import pickle

import pytest
import torch


def layer(native, recipe, inference=False):
    E, H, I, K = 2, 64, 64, 1
    with torch.inference_mode(inference):
        if recipe == "mxfp4":
            s13, s2 = (torch.full((E, n, k // 32), 120, dtype=torch.uint8) for n, k in ((2 * I, H), (H, I)))
        else:
            s13, s2 = (torch.ones(E, n, k // 32, dtype=torch.bfloat16) for n, k in ((2 * I, H), (H, I)))
    kind = torch.float4_e2m1fn_x2 if recipe == "mxfp4" else torch.uint8
    w13, w2 = (torch.zeros(E, n, k // 2, dtype=torch.uint8).view(kind) for n, k in ((2 * I, H), (H, I)))
    return native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E, few_tokens=True)


def call(layer):
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    layer.apply(torch.empty_like(x), x, torch.ones(3, 1), torch.zeros(3, 1, dtype=torch.int32))


@pytest.mark.parametrize("recipe", ["mxfp4", "int4"])
@pytest.mark.parametrize("inference", [False, True])
def test_a_call_reads_no_scales_on_the_host(native, recipe, inference):
    """It gets as far as the native code's first check, whatever the scales are, and leaves no tensor on the layer."""
    c = layer(native, recipe, inference)
    before = {n for n, v in vars(c).items() if isinstance(v, (torch.Tensor, tuple, list))}
    with pytest.raises(NotImplementedError, match="no CPU path"):
        call(c)
    assert {n for n, v in vars(c).items() if isinstance(v, (torch.Tensor, tuple, list))} == before


@pytest.mark.parametrize("recipe", ["mxfp4", "int4"])
def test_copies_of_a_layer(native, recipe):
    c = layer(native, recipe)
    for other in (copy.copy(c), copy.deepcopy(c), pickle.loads(pickle.dumps(c)) if recipe == "int4" else copy.copy(c)):
        with pytest.raises(NotImplementedError, match="no CPU path"):
            call(other)
