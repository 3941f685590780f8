"""CPU: layers that the form for a few tokens does not take are refused when they are built, not by their small calls."""
import pytest
import torch


@pytest.mark.parametrize("topk,taken", [(32, True), (33, False), (64, False)])
def test_experts_a_token(native, topk, taken):
    w13, w2 = torch.zeros(64, 64, 64, dtype=torch.bfloat16), torch.zeros(64, 32, 64, dtype=torch.bfloat16)
    if taken:
        native.XpuFusedMoe(w13, None, None, w2, None, None, topk, "silu", 64, few_tokens=True)
    else:
        with pytest.raises(NotImplementedError, match="up to 32 experts a token"):
            native.XpuFusedMoe(w13, None, None, w2, None, None, topk, "silu", 64, few_tokens=True)
    native.XpuFusedMoe(w13, None, None, w2, None, None, topk, "silu", 64)
