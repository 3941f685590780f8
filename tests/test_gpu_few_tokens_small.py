"""GPU: calls of the layer for a few tokens with up to 32 routed slots, which find their experts in one pass, and what else the tests of
test_gpu_few_tokens leave open: both terms of h next to 16-bit weights, limits on the blocks, tensors that do not fit one another."""
import pytest
import torch

from test_gpu_few_tokens import BF16, DEV, F16, Case, reference

pytestmark = pytest.mark.gpu
RECIPES = ["w16", "fp8", "mxfp4", "int4"]
SLOTS = [(1, 1), (1, 8), (1, 32), (2, 16), (3, 5), (4, 8), (5, 6), (8, 4), (16, 2), (3, 11), (11, 3)]       # 33 slots: the last two


@pytest.mark.parametrize("recipe", RECIPES)
@pytest.mark.parametrize("T,K", SLOTS)
def test_a_rank_of_an_expert_parallel_layer(native, recipe, T, K):
    """Most slots belong to other ranks; by the caller's map and by the layer's own."""
    for rank in range(4):
        c = Case(native, recipe, T, 256, 256, 16, K, ranks=4, rank=rank, seed=10 * T + rank)
        out = c.run()
        c.check(out)
        own = torch.empty_like(out)
        c.layer.apply(own, c.x, c.weights, c.ids)
        assert torch.equal(own, out)


@pytest.mark.parametrize("recipe", RECIPES)
@pytest.mark.parametrize("T,K", SLOTS)
@pytest.mark.parametrize("wide", [False, True])
def test_slots_of_every_kind(native, recipe, T, K, wide):
    """Experts named twice and more by a token, tokens and slots without an expert, everyone at one expert; ids of 32 and 64 bits."""
    c = Case(native, recipe, T, 256, 256, 6, K, seed=T + K)
    g = torch.Generator().manual_seed(T * K)
    low, high = (-(1 << 40), (1 << 32) + 1) if wide else (-(1 << 31), 1 << 30)
    kinds = [torch.randint(0, 6, (T, K), generator=g), torch.randint(0, 2, (T, K), generator=g), torch.full((T, K), 5), torch.full((T, K), -1)]
    some = torch.randint(0, 6, (T, K), generator=g)
    some[torch.rand(T, K, generator=g) < 0.3] = low
    some[torch.rand(T, K, generator=g) < 0.3] = high
    some[T // 2] = 6
    kinds.append(some)
    last = torch.full((T, K), -1)
    last[-1, -1] = 3
    kinds.append(last)
    for ids in kinds:
        c.ids = ids.to(DEV, torch.int64 if wide else torch.int32)
        out = c.run()
        c.check(out)
        if not ((ids >= 0) & (ids < 6)).any():
            assert (out == 0).all()


@pytest.mark.parametrize("recipe", RECIPES)
def test_one_token_next_to_the_same_among_others(native, recipe):
    """A slot more and the experts are found the other way: the token's rows of both calls are within their bounds."""
    c = Case(native, recipe, 9, 256, 384, 12, 4, bias=True, seed=2)
    c.check(c.run())
    for T in (1, 8):
        few = Case(native, recipe, 9, 256, 384, 12, 4, bias=True, seed=2)
        few.x, few.ids, few.weights, few.T = c.x[:T], c.ids[:T], c.weights[:T], T
        few.check(few.run())


@pytest.mark.parametrize("dtype,small", [(BF16, 2.0 ** -9), (F16, 2.0 ** -13)], ids=str)
@pytest.mark.parametrize("T", [1, 3, 16])
def test_both_terms_of_h_next_to_16_bit_weights(native, dtype, small, T):
    """h is 20 (1 + small) in one half of the features and 20 in the other, which W2 takes off: with one rounding to 16 bits nothing is
    left.  Two terms leave 2^-16 of a bfloat16 h, 2^-22 of a float16 one."""
    H, I = 64, 64
    c = Case(native, "w16", T, H, I, 2, 1, dtype=dtype)
    w13, w2 = torch.zeros_like(c.w13), torch.zeros_like(c.w2)
    w13[:, 0, :I] = 20.0
    w13[:, 0, I:] = 1.0
    w13[:, 1, I:I + I // 2] = small
    w2[:, :I // 2], w2[:, I // 2:] = 1.0, -1.0
    c.w13.copy_(w13)
    c.w2.copy_(w2)
    c.d13, c.d2 = w13.double().transpose(1, 2), w2.double().transpose(1, 2)
    c.x.zero_()
    c.x[:, :2] = 1.0
    c.h_half = 2.0 ** -16 if dtype == BF16 else 2.0 ** -22
    c.weights.fill_(1.0)
    ref, bound = reference(c.x, c.weights, c.ids, c.d13, None, c.d2, None, c.act, None, None, c.h_half, torch.finfo(dtype).eps / 2)
    h = torch.tensor([20 * (1 + small), 20.0], dtype=torch.float64).to(dtype).double()
    # one rounding makes 0 of it, whose error is the result itself: out of the bound
    assert h[0] == h[1] and (ref.abs() > bound).all()
    c.check(c.run())


@pytest.mark.parametrize("recipe,group", [("w16", 0), ("fp8", 0), ("mxfp4", 0), ("int4", 128), ("int4", 32)])
@pytest.mark.parametrize("blocks", [1, 7, 20, 147])
def test_a_limit_on_the_blocks(native, recipe, group, blocks):
    for T in (1, 7):
        c = Case(native, recipe, T, 512, 384, 8, 3, group=group, seed=T)
        c.layer.gemm_max_ctas = blocks
        c.check(c.run())


@pytest.mark.parametrize("recipe", RECIPES)
def test_sizes_that_do_not_fit(native, recipe):
    c = Case(native, recipe, 4, 256, 256, 4, 2, bias=True)
    narrow = c.x[:, :128].contiguous()
    with pytest.raises(RuntimeError, match="K dimension must match|must be \\[num_experts, N, K\\]"):
        c.layer.apply(torch.empty_like(narrow), narrow, c.weights, c.ids)
    other = Case(native, recipe, 4, 256, 512, 4, 2, bias=True)
    for name, message in (("w2", "K dimension must match|must be \\[num_experts, N, K\\]"), ("w13", "N dimension must match|must be \\[num_experts, N, K\\]"),
                          ("w13_bias", "ptr_bias.size\\(1\\) must match N")):
        kept = getattr(c.layer, name)
        setattr(c.layer, name, getattr(other.layer, name))
        with pytest.raises(RuntimeError, match=message):
            c.run()
        setattr(c.layer, name, kept)
    for name in () if recipe == "w16" else ("gemm1_wei_scales", "gemm2_wei_scales"):
        kept = getattr(c.layer, name)
        setattr(c.layer, name, kept[:3])
        with pytest.raises(RuntimeError, match="num_experts|ptr_scales|scales"):
            c.run()
        setattr(c.layer, name, kept)
    c.check(c.run())
