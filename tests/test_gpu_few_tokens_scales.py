"""GPU: the scales of 4-bit weights in the layer for a few tokens are the caller's, as they are when a call runs: written without a
version count, between replays of a graph, in inference mode, with first calls under capture and on two streams."""
import ctypes

import pytest
import torch

from conftest import PKG_DIR
from test_few_tokens_cpu import INT4, MXFP4, FewTokensArgs
from test_gpu_few_tokens import BF16, DEV, E2M1, Case

pytestmark = pytest.mark.gpu
RECIPES = [("mxfp4", 128), ("int4", 128), ("int4", 32)]


def other_scales(s, seed):
    """Scales of the same kind: bytes of the same range, 16-bit scales in another order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if s.dtype == torch.uint8:
        return torch.randint(117, 124, s.shape, generator=g, device=DEV, dtype=torch.uint8)
    return s.flatten()[torch.randperm(s.numel(), generator=g, device=DEV)].view_as(s).clone()


def write(c, seed, how):
    """Other scales in the layer's tensors, and the 64-bit weights that go with them."""
    for s, d, group in ((c.s13, c.d13, None), (c.s2, c.d2, None)):
        new = other_scales(s, seed)
        per = d.shape[-1] // s.shape[-1]
        if s.dtype == torch.uint8:
            d.mul_(torch.exp2(new.double() - s.double()).repeat_interleave(per, 2))
        else:
            d.mul_((new.double() / s.double()).repeat_interleave(per, 2))
        how(s, new)


def counted(s, new):
    s.copy_(new)


def uncounted(s, new):
    before = s._version
    s.data.copy_(new)
    assert s._version == before


def fresh(native, c):
    """The result of a layer object made now, on the same tensors."""
    layer = native.XpuFusedMoe(c.w13, c.s13, c.b13, c.w2, c.s2, c.b2, c.ids.shape[1], c.act, c.w13.shape[0], few_tokens=True)
    out = torch.empty_like(c.x)
    layer.apply(out, c.x, c.weights, c.ids)
    return out


@pytest.mark.parametrize("recipe,group", RECIPES)
@pytest.mark.parametrize("how", [counted, uncounted])
def test_scales_written_between_calls(native, recipe, group, how):
    c = Case(native, recipe, 5, 256, 384, 6, 2, group=group)
    first = c.run()
    c.check(first)
    write(c, 1, how)
    out = c.run()
    assert not torch.equal(out, first)
    c.check(out)
    assert torch.equal(out, fresh(native, c))


@pytest.mark.parametrize("recipe,group", RECIPES)
def test_scales_made_in_inference_mode(native, recipe, group):
    plain = Case(native, recipe, 3, 256, 256, 4, 2, group=group)
    with torch.inference_mode():
        s13, s2 = plain.s13.clone(), plain.s2.clone()
    assert s13.is_inference()
    layer = native.XpuFusedMoe(plain.w13, s13, None, plain.w2, s2, None, 2, "silu", 4, few_tokens=True)
    out = torch.empty_like(plain.x)
    layer.apply(out, plain.x, plain.weights, plain.ids)
    assert torch.equal(out, plain.run())


@pytest.mark.parametrize("recipe,group", RECIPES)
@pytest.mark.parametrize("how", [counted, uncounted])
def test_scales_written_between_replays(native, recipe, group, how):
    """A replayed graph reads what the tensors hold then, also after eager calls with the new scales."""
    c = Case(native, recipe, 5, 256, 384, 6, 2, group=group)
    c.run()
    out, graph, stream = torch.zeros_like(c.x), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        c.run(out)
    for seed in (1, 2, 3):
        write(c, seed, how)
        if seed > 1:
            c.run()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
        assert torch.equal(out, c.run())


@pytest.mark.parametrize("recipe,group", RECIPES)
def test_a_first_call_under_capture(native, recipe, group):
    """Another layer has loaded the kernels; this one's first call is captured, and an eager call and another graph come before its
    first replay."""
    warm = Case(native, recipe, 5, 256, 384, 6, 2, group=group, seed=1)
    warm.run()
    c = Case(native, recipe, 5, 256, 384, 6, 2, group=group, seed=2)
    torch.cuda.synchronize()
    outs, graphs = [torch.zeros_like(c.x) for _ in range(2)], []
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            c.run(out)
        graphs.append(graph)
    eager = c.run()
    c.check(eager)
    for graph, out in reversed(list(zip(graphs, outs))):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("recipe,group", RECIPES)
def test_first_calls_on_two_streams(native, recipe, group):
    for seed in range(4):
        c = Case(native, recipe, 5, 512, 768, 16, 4, group=group, seed=seed)
        streams, outs = [torch.cuda.Stream() for _ in range(2)], []
        torch.cuda.synchronize()
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(c.run())
        torch.cuda.synchronize()
        c.check(outs[0])
        assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("recipe,group", RECIPES)
def test_a_layer_keeps_no_second_copy(native, recipe, group):
    c = Case(native, recipe, 2, 256, 1024, 64, 2, group=group)
    c.layer.persistent_workspace = False
    out = torch.empty_like(c.x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    c.run(out)
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("recipe,H,I,group", [("mxfp4", 32, 32, 0), ("mxfp4", 96, 160, 0), ("mxfp4", 416, 2880, 0), ("mxfp4", 256, 512, 0),
                                              ("int4", 96, 160, 32), ("int4", 64, 192, 64), ("int4", 128, 384, 128), ("int4", 768, 256, 256)])
@pytest.mark.parametrize("T", [1, 11])
def test_what_is_around_the_scales_is_not_used(native, recipe, H, I, group, T):
    """Scales in the middle of memory that holds NaN (bytes of 255): rows of every length modulo four bytes."""
    c = Case(native, recipe, T, H, I, 3, 2, group=group)
    want = c.run()
    c.check(want)
    around = []
    for s in (c.s13, c.s2):
        buf = torch.full((s.numel() * s.element_size() + 256,), 255, dtype=torch.uint8, device=DEV)
        inside = buf[128:-128].view(s.dtype).view_as(s)
        inside.copy_(s)
        around.append(inside)
    layer = native.XpuFusedMoe(c.w13, around[0], None, c.w2, around[1], None, 2, "silu", 3, few_tokens=True)
    out = torch.empty_like(c.x)
    layer.apply(out, c.x, c.weights, c.ids)
    assert torch.equal(out, want)


@pytest.mark.parametrize("recipe,H,I,group", [("mxfp4", 416, 608, 0), ("mxfp4", 40 * 32, 64, 0), ("int4", 96, 160, 32), ("int4", 192, 320, 64),
                                              ("int4", 384, 640, 128), ("int4", 256, 768, 256)])
@pytest.mark.parametrize("T", [1, 12])
def test_scales_that_the_caller_has_laid_out_by_step(native, recipe, H, I, group, T):
    """b200moe_few_tokens_layer of the C ABI with the words of step_scales: the same results, bit for bit."""
    from vllm_xpu_kernels.fused_moe_interface import step_scales
    lib = ctypes.CDLL(str(PKG_DIR / "vllm_xpu_kernels" / "libb200moe.so"))
    lib.b200moe_few_tokens_workspace_bytes.restype = ctypes.c_size_t
    lib.b200moe_last_error.restype = ctypes.c_char_p
    c = Case(native, recipe, T, H, I, 3, 2, group=group)
    out, fmt = torch.empty_like(c.x), MXFP4 if recipe == "mxfp4" else INT4
    s13, s2 = step_scales(c.s13, H), step_scales(c.s2, I)
    need = lib.b200moe_few_tokens_workspace_bytes(T, 2, H, I)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    args = FewTokensArgs()
    for name, value in dict(x=c.x, topk_ids=c.ids, topk_weights=c.weights, out=out, w13=c.layer.w13, w2=c.layer.w2, w13_scale=s13, w2_scale=s2,
                            workspace=ws).items():
        setattr(args, name, value.data_ptr())
    for name, value in dict(workspace_bytes=need, w13_format=fmt, w2_format=fmt, w13_group=group, w2_group=group, num_tokens=T, hidden=H,
                            inter=I, topk=2, num_experts=3, total_experts=3, dtype=2, ids_dtype=5, activation=0).items():
        setattr(args, name, value)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.b200moe_few_tokens_layer(ctypes.byref(args), ctypes.c_void_p(stream)) == 0, lib.b200moe_last_error()
    assert torch.equal(out, c.run())
    c.check(out)
