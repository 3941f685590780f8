"""CPU: the checks that b200moe_few_tokens_layer makes before any launch, the scales as its kernels read them, and what
``XpuFusedMoe(few_tokens=True)`` refuses."""
import ctypes

import pytest
import torch

from conftest import PKG_DIR

W16, W16_NK, FP8_NK, MXFP4, INT4 = 0, 1, 3, 5, 7


class FewTokensArgs(ctypes.Structure):
    """b200moe_few_tokens_args of include/b200moe.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "topk_ids", "topk_weights", "expert_map", "out", "w13", "w13_scale", "w13_bias",
                                                "w2", "w2_scale", "w2_bias", "workspace")] +
                [("workspace_bytes", ctypes.c_size_t)] +
                [(n, ctypes.c_int) for n in ("w13_format", "w2_format", "w13_group", "w2_group", "num_tokens", "hidden", "inter", "topk",
                                             "num_experts", "total_experts", "dtype", "ids_dtype", "activation")] +
                [(n, ctypes.c_float) for n in ("act_alpha", "act_limit", "clamp_limit")] +
                [("max_ctas", ctypes.c_int), ("status", ctypes.c_void_p)])


def library():
    lib = ctypes.CDLL(str(PKG_DIR / "vllm_xpu_kernels" / "libb200moe.so"))
    lib.b200moe_last_error.restype = ctypes.c_char_p
    lib.b200moe_few_tokens_workspace_bytes.restype = ctypes.c_size_t
    return lib


def arguments(**change):
    a = {n: 256 for n in ("x", "topk_ids", "topk_weights", "out", "w13", "w2", "w13_scale", "w2_scale", "workspace")}
    a.update(workspace_bytes=1 << 30, w13_format=FP8_NK, w2_format=FP8_NK, num_tokens=4, hidden=256, inter=256, topk=2,
             num_experts=8, total_experts=8, dtype=2, ids_dtype=5)
    a.update(change)
    args = FewTokensArgs()
    for name, value in a.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("change,message", [
    (dict(dtype=0), b"bfloat16 or float16"),
    (dict(num_tokens=17), b"at most 16 tokens"),
    (dict(num_tokens=-1), b"at most 16 tokens"),
    (dict(hidden=0), b"between 1 and 2^20"),
    (dict(inter=(1 << 20) + 1), b"between 1 and 2^20"),
    (dict(topk=0), b"topk must be in"),
    (dict(topk=33), b"topk must be in"),
    (dict(num_experts=0), b"num_experts must be in"),
    (dict(num_experts=1025), b"num_experts must be in"),
    (dict(ids_dtype=2), b"topk_ids must be int32 or int64"),
    (dict(activation=99), b"unknown activation"),
    (dict(w13=None), b"w13 or its scales are missing"),
    (dict(w2_scale=None), b"w2 or its scales are missing"),
    (dict(inter=192), b"needs sizes divisible by 128"),
    (dict(w13_format=MXFP4, w2_format=MXFP4, inter=40), b"rows of a multiple of 32"),
    (dict(w13_format=INT4, w2_format=INT4, w13_group=48, w2_group=32), b"groups of 32, 64, 128 or 256"),
    (dict(w13_format=INT4, w2_format=INT4, w13_group=128, w2_group=128, inter=320), b"groups of 32, 64, 128 or 256"),
    (dict(w13_format=W16), b"the same format"),
    (dict(x=None), b"null pointer"),
    (dict(out=None), b"null pointer"),
])
def test_refused_before_any_launch(change, message):
    lib = library()
    assert lib.b200moe_few_tokens_layer(ctypes.byref(arguments(**change)), None) == -1
    assert message in lib.b200moe_last_error()


def test_refused_formats_and_workspaces():
    lib = library()
    assert lib.b200moe_few_tokens_layer(None, None) == -1
    assert lib.b200moe_few_tokens_layer(ctypes.byref(arguments(w13_format=W16_NK, w2_format=W16_NK)), None) not in (0, -1)
    assert b"16-bit [E,K,N], block-scaled fp8, MXFP4 and int4 weights only" in lib.b200moe_last_error()
    need = lib.b200moe_few_tokens_workspace_bytes(4, 2, 256, 256)
    for change in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=264)):
        assert lib.b200moe_few_tokens_layer(ctypes.byref(arguments(**change)), None) not in (0, -1)
        assert f"needs {need} bytes".encode() in lib.b200moe_last_error()
    assert lib.b200moe_few_tokens_layer(ctypes.byref(arguments(num_tokens=0, x=None, workspace=None)), None) == 0


def test_workspace_holds_h_and_the_shares():
    lib = library()
    for T, K, H, I in ((1, 1, 8, 8), (16, 8, 7168, 2048), (16, 32, 256, 65536), (3, 2, 16384, 100)):
        need = lib.b200moe_few_tokens_workspace_bytes(T, K, H, I)
        assert need >= T * K * I * 4 + 9 * T * H * 4 + 160 * 4
    assert lib.b200moe_few_tokens_workspace_bytes(0, 1, 8, 8) == 0


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("K", [256, 512, 768, 1536])
def test_step_scales_of_int4(group, K):
    """Words of two scales: group 32 and 64 those of 64 or 128 values, from 128 on those of 256."""
    from vllm_xpu_kernels.fused_moe_interface import step_scales
    E, N = 2, 5
    s = torch.arange(E * N * (K // group), dtype=torch.int16).view(E, N, K // group).view(torch.float16)
    words = step_scales(s, K)
    lib = library()
    assert words.dtype == torch.int32 and words.shape == (E, lib.b200moe_few_tokens_scale_words(INT4, group, K), N)
    per = {32: 32, 64: 64}.get(group, 128)                    # values per half of a word
    halves = words.transpose(1, 2).contiguous().view(torch.int16)   # [E, N, 2 words]
    for i in range(halves.shape[-1]):
        want = s.view(torch.int16)[:, :, i * per // group] if i * per < K else torch.zeros(E, N, dtype=torch.int16)
        assert torch.equal(halves[:, :, i], want)


@pytest.mark.parametrize("K", [32, 96, 128, 2880])
def test_step_scales_of_mxfp4(K):
    from vllm_xpu_kernels.fused_moe_interface import step_scales
    E, N = 3, 7
    s = torch.randint(0, 256, (E, N, K // 32), dtype=torch.uint8)
    words = step_scales(s, K)
    assert words.shape == (E, library().b200moe_few_tokens_scale_words(MXFP4, 0, K), N) and words.is_contiguous()
    rows = words.transpose(1, 2).contiguous().view(torch.uint8)
    assert torch.equal(rows[:, :, :K // 32], s) and not rows[:, :, K // 32:].any()


def test_scale_words_of_other_formats():
    lib = library()
    assert lib.b200moe_few_tokens_scale_words(FP8_NK, 128, 256) == 0 and lib.b200moe_few_tokens_scale_words(MXFP4, 0, 0) == 0


def test_layers_that_have_no_such_form(native):
    w13, w2 = torch.zeros(2, 64, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="relu2_no_mul"):
        native.XpuFusedMoe(w13[..., :32].contiguous(), None, None, w2, None, None, 2, "relu2_no_mul", 2, few_tokens=True)
    q13, q2 = w13.to(torch.float8_e4m3fn), w2.to(torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError, match="16-bit, block-scaled fp8, MXFP4 and int4"):
        native.XpuFusedMoe(q13, torch.ones(2), None, q2, torch.ones(2), None, 2, "silu", 2, few_tokens=True)
