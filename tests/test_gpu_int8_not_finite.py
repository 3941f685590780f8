"""GPU: a NaN or an infinity in a row of an int8 call stays visible behind a clamp and behind activations with limits, in that row alone."""
import pytest
import torch

import int8_ref as ref
from oracle import torch_oracle as to
from test_gpu_int8_layer import _routing, _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("T", [3, 90])            # the kernel for a few rows, and that for many
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("form", [dict(gemm1_clamp_limit=0.7), dict(gemm1_clamp_limit=0.7, fuse_activation=False), dict(activation="gelu"),
                                  dict(activation="gelu_tanh"), dict(activation="swigluoai"), dict(activation="swiglustep"),
                                  dict(activation="relu2_no_mul"), dict(activation="swigluoai", gemm1_clamp_limit=0.7)])
def test_layers(native, T, bad, form):
    gen = torch.Generator().manual_seed(T)
    E, K, H, I = 4, 2, 64, 32
    form = dict(form)
    act = form.pop("activation", "silu")
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    if act == "relu2_no_mul":                      # gemm2 takes both halves
        w2 = torch.cat((w2, w2), dim=-1).contiguous()
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, act, E, **form)
    want, got = (torch.empty(T, H, dtype=B16, device=DEV) for _ in range(2))
    layer.apply(want, x, weights, ids)
    x[2, 5] = bad
    layer.apply(got, x, weights, ids)
    others = torch.arange(T, device=DEV) != 2
    assert torch.isnan(got[2]).all() and torch.isfinite(want).all()
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("counts", [[2, 0, 1], [100, 0, 60]])
@pytest.mark.parametrize("dtype", [B16, F16, F32])
def test_grouped_product_with_a_clamp(native, counts, dtype):
    gen = torch.Generator().manual_seed(sum(counts))
    E, n, k, M = len(counts), 80, 48, sum(counts)
    q, qs = ref.weights(M, k, gen)
    w, ws = ref.weights(n, k, gen, E)
    rows = torch.tensor(counts, dtype=torch.int32, device=DEV)

    def run(scales):
        d = torch.empty(M, n // 2, dtype=dtype, device=DEV)
        torch.ops._xpu_C.b200_grouped_gemm(q, scales, w, ws, None, d, rows, n, k, E, 0, 1, 1.702, 7.0, 1.5)
        return d
    want = run(qs)
    broken = qs.clone()
    broken[1] = float("nan")
    got = run(broken)
    others = torch.arange(M, device=DEV) != 1
    assert torch.isnan(got[1]).all() and torch.isfinite(want).all()
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("dtype", [B16, F16, F32])
@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("op,plain,width", [("swigluoai_and_mul", lambda x: to.swigluoai_and_mul(x, 1.702, 7.0), 2),
                                            ("swiglustep_and_mul", lambda x: to.swiglustep_and_mul(x, 7.0), 2),
                                            ("relu2_no_mul", to.relu2_no_mul, 1)])
def test_activations(native, op, plain, width, d, dtype):
    gen = torch.Generator().manual_seed(d)
    x = (torch.randn(5, width * d, generator=gen) * 6).to(dtype)
    limits = {"swigluoai_and_mul": (1.702, 7.0), "swiglustep_and_mul": (7.0,)}.get(op, ())

    def run(x):
        out = torch.empty(5, d, dtype=dtype, device=DEV)
        getattr(torch.ops._C, op)(out, x.to(DEV), *limits)
        return out.cpu()
    want = run(x)
    x[1, 7] = x[2, 8] = x[3, width * d - 1] = x[4, width * d - 2] = float("nan")
    got, nan = run(x), plain(x.float()).isnan()
    assert nan.sum() == 4 and torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], want[~nan])
