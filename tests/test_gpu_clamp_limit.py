"""GPU: ``gemm1_clamp_limit`` with SwigluOAI, whose gates are the even and whose ups the odd features: every form of a layer (two
kernels for a few tokens, activation in the first GEMM's epilogue, activation as a kernel of its own) limits gates and ups.

Two roundings to e4m3 (rows and h: half a step, 2^-4, whose mean square over a binade is below (2^-4)^2 / 3) are the most that a form
has; they pass on with factors of at most 1.2 (|d (g sigmoid(1.702 g))|) and 1 + limit: sqrt((1.2 * 1.5)^2 + 1) * 2^-4 / sqrt(3) of
h's magnitude before the limits, at random signs.  2^-3 leaves room for rows whose limits take away a part of that
magnitude, and a layer that limits the halves of the features instead is farther away than 2^-1.
"""
import pytest
import torch

from test_gpu_few_tokens import BF16, Case

pytestmark = pytest.mark.gpu
LIMIT = 0.5


def formula(c, halves=False):
    """In 64 bits; `halves`: the limit on features [0, I) and [I, 2I)."""
    out = torch.zeros(c.x.shape, dtype=torch.float64, device=c.x.device)
    for t in range(c.x.shape[0]):
        for k in range(c.ids.shape[1]):
            e = int(c.ids[t, k])
            a = c.d13[e] @ c.x[t].double()
            if halves:
                a[:a.numel() // 2].clamp_(max=LIMIT)
                a[a.numel() // 2:].clamp_(-LIMIT, LIMIT)
            gate, up = a[0::2], a[1::2]
            if not halves:
                gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
            gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0)
            out[t] += c.weights[t, k].double() * (c.d2[e] @ ((up + 1) * gate * torch.sigmoid(1.702 * gate)))
    return out


FORMS = [("w16", dict(few=True)), ("w16", dict(few=False)), ("w16", dict(few=False, fuse_activation=False)),
         ("fp8", dict(few=True)), ("fp8", dict(few=False)), ("fp8_kn", dict(few=True)), ("fp8_kn", dict(few=False)),
         ("mxfp4", dict(few=True)), ("mxfp4", dict(few=False)), ("mxfp4", dict(few=False, fuse_activation=False)),
         ("mxfp4", dict(few=False, mxfp4_activations="bf16")),
         ("mxfp4", dict(few=False, mxfp4_activations="bf16", fuse_activation=False)),
         ("int4", dict(few=True)), ("int4", dict(few=False)), ("int4", dict(few=False, fuse_activation=True))]


@pytest.mark.parametrize("recipe,form", FORMS, ids=str)
@pytest.mark.parametrize("T", [3, 16])
def test_every_form_limits_gates_and_ups(native, recipe, form, T):
    c = Case(native, recipe, T, 256, 384, 4, 2, dtype=BF16, act="swigluoai", clamp=LIMIT, seed=T, **form)
    c.x *= 3
    want = formula(c)
    assert (formula(c, halves=True) - want).norm() >= 2.0 ** -1 * want.norm()
    assert (c.run().double() - want).norm() <= 2.0 ** -3 * want.norm()


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_sixteen_and_seventeen_tokens(native, recipe):
    """The sixteen tokens that a call of two kernels has in common with one of seventeen."""
    c = Case(native, recipe, 17, 256, 384, 4, 2, act="swigluoai", clamp=LIMIT, seed=17)
    c.x *= 3
    more = c.run()
    few = torch.empty_like(c.x[:16])
    c.layer.apply(few, c.x[:16], c.weights[:16], c.ids[:16])
    assert (few.double() - more[:16].double()).norm() <= 2.0 ** -3 * more[:16].double().norm()


@pytest.mark.parametrize("recipe", ["w16", "fp8"])
def test_rows_that_are_sorted_already(native, recipe):
    c = Case(native, recipe, 8, 256, 384, 1, 1, act="swigluoai", clamp=LIMIT, few=False, fuse_activation=False, seed=3)
    c.x *= 3
    c.ids.zero_()
    c.weights.fill_(1.0)
    rows, scale = c.x, None
    if recipe == "fp8":
        rows, scale = torch.empty(8, 256, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(8, 2, device="cuda")
        torch.ops._C.per_token_group_fp8_quant(c.x, rows, scale, 128, 1e-10, -448.0, 448.0, False, False, False)
    out = torch.empty_like(c.x)
    c.layer.apply_sorted(out, rows, torch.tensor([8], dtype=torch.int32, device="cuda"), scale)
    want = formula(c)
    assert (out.double() - want).norm() <= 2.0 ** -3 * want.norm()
