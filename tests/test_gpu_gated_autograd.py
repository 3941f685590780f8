"""GPU: what autograd may ask of the gated product beyond a first gradient: derivatives that it does not have are refused, not dropped, and
gradients that nobody wants are not computed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16 = torch.bfloat16


@pytest.fixture(scope="module")
def gated_linear(native):
    from vllm_xpu_kernels.gated_linear import gated_linear
    return gated_linear


def _inputs(rows=20, hidden=64, inter=24, grad=True):
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, hidden, generator=gen).to(B16).to(DEV).requires_grad_(grad)
    w = (torch.randn(2 * inter, hidden, generator=gen) * hidden ** -0.5).to(B16).to(DEV).requires_grad_(grad)
    return x, w, torch.randn(rows, inter, generator=gen).to(B16).to(DEV)


# ---- forward mode -------------------------------------------------------------------

@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("operand", [0, 1])
def test_forward_mode_is_refused(gated_linear, operand, grad):
    operands = list(_inputs(grad=grad)[:2])
    with torch.autograd.forward_ad.dual_level():
        operands[operand] = torch.autograd.forward_ad.make_dual(operands[operand], torch.ones_like(operands[operand]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_linear(*operands)


def test_jvp_is_refused(gated_linear):
    x, w, _ = _inputs(grad=False)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: gated_linear(t, w), (x,), (torch.ones_like(x),))


def test_a_gradient_with_a_tangent_is_refused(gated_linear):
    x, w, d = _inputs()
    y = gated_linear(x, w)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, torch.autograd.forward_ad.make_dual(d, torch.ones_like(d)))
