"""GPU: what autograd may ask of the gated product beyond a first gradient: derivatives that it does not have are refused, not dropped, and
gradients that nobody wants are not computed."""
import gc

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


# ---- second order -------------------------------------------------------------------

def _odd(x):
    """The same rows, one value off a boundary of 16 bytes: the product reads a copy."""
    room = torch.zeros(x.shape[0], x.shape[1] + 9, dtype=x.dtype, device=x.device)
    return torch.cat((room[:, :1], x, room[:, 1:9]), dim=1)[:, 1:1 + x.shape[1]]


@pytest.mark.parametrize("consumer", ["linear", "nonlinear"])
@pytest.mark.parametrize("wanted", ["x", "w"])
@pytest.mark.parametrize("copied", [False, True])
def test_second_order_terms_are_refused(gated_linear, consumer, wanted, copied):
    x, w, _ = _inputs()
    if wanted == "x":
        w.requires_grad_(False)      # (the gradient of x is one of x alone)
    y = gated_linear(_odd(x) if copied else x, w)
    loss = y.sum() if consumer == "linear" else y.float().pow(2).sum()
    first, = torch.autograd.grad(loss, x if wanted == "x" else w, create_graph=True)
    assert first.requires_grad
    total = loss + first.float().pow(2).sum()          # (a penalty beside a loss that has a graph of its own)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        torch.autograd.grad(total, x, retain_graph=True)
    if wanted == "w":
        with pytest.raises(RuntimeError, match="not differentiable twice"):
            torch.autograd.grad(total, w, retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        total.backward()


def test_the_incoming_gradient_is_not_differentiated_either(gated_linear):
    x, w, d = _inputs()
    d.requires_grad_(True)
    dx, = torch.autograd.grad(gated_linear(x, w), x, d, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        torch.autograd.grad(dx.sum(), d)


def test_a_graph_that_nobody_differentiates_changes_nothing(gated_linear):
    x, w, d = _inputs()
    want = torch.autograd.grad(gated_linear(x, w), (x, w), d)
    got = torch.autograd.grad(gated_linear(x, w), (x, w), d, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    gated_linear(x, w).backward(d, create_graph=True)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    x.grad = w.grad = None


# ---- which gradients ----------------------------------------------------------------

def test_only_the_gradients_that_are_asked_for(gated_linear):
    """... are computed: a call takes no memory for the other one."""
    for rows, hidden, inter, operand in ((8, 2048, 1024, 0), (4096, 2048, 8, 1)):
        x, w, d = _inputs(rows, hidden, inter)
        both = torch.autograd.grad(gated_linear(x, w), (x, w), d)
        y = gated_linear(x, w)
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got, = torch.autograd.grad(y, (x, w)[operand], d)
        grown = torch.cuda.max_memory_allocated() - before
        other = (w, x)[operand]
        assert torch.equal(got, both[operand])
        assert grown < other.numel() * other.element_size(), grown
        y = gated_linear(x, w)
        y.backward(d, inputs=[(x, w)[operand]])
        assert torch.equal((x, w)[operand].grad, both[operand]) and other.grad is None


# ---- capture ------------------------------------------------------------------------

@pytest.mark.parametrize("view", [lambda w: w.view(2, 24, 64).view(48, 64), lambda w: w * 1, lambda w: w.t().t()[:40]])
def test_operands_made_of_a_leaf_that_lives_outside_the_capture_are_refused(gated_linear, view):
    x, w, d = _inputs()
    x.requires_grad_(False)
    alive = gated_linear(x, w)
    for operands in ((lambda: (x, view(w))), (lambda: (view(w), torch.ones(16, 64, dtype=B16, device=DEV)))):
        with pytest.raises(RuntimeError, match="outside this stream capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                gated_linear(*operands())
    del alive
    gc.collect()          # (an exception's frames hold on to what they had)
    want, = torch.autograd.grad(gated_linear(x, view(w)), w, d[:, :view(w).shape[0] // 2])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, = torch.autograd.grad(gated_linear(x, view(w)), w, d[:, :view(w).shape[0] // 2])
    g.replay()
    assert torch.equal(got, want)


def test_a_leaf_of_another_stream_of_the_same_capture_is_taken(gated_linear):
    x, w, d = _inputs()
    want = torch.autograd.grad(gated_linear(x, w), (x, w), d)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            view = w * 1                          # (w's accumulator belongs to the side stream)
            keep = w.view(-1)
        main.wait_stream(side)
        y = gated_linear(x, view)
        got = torch.autograd.grad(y, (x, w), d)
        main.wait_stream(side)
    g.replay()
    assert keep.requires_grad and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("made", [lambda w: w, lambda w: w * 1])
def test_a_leaf_of_a_graph_on_another_stream_outside_the_capture_is_taken(gated_linear, made):
    """(That stream joins the capture.  Modules whose hooks keep the leaves' nodes for good are set up so.)"""
    x, w, d = _inputs()
    want = torch.autograd.grad(gated_linear(x, w), (x, w), d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = gated_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(gated_linear(x, made(w)), (x, w), d)
    g.replay()
    assert alive.requires_grad and all(torch.equal(a, b) for a, b in zip(got, want))


# ---- range --------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [6, 300])
def test_float16_gradients_that_overflow_between_the_kernels_show(gated_linear, rows):
    """dg and du are float16: the row and the weight row of one beyond 65504 have gradients that are not finite, and no others.  Every weight row is
    a unit vector, so that g and u are values of x."""
    gen = torch.Generator().manual_seed(rows)
    x, d = torch.randn(rows, 64, generator=gen), torch.randn(rows, 24, generator=gen)
    x[1, 3], x[1, 24 + 3], d[1, 3] = 8.0, 100.0, 1000.0         # dg = 1000 * 100 * 1.002..., du = 1000 * 8 * 0.9996...
    x[4, 5], x[4, 24 + 5], d[4, 5] = 100.0, 0.0, 1000.0         # dg = 0, du = 1000 * 100
    x, d, w = x.half().to(DEV).requires_grad_(True), d.half().to(DEV), torch.eye(64)[:48].half().to(DEV).requires_grad_(True)
    dx, dw = torch.autograd.grad(gated_linear(x, w), (x, w), d)
    broken_rows, broken_features = torch.zeros(rows, dtype=torch.bool, device=DEV), torch.zeros(48, dtype=torch.bool, device=DEV)
    broken_rows[1] = broken_rows[4] = broken_features[3] = broken_features[24 + 5] = True
    g, u = (x.detach().double() @ w.detach().double().t()).chunk(2, -1)
    both = torch.cat((d.double() * u * torch.sigmoid(g) * (1 + g * (1 - torch.sigmoid(g))), d.double() * g * torch.sigmoid(g)), -1)
    # (dw[24 + 3, 24 + 3] is 8000 * 100 and more: that one value is beyond float16 itself, without any help)
    for got, exact, broken in ((dx, both @ w.detach().double(), broken_rows), (dw, both.t() @ x.detach().double(), broken_features)):
        assert not torch.isfinite(got[broken]).any()
        assert torch.isfinite(got[~broken][exact[~broken].abs() < 65000]).all()
        assert (exact[~broken].abs() >= 65000).sum() <= 1
