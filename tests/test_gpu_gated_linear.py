"""The gated product and its gradients against 64 bits."""
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def gl(native):
    import vllm_xpu_kernels.gated_linear as module
    return module


def _inputs(rows, hidden, inter, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + rows + hidden + inter)
    x = torch.randn(rows, hidden, generator=gen).to(dtype).to(DEV)
    w = (torch.randn(2 * inter, hidden, generator=gen) * hidden ** -0.5).to(dtype).to(DEV)
    d = torch.randn(rows, inter, generator=gen).to(dtype).to(DEV)
    return x, w, d


class Exact:
    """Results in 64 bits, and how far fp32 sums and 16-bit roundings may be off them."""

    def __init__(self, x, w, d=None):
        half, dtype = w.shape[0] // 2, x.dtype
        step = torch.finfo(dtype).eps / 2
        least = torch.finfo(dtype).smallest_normal * step
        x, w = x.double(), w.double()
        H, T = x.shape[1], x.shape[0]
        g, u = (x @ w.t()).chunk(2, dim=-1)
        # sums of H exact products: each addition is off by at most one unit (2^-23) of a partial sum
        eg, eu = (x.abs() @ w.abs().t() * (H * 2.0 ** -23)).chunk(2, dim=-1)
        self.g, self.u, self.eg, self.eu = g, u, eg, eu
        s = torch.sigmoid(g)
        approx = 2.0 ** -20 + g.abs() * 2.0 ** -23     # of the exponential (its argument is rounded twice), quotient and products
        self.out = g * s * u
        err = 1.1 * u.abs() * eg + (g * s).abs() * eu + self.out.abs() * approx       # |silu'| < 1.1
        self.out_tol = err + (self.out.abs() + err) * step * (1 + 2.0 ** -10) + least
        if d is None:
            return
        d = d.double()
        dg, du = d * u * s * (1 + g * (1 - s)), d * g * s
        # |silu''| <= 1/2; 1 + g (1 - s) is a sum of parts up to 1 + |g|, s is off by `approx` of itself
        eg2 = d.abs() * (0.5 * u.abs() * eg + 1.1 * eu) + (d * u).abs() * s * (1 + g.abs()) * 3 * approx
        eu2 = d.abs() * 1.1 * eg + du.abs() * approx
        both, eb = torch.cat((dg, du), dim=-1), torch.cat((eg2, eu2), dim=-1)
        eb = eb + (both.abs() + eb) * step + least                                     # their rounding to 16 bits
        self.dx, self.dw = both @ w, both.t() @ x
        ex = eb @ w.abs() + (both.abs() + eb) @ w.abs() * (2 * half * 2.0 ** -23)
        ew = eb.t() @ x.abs() + (both.abs() + eb).t() @ x.abs() * (T * 2.0 ** -23)
        self.dx_tol = ex + (self.dx.abs() + ex) * step * (1 + 2.0 ** -10) + least
        self.dw_tol = ew + (self.dw.abs() + ew) * step * (1 + 2.0 ** -10) + least


def _near(got, want, tol, what):
    err = (got.double() - want).abs()
    assert torch.all(err <= tol), f"{what}: {float((err / tol).max())} of the tolerance"


SIZES = [(1, 8, 1), (1, 64, 16), (2, 72, 33), (8, 512, 100), (9, 264, 7), (16, 1024, 256), (17, 128, 8), (33, 200, 130), (128, 512, 129),
         (255, 136, 300), (257, 264, 128), (600, 1032, 520), (40, 4096, 130), (300, 2056, 77), (40, 256, 2100), (3000, 64, 40), (270, 512, 1500)]


@pytest.mark.parametrize("dtype", [B16, F16])
@pytest.mark.parametrize("rows,hidden,inter", SIZES)
def test_forward(gl, rows, hidden, inter, dtype):
    x, w, _ = _inputs(rows, hidden, inter, dtype)
    exact = Exact(x, w)
    out = torch.full((rows, inter), float("nan"), dtype=dtype, device=DEV)
    pre = torch.full((rows, 2 * inter), float("nan"), device=DEV)
    torch.ops._xpu_C.b200_gated_linear(out, x, w, pre)
    _near(out, exact.out, exact.out_tol, "out")
    _near(pre, torch.cat((exact.g, exact.u), -1), torch.cat((exact.eg, exact.eu), -1) + 1e-30, "pre")
    assert torch.equal(gl.gated_linear(x, w), out)


@pytest.mark.parametrize("dtype", [B16, F16])
@pytest.mark.parametrize("rows,hidden,inter", SIZES)
def test_gradients(gl, rows, hidden, inter, dtype):
    x, w, d = _inputs(rows, hidden, inter, dtype)
    x.requires_grad_(True)
    w.requires_grad_(True)
    out = gl.gated_linear(x, w)
    dx, dw = torch.autograd.grad(out, (x, w), d)
    exact = Exact(x.detach(), w.detach(), d)
    _near(out.detach(), exact.out, exact.out_tol, "out")
    _near(dx, exact.dx, exact.dx_tol, "dx")
    _near(dw, exact.dw, exact.dw_tol, "dw")


def test_gradients_against_differences(gl):
    x, w, d = _inputs(40, 64, 24, B16)
    exact = Exact(x, w, d)
    f = lambda a, b: float((ref.silu(a @ b[:24].t()) * (a @ b[24:].t()) * d.double()).sum())  # noqa: E731
    gen = torch.Generator().manual_seed(3)
    vx, vw = torch.randn(x.shape, generator=gen).double().to(DEV), torch.randn(w.shape, generator=gen).double().to(DEV)
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(gl.gated_linear(x, w), (x, w), d)
    a, b, h = x.detach().double(), w.detach().double(), 1e-5
    for got, tol, v, along in ((dx, exact.dx_tol, vx, f(a + h * vx, b) - f(a - h * vx, b)),
                               (dw, exact.dw_tol, vw, f(a, b + h * vw) - f(a, b - h * vw))):
        # (the difference itself: h^2 of a third derivative, and 64-bit sums divided by h)
        assert abs(float((got.double() * v).sum()) - along / (2 * h)) <= float((tol * v.abs()).sum()) + 1e-4


def test_gradient_of_one_operand(gl):
    x, w, d = _inputs(50, 128, 40, F16)
    both = torch.autograd.grad(gl.gated_linear(x.requires_grad_(True), w.requires_grad_(True)), (x, w), d)
    assert torch.equal(torch.autograd.grad(gl.gated_linear(x, w.detach()), x, d)[0], both[0])
    assert torch.equal(torch.autograd.grad(gl.gated_linear(x.detach(), w), w, d)[0], both[1])
    with torch.no_grad():
        assert not gl.gated_linear(x, w).requires_grad


def test_shared_and_broadcast_inputs(gl):
    """A weight used twice, a row given to several calls, an expanded input and an expanded gradient."""
    x, w, d = _inputs(24, 64, 16, B16)
    e = Exact(x, w, torch.ones_like(d))
    x.requires_grad_(True)
    w.requires_grad_(True)
    gl.gated_linear(x, w).sum().backward()                      # (a gradient of stride 0)
    _near(x.grad, e.dx, e.dx_tol, "dx")
    _near(w.grad, e.dw, e.dw_tol, "dw")
    row = x.detach()[:1].clone().requires_grad_(True)
    out = gl.gated_linear(row.expand(24, 64), w)
    got, = torch.autograd.grad(out, row, d)
    many = row.detach().expand(24, 64).contiguous()
    e = Exact(many, w.detach(), d)
    # the sum over the copies is torch's, of values rounded to 16 bits
    _near(got, e.dx.sum(0, keepdim=True), e.dx_tol.sum(0, keepdim=True) + e.dx.abs().sum(0, keepdim=True) * 2.0 ** -7, "row")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(gl.gated_linear(x, w).sum(), x, create_graph=True)[0].sum(), x)


def test_layouts(gl):
    x, w, d = _inputs(30, 64, 24, B16)
    want = gl.gated_linear(x, w)
    wide = torch.zeros(30, 80, dtype=B16, device=DEV)
    wide[:, 8:72] = x
    odd = torch.zeros(30, 77, dtype=B16, device=DEV)
    odd[:, 5:69] = x
    for y in (wide[:, 8:72], odd[:, 5:69], x.t().contiguous().t()):
        assert torch.equal(gl.gated_linear(y, w), want)
    assert torch.equal(gl.gated_linear(x.view(2, 3, 5, 64), w).view(30, 24), want)
    assert torch.equal(gl.gated_linear(x[7], w), want[7])
    assert torch.equal(gl.gated_linear(x, w.t().contiguous().t()), want)
    room = torch.full((31, 33), 5.0, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_gated_linear(room[:30, 4:28], wide[:, 8:72], w)
    assert torch.equal(room[:30, 4:28], want) and torch.all(room[30] == 5) and torch.all(room[:, :4] == 5) and torch.all(room[:, 28:] == 5)
    # gradients of rows that are further apart than long
    pre = torch.empty(30, 48, device=DEV)
    out = torch.empty(30, 24, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_gated_linear(out, x, w, pre)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    torch.ops._xpu_C.b200_gated_linear_backward(d, pre, x, w, dx, dw)
    grads = torch.full((30, 37), 5.0, dtype=B16, device=DEV)
    grads[:, 7:31] = d
    dx_room, dw2 = torch.full((30, 71), 5.0, dtype=B16, device=DEV), torch.empty_like(w)
    torch.ops._xpu_C.b200_gated_linear_backward(grads[:, 7:31], pre, wide[:, 8:72], w, dx_room[:, 3:67], dw2)
    assert torch.equal(dx_room[:, 3:67], dx) and torch.equal(dw2, dw)
    assert torch.all(dx_room[:, :3] == 5) and torch.all(dx_room[:, 67:] == 5)


def test_nothing(gl):
    x, w, d = _inputs(4, 64, 24, B16)
    x = x[:0].requires_grad_(True)
    w.requires_grad_(True)
    out = gl.gated_linear(x, w)
    dx, dw = torch.autograd.grad(out, (x, w), d[:0])
    assert out.shape == (0, 24) and dx.shape == (0, 64) and torch.all(dw == 0)
    x = _inputs(4, 64, 24, B16)[0].requires_grad_(True)
    out = gl.gated_linear(x, w[:0])
    dx, = torch.autograd.grad(out, x, torch.empty(4, 0, dtype=B16, device=DEV))
    assert out.shape == (4, 0) and torch.all(dx == 0)


def test_the_same_bits_every_time(gl):
    x, w, d = _inputs(300, 264, 200, B16)
    x.requires_grad_(True)
    w.requires_grad_(True)
    runs = [torch.autograd.grad(gl.gated_linear(x, w), (x, w), d) for _ in range(3)]
    for r in runs[1:]:
        assert torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1])


@pytest.mark.parametrize("rows", [5, 100])
def test_graph_and_other_stream(gl, rows):
    x, w, d = _inputs(rows, 128, 72, B16)
    x2, _, d2 = _inputs(rows, 128, 72, B16, seed=9)

    def step(x, d):
        pre = torch.empty(rows, 144, device=DEV)
        out, dx, dw = torch.empty(rows, 72, dtype=B16, device=DEV), torch.empty_like(x), torch.empty_like(w)
        torch.ops._xpu_C.b200_gated_linear(out, x, w, pre)
        torch.ops._xpu_C.b200_gated_linear_backward(d, pre, x, w, dx, dw)
        return out, dx, dw
    want, want2 = step(x, d), step(x2, d2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, d)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    a, b = x.clone(), d.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(a, b)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    a.copy_(x2)
    b.copy_(d2)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want2))


def test_autograd_under_capture(gl):
    x, w, d = _inputs(20, 64, 24, B16)
    x.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(gl.gated_linear(x, w), (x, w), d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(gl.gated_linear(x, w), (x, w), d)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_leaves_of_a_graph_outside_the_capture_are_refused(gl):
    x, w, d = _inputs(20, 64, 24, B16)
    w.requires_grad_(True)
    alive = gl.gated_linear(x, w)
    with pytest.raises(RuntimeError, match="outside this stream capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gl.gated_linear(x, w)
    want, = torch.autograd.grad(alive, w, d)
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = gl.gated_linear(x, w) + gl.gated_linear(x, w)      # (a leaf used twice inside is none of that)
        loss.backward(d)
    g.replay()
    torch.testing.assert_close(w.grad, 2 * want, rtol=0, atol=0)   # (equal parts: their sum is exact)


def test_two_graphs_replayed_in_turn(gl):
    """Steps of two sizes captured one after the other: each keeps its own workspace."""
    steps, replays = [], []
    for rows, inter in ((40, 72), (150, 130)):
        x, w, d = _inputs(rows, 128, inter, B16)
        pre = torch.empty(rows, 2 * inter, device=DEV)
        out, dx, dw = torch.empty(rows, inter, dtype=B16, device=DEV), torch.empty_like(x), torch.empty_like(w)

        def step(x=x, w=w, d=d, pre=pre, out=out, dx=dx, dw=dw):
            torch.ops._xpu_C.b200_gated_linear(out, x, w, pre)
            torch.ops._xpu_C.b200_gated_linear_backward(d, pre, x, w, dx, dw)
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        steps.append((step, x, (out, dx, dw)))
        replays.append(g)
    gen = torch.Generator().manual_seed(1)
    for turn in range(3):
        wants = []
        for step, x, results in steps:
            x.copy_(torch.randn(x.shape, generator=gen).to(B16))
            step()
            wants.append([r.clone() for r in results])
            for r in results:
                r.fill_(float("nan"))
        for i in (turn % 2, 1 - turn % 2):
            replays[i].replay()
        for (_, _, results), want in zip(steps, wants):
            assert all(torch.equal(r, v) for r, v in zip(results, want))


def test_a_row_that_is_not_finite_stays_alone(gl):
    for rows in (6, 200):
        x, w, d = _inputs(rows, 64, 24, B16)
        want = gl.gated_linear(x, w)
        x[3, 7] = float("nan")
        x[4, 9] = float("inf")
        got = gl.gated_linear(x, w)
        assert torch.isnan(got[3]).all()
        assert not torch.isfinite(got[4]).all()
        others = [r for r in range(rows) if r not in (3, 4)]
        assert torch.equal(got[others], want[others])


def test_refusals(gl):
    x, w, d = _inputs(6, 64, 24, B16)
    out, pre = torch.empty(6, 24, dtype=B16, device=DEV), torch.empty(6, 48, device=DEV)
    op, back = torch.ops._xpu_C.b200_gated_linear, torch.ops._xpu_C.b200_gated_linear_backward
    odd = torch.zeros(6, 66, dtype=B16, device=DEV)
    for args, message in [
        ((out, x, w[:47]), "weight must be"), ((out, x[:, :56], w), "weight must be"), ((out, x, w.half()), "dtype"),
        ((out.half(), x, w), "dtype"), ((out[:, :20], x, w), "out must be"), ((out[:5], x, w), "out must be"),
        ((out, x.float(), w.float()), "only float16 and bfloat16"), ((out, x[:, :60].contiguous(), w[:, :60].contiguous()), "multiples of 8"),
        ((out, x, w[:, ::1].t().contiguous().t()), "contiguous"), ((out, odd[:, :64], w), "multiples of 8"),
        ((out, odd.view(-1)[4:4 + 384].view(6, 64), w), "aligned"), ((out[:1].expand(6, 24), x, w), "overlap|expanded"),
        ((out, x, w, pre.half()), "pre must be"), ((out, x, w, pre[:, :40]), "pre must be"), ((out, x, w.cpu()), "device"),
        ((x[:, :24].contiguous().view(-1)[:144].view(6, 24), x, w, pre.view(-1)[:0]), "pre must be"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            op(*args)
    for args in [(d[:, :20], pre, x, w, None, None), (d.half(), pre, x, w, None, None), (d, pre[:3], x, w, None, None),
                 (d, pre, x, w, x, None), (d, pre, x, w, x[:3], None), (d, pre, x, w, None, w), (d, pre, x, w, None, w[:20])]:
        with pytest.raises(RuntimeError):
            back(*args)
    with pytest.raises(NotImplementedError):
        gl.gated_linear(x.cpu(), w.cpu())
