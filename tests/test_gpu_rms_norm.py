"""GPU: the norm with the residual's addition and 8-bit rows (torch.ops._C.b200_add_rms_norm) against its
formula in 64 bits.

Bounds, before any rounding to fewer bits: a thread sums at most hidden / 32 squares one after the other (at
least 32 threads a row, each addition and product 2^-24 of it at most), the joins of the threads add 12 more; the mean's
error halves under the root; root, product with the root and with the weight, and what they start from, are 8 roundings
of 2^-24 at most.  A rounding to T is eps(T) / 2 of the value, or half the smallest subnormal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
T16 = [torch.bfloat16, torch.float16]
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}


def fp32_bound(hidden):
    return ((hidden / 32 + 12) / 2 + 8) * 2.0 ** -24


def call(x, residual, weight, out, q, scales, group=0, pow2=False, eps=1e-6):
    torch.ops._C.b200_add_rms_norm(x, residual, weight, eps, out, q, scales, group, pow2)


def reference(x, residual, weight, eps=1e-6):
    """-> the residual as it is stored, y in 64 bits."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = s.double()
    y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    return s, y if weight is None else y * weight.double()


def check(x, residual0, residual, weight, out, q, scales, group, pow2):
    hidden = x.shape[-1]
    s, y = reference(x, residual0, weight)
    fp = fp32_bound(hidden)
    if residual is not None:
        assert torch.equal(residual, s)
    if out is not None:
        half = torch.finfo(out.dtype).eps / 2
        assert ((out.double() - y).abs() <= y.abs() * (half + fp * (1 + half)) + SMALLEST[out.dtype] / 2).all()
    if q is not None:
        g = group or hidden
        parts = y.view(-1, hidden // g, g)
        want = (parts.abs().amax(-1) / 448).clamp(min=1 / (448 * 512))
        got = scales.double()
        if pow2:
            low, high = (torch.exp2(torch.ceil(torch.log2(want * f))) for f in (1 - 2 * fp, 1 + 2 * fp))
            assert ((got == low) | (got == high)).all()
        else:
            assert ((got - want).abs() <= want * (fp + 3 * 2.0 ** -24)).all()
        codes = q.double().view_as(parts)
        real = parts / got[..., None]
        slack = 2.0 ** -4 + 2 * fp
        assert ((codes - real).abs() <= real.abs() * slack + 2.0 ** -10 * (1 + slack)).all()


def make(rows, hidden, dtype, with_residual, weight_dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g, device=DEV).to(dtype)
    residual = (3 * torch.randn(rows, hidden, generator=g, device=DEV)).to(dtype) if with_residual else None
    weight = None if weight_dtype is None else (1 + 0.3 * torch.randn(hidden, generator=g, device=DEV)).to(weight_dtype)
    return x, residual, weight


def outputs(rows, hidden, dtype, group, with_out=True, with_q=True):
    out = torch.empty(rows, hidden, dtype=dtype, device=DEV) if with_out else None
    q = torch.empty(rows, hidden, dtype=torch.float8_e4m3fn, device=DEV) if with_q else None
    scales = torch.empty(rows, hidden // (group or hidden), dtype=torch.float32, device=DEV) if with_q else None
    return out, q, scales


SIZES = [(1, 1, 0), (1, 1, 1), (3, 17, 0), (2, 24, 8), (1, 32, 32), (5, 96, 48), (4, 512, 128), (1, 7168, 128), (3, 1411, 0),
         (3, 1411, 83), (7, 2880, 0), (7, 2880, 96), (33, 2048, 32), (2, 9000, 0), (2, 65536, 128), (2, 131080, 0), (1, 40960, 64),
         (300, 264, 0), (70, 4096, 64), (9, 4104, 8), (5, 4100, 4), (3, 1024, 256), (3, 2048, 1024)]


@pytest.mark.parametrize("dtype", T16 + [torch.float32], ids=str)
@pytest.mark.parametrize("rows,hidden,group", SIZES)
def test_sizes_and_groups(native, rows, hidden, group, dtype):
    """Every size with all outputs, in turn with the 16-bit rows or the 8-bit rows alone."""
    for seed, (with_residual, weight_dtype, with_out, with_q, pow2) in enumerate(
            [(True, dtype, True, True, False), (False, torch.float32, True, False, False), (True, None, False, True, True)]):
        x, residual, weight = make(rows, hidden, dtype, with_residual, weight_dtype, seed)
        before = None if residual is None else residual.clone()
        out, q, scales = outputs(rows, hidden, dtype, group, with_out, with_q)
        call(x, residual, weight, out, q, scales, group, pow2)
        check(x, before, residual, weight, out, q, scales, group, pow2)


@pytest.mark.parametrize("hidden,group", [(512, 128), (1411, 83), (2880, 0), (7168, 64)])
def test_eight_bit_rows_are_those_of_the_quantiser(native, hidden, group):
    """For fp32 rows `out` is y itself: the quantisation op makes the same codes and scales of it."""
    x, residual, weight = make(19, hidden, torch.float32, True, torch.float32, 5)
    for pow2 in (False, True):
        out, q, scales = outputs(19, hidden, torch.float32, group)
        call(x, residual.clone(), weight, out, q, scales, group, pow2)
        q2, s2 = torch.empty_like(q), torch.empty_like(scales)
        if group:
            torch.ops._C.per_token_group_fp8_quant(out, q2, s2, group, 1e-10, -448.0, 448.0, pow2, False, False)
            assert torch.equal(scales, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
        elif not pow2:   # one scale a row is taken from the largest |s * weight|: two roundings apart
            torch.ops._C.per_token_group_fp8_quant(out, q2, s2, hidden, 1e-10, -448.0, 448.0, pow2, False, False)
            assert ((scales - s2).abs() <= 3 * 2.0 ** -24 * s2).all()


@pytest.mark.parametrize("dtype", T16, ids=str)
@pytest.mark.parametrize("hidden,group", [(2048, 128), (1030, 0)])
def test_strided_rows(native, hidden, group, dtype):
    """Rows inside wider buffers, whose other columns stay as they are; scales group-major."""
    rows = 11
    wide = torch.randn(rows, hidden + 72, device=DEV).to(dtype)
    x = wide[:, 8:8 + hidden]
    rbuf = torch.randn(rows, hidden + 40, device=DEV).to(dtype)
    obuf = torch.full((rows, hidden + 24), 7.0, device=DEV).to(dtype)
    qbuf = torch.full((rows, hidden + 16), 3.0, device=DEV).to(torch.float8_e4m3fn)
    groups = hidden // (group or hidden)
    scales = torch.empty(groups, rows, device=DEV).t()
    weight = torch.rand(hidden, device=DEV).to(dtype)
    residual, out, q = rbuf[:, 16:16 + hidden], obuf[:, 8:8 + hidden], qbuf[:, 16:16 + hidden]
    before, edge = residual.clone(), rbuf.clone()
    call(x, residual, weight, out, q, scales, group)
    check(x.contiguous(), before, residual, weight, out, q, scales, group, False)
    assert torch.equal(rbuf[:, :16], edge[:, :16]) and torch.equal(rbuf[:, 16 + hidden:], edge[:, 16 + hidden:])
    assert (obuf[:, :8] == 7).all() and (obuf[:, 8 + hidden:] == 7).all()
    assert (qbuf[:, :16].float() == 3).all() and (qbuf[:, 16 + hidden:].float() == 3).all()


def test_odd_addresses_and_more_dimensions(native):
    """Rows that begin in the middle of 16 bytes, and leading dimensions."""
    buf = torch.randn(2 * 3 * 256 + 3, device=DEV).to(torch.bfloat16)
    x = buf[3:].view(2, 3, 256)
    residual, weight = torch.randn_like(x), torch.rand(256, device=DEV)
    out, q = torch.empty_like(residual), torch.empty(2, 3, 256, device=DEV, dtype=torch.float8_e4m3fn)
    scales = torch.empty(6, 2, device=DEV)
    before = residual.clone()
    call(x, residual, weight, out, q, scales, 128)
    f = lambda t: t.reshape(6, 256)  # noqa: E731
    check(f(x), f(before), f(residual), weight, f(out), f(q), scales, 128, False)


@pytest.mark.parametrize("hidden", [2048, 1411])
@pytest.mark.parametrize("with_residual", [False, True])
def test_in_place(native, hidden, with_residual):
    x, residual, weight = make(6, hidden, torch.bfloat16, with_residual, torch.bfloat16)
    x0, r0 = x.clone(), None if residual is None else residual.clone()
    _, q, scales = outputs(6, hidden, torch.bfloat16, 0)
    call(x, residual, weight, x, q, scales)
    check(x0, r0, residual, weight, x, q, scales, 0, False)


@pytest.mark.parametrize("hidden,group", [(2048, 128), (2048, 0), (1411, 83)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_stay_visible(native, hidden, group, value):
    x, residual, weight = make(3, hidden, torch.bfloat16, True, torch.bfloat16)
    x[1, 5] = value
    out, q, scales = outputs(3, hidden, torch.bfloat16, group)
    call(x, residual, weight, out, q, scales, group)
    assert out[1, 5].isnan() and scales[1, 0].isnan() and q[1, 5].float().isnan()
    assert out[[0, 2]].isfinite().all() and scales[[0, 2]].isfinite().all()


def test_rows_of_zeros(native):
    x = torch.zeros(2, 512, device=DEV, dtype=torch.float16)
    out, q, scales = outputs(2, 512, torch.float16, 128)
    call(x, None, None, out, q, scales, 128)
    assert (out == 0).all() and (q.float() == 0).all() and torch.equal(scales, torch.full_like(scales, 1 / (448 * 512)))


def test_nothing_to_do(native):
    x = torch.empty(0, 512, device=DEV, dtype=torch.float16)
    out, q, scales = outputs(0, 512, torch.float16, 128)
    call(x, None, None, out, q, scales, 128)


def test_another_stream_and_a_graph(native):
    """Captured once, replayed on new inputs in the same buffers: the residual moves on with every replay."""
    x, residual, weight = make(5, 2880, torch.bfloat16, True, torch.bfloat16)
    out, q, scales = outputs(5, 2880, torch.bfloat16, 0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(x, residual, weight, out, q, scales)
    for seed in (1, 2):
        new, _, _ = make(5, 2880, torch.bfloat16, False, None, seed)
        x.copy_(new)
        before = residual.clone()
        graph.replay()
        torch.cuda.synchronize()
        check(x, before, residual, weight, out, q, scales, 0, False)


def test_refusals(native):
    x, residual, weight = make(4, 256, torch.bfloat16, True, torch.bfloat16)
    out, q, scales = outputs(4, 256, torch.bfloat16, 128)
    bad = [
        (dict(out=None, q=None, scales=None), "out or out_q is needed"),
        (dict(scales=None), "go together"),
        (dict(group=100), "divisible by group_size"),
        (dict(group=-1), "divisible by group_size"),
        (dict(group=64), "scales must be float32"),
        (dict(scales=scales.double()), "scales must be float32"),
        (dict(scales=torch.empty(4, 1, device=DEV).expand(4, 2)), "must not be expanded"),
        (dict(weight=weight[:255]), "weight must be contiguous"),
        (dict(weight=weight.to(torch.float16)), "weight must be float32 or"),
        (dict(residual=residual.float()), "residual must have the input's dtype"),
        (dict(residual=residual[:3]), "residual must have the input's shape"),
        (dict(residual=x), "residual must not overlap the input"),
        (dict(residual=residual[:1].expand(4, 256)), "rows of residual must not overlap"),
        (dict(out=out.float()), "out must have the input's dtype"),
        (dict(out=residual), "must not overlap"),
        (dict(out=out.t().contiguous().t()), "last dimension of out"),
        (dict(q=q.view(torch.uint8)), "float8_e4m3fn"),
        (dict(x=x.double(), residual=None, out=None), "only float32, float16 and bfloat16"),
        (dict(weight=weight.cpu()), "input's device"),
    ]
    for change, message in bad:
        a = dict(x=x, residual=residual, weight=weight, out=out, q=q, scales=scales, group=128)
        a.update(change)
        with pytest.raises(RuntimeError, match=message):
            call(a["x"], a["residual"], a["weight"], a["out"], a["q"], a["scales"], a["group"])
