"""The int8 row quantisers and the int8 product, dense and by expert, against 64 bits."""
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rows(shape, dtype, gen, spread=1.0):
    return (torch.randn(shape, generator=gen) * spread).to(dtype)


# ---- rows ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [B16, F16, F32])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 16), (3, 31), (2, 100), (5, 128), (7, 1000), (4, 2048), (300, 768), (2, 14336),
                                         (1, 32768), (2, 40000), (1, 65537)])
def test_codes_and_scales_are_the_formulas(native, dtype, rows, hidden):
    x = _rows((rows, hidden), dtype, torch.Generator().manual_seed(rows * 7 + hidden))
    x[0, hidden // 2] = 0
    if rows > 2:
        x[1] = 0                                  # scale of the least maximum
        x[2] = torch.finfo(dtype).smallest_normal
    q = torch.full((rows, hidden), 99, dtype=torch.int8, device=DEV)
    s = torch.full((rows,), float("nan"), device=DEV)
    torch.ops._C.b200_quant_int8_rows(x.to(DEV), q, s)
    want_q, want_s = ref.quant_rows(x)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("dtype,bits", [(B16, 8), (F16, 11)])
def test_every_mantissa_and_tie_of_16_bits(native, dtype, bits):
    """Rows whose largest value has each mantissa, with every value that the type has in the three powers of two below it: ties among them."""
    m = torch.arange(2 ** (bits - 1), 2 ** bits, dtype=torch.float64)
    below = torch.cat([m * 2.0 ** -s for s in range(4)])
    rows = torch.where(below[None] <= m[:, None], below[None], 0.0 * below[None])
    x = torch.cat((m[:, None], rows, -rows, torch.zeros(len(m), 7, dtype=torch.float64)), dim=1) / 2 ** bits
    x = x.to(dtype)
    want_q, want_s = ref.quant_rows(x)
    tie = 254 * x.double().abs() / x[:, :1].double()
    assert int(((tie == torch.floor(tie)) & (tie % 2 == 1)).sum()) > len(m)            # (there are ties)
    for part in (x[:, :-7].contiguous(), x[:, :-6].contiguous()):                      # (an odd length too)
        q, s = torch.empty(part.shape, dtype=torch.int8, device=DEV), torch.empty(len(m), device=DEV)
        torch.ops._C.b200_quant_int8_rows(part.to(DEV), q, s)
        assert torch.equal(q.cpu(), want_q[:, :part.shape[1]]) and torch.equal(s.cpu(), want_s)


@pytest.mark.parametrize("dtype", [B16, F16, F32])
@pytest.mark.parametrize("rows,hidden", [(1, 8), (2, 33), (5, 768), (300, 1408), (2, 14336), (1, 33000)])
def test_gated_codes(native, dtype, rows, hidden):
    x = _rows((rows, 2 * hidden), dtype, torch.Generator().manual_seed(hidden), 3.0)
    q = torch.empty(rows, hidden, dtype=torch.int8, device=DEV)
    s = torch.empty(rows, device=DEV)
    torch.ops._C.b200_silu_and_mul_quant_int8_rows(q, x.to(DEV), s)
    g, u = x.double().chunk(2, dim=-1)
    v = ref.silu(g) * u
    scale = v.abs().amax(dim=-1).clamp(min=ref.LEAST) / 127
    # v: exponential, quotient and products 2^-20, the exponential's argument rounded twice: 2^-23 |gate|; the scale, and its reciprocal,
    # that of the row's largest and a division; the code those of both, of at most 127
    off = 2.0 ** -20 + g.abs().amax(dim=-1) * 2.0 ** -23
    assert torch.all((s.cpu().double() / scale - 1).abs() <= off + 2.0 ** -24)
    assert torch.all((q.cpu().double() - v / scale[:, None]).abs() <= 0.5 + 127 * (2 * off[:, None] + 2.0 ** -23))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hidden", [32, 33])
def test_rows_that_are_not_finite_stay_visible(native, bad, hidden):
    x = torch.ones(3, hidden, dtype=B16, device=DEV)
    x[1, hidden - 1] = bad
    q, s = torch.empty(3, hidden, dtype=torch.int8, device=DEV), torch.empty(3, device=DEV)
    torch.ops._C.b200_quant_int8_rows(x, q, s)
    assert not torch.isfinite(s[1]) and torch.isfinite(s[0]) and torch.isfinite(s[2])
    assert torch.all(q[0] == 127) and torch.isnan(s[1])
    if hidden % 16 == 0:
        out = torch.empty(3, 5, dtype=B16, device=DEV)
        torch.ops._xpu_C.b200_int8_linear(out, x, None, torch.ones(5, hidden, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))
        assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()


def test_quantised_rows_of_strided_tensors(native):
    gen = torch.Generator().manual_seed(5)
    wide = _rows((4, 3, 200), B16, gen).to(DEV)
    for x in (wide[:, :, 8:104], wide[:, :, 3:67], wide[:, 1:2, :96], wide[1, 2, 16:80]):
        room = torch.full((*x.shape[:-1], x.shape[-1] + 5), 77, dtype=torch.int8, device=DEV)
        q, s = room[..., 2:-3], torch.empty(x.shape[:-1], device=DEV)
        torch.ops._C.b200_quant_int8_rows(x, q, s)
        want_q, want_s = ref.quant_rows(x)
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
        assert torch.all(room[..., :2] == 77) and torch.all(room[..., -3:] == 77)


# ---- the dense product ---------------------------------------------------------------

def _check(out, q, qs, w, ws, bias):
    y, p = ref.linear(q, qs, w, ws, bias)
    err = (out.double() - y).abs()
    assert torch.all(err <= ref.linear_tolerance(y, p, out.dtype)), float((err - ref.linear_tolerance(y, p, out.dtype)).max())


@pytest.mark.parametrize("out_dtype,bias", [(B16, False), (F16, True), (F32, True)])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 16), (1, 33, 48), (2, 31, 1040), (8, 100, 128), (9, 64, 2048), (16, 130, 4096),
                                      (17, 1, 16), (17, 255, 144), (40, 257, 128), (129, 300, 272), (256, 256, 512), (257, 513, 1040),
                                      (700, 1000, 2048), (40, 256, 4096), (130, 40, 6160), (300, 521, 7168), (64, 300, 2064),
                                      (513, 250, 16384), (20, 2000, 4096)])
def test_product_of_codes(native, rows, n, k, out_dtype, bias):
    gen = torch.Generator().manual_seed(rows + n + k)
    q, qs = ref.weights(rows, k, gen)
    w, ws = ref.weights(n, k, gen)
    b = _rows((n,), F16 if out_dtype == F32 else out_dtype, gen).to(DEV) if bias else None
    out = torch.full((rows, n), float("nan"), dtype=out_dtype, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(out, q, qs, w, ws, b)
    _check(out, q, qs, w, ws, b)


def test_sums_beyond_24_bits_are_exact(native):
    """All products 128 * 128: a sum of 2^31 - 2^14 - ... that fp32 sums would round."""
    k = 131056
    for rows in (1, 40):
        q = torch.full((rows, k), -128, dtype=torch.int8, device=DEV)
        w = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
        q[:, 0] = 1                                # 128 * 128 * (k - 1) - 128
        out = torch.empty(rows, 3, device=DEV)
        one = torch.ones(max(rows, 3), device=DEV)
        torch.ops._xpu_C.b200_int8_linear(out, q, one[:rows], w, one[:3])
        assert torch.all(out == float(torch.tensor(16384 * (k - 1) - 128, dtype=torch.int64).float()))


@pytest.mark.parametrize("rows", [1, 5, 33, 300])
@pytest.mark.parametrize("dtype", [B16, F16, F32])
def test_linear_quantises_its_rows(native, rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    n, k = 200, 1056
    x = _rows((rows, k), dtype, gen)
    w, ws = ref.weights(n, k, gen)
    out_dtype = B16 if dtype == F32 else dtype
    out = torch.empty(rows, n, dtype=out_dtype, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(out, x.to(DEV), None, w, ws)
    q, qs = ref.quant_rows(x)
    _check(out, q.to(DEV), qs.to(DEV), w, ws, None)


@pytest.mark.parametrize("rows", [3, 70])
def test_linear_of_strided_rows_leaves_the_rest_alone(native, rows):
    gen = torch.Generator().manual_seed(rows)
    n, k = 72, 96
    q, qs = ref.weights(rows, 160, gen)
    q = q[:, 32:32 + k]
    w, ws = ref.weights(n, k, gen)
    for left, right in ((0, 8), (8, 8), (3, 2), (16, 16)):
        room = torch.full((rows + 1, left + n + right), 7.0, dtype=B16, device=DEV)
        torch.ops._xpu_C.b200_int8_linear(room[:rows, left:left + n], q, qs, w, ws)
        _check(room[:rows, left:left + n], q, qs, w, ws, None)
        assert torch.all(room[:, :left] == 7) and torch.all(room[:, left + n:] == 7) and torch.all(room[rows] == 7)


@pytest.mark.parametrize("rows", [3, 70])
def test_columns_of_one_buffer(native, rows):
    """Input and output as columns of the same rows; those that share a byte are refused."""
    gen = torch.Generator().manual_seed(rows)
    n, k = 40, 64
    w, ws = ref.weights(n, k, gen)
    room = torch.zeros(rows, k + n + 8, dtype=B16, device=DEV)
    room[:, :k] = _rows((rows, k), B16, gen).to(DEV)
    x = room[:, :k].clone()
    torch.ops._xpu_C.b200_int8_linear(room[:, k:k + n], room[:, :k], None, w, ws)
    want = torch.empty(rows, n, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(want, x, None, w, ws)
    assert torch.equal(room[:, k:k + n], want) and torch.equal(room[:, :k], x)
    for bad in (room[:, k - 1:k - 1 + n], room[:, 8:8 + n]):
        with pytest.raises(RuntimeError, match="share memory"):
            torch.ops._xpu_C.b200_int8_linear(bad, room[:, :k], None, w, ws)


def test_linear_of_more_dimensions_and_of_none(native):
    gen = torch.Generator().manual_seed(2)
    w, ws = ref.weights(40, 64, gen)
    x = _rows((2, 3, 64), B16, gen).to(DEV)
    out = torch.empty(2, 3, 40, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(out, x, None, w, ws)
    flat = torch.empty(6, 40, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(flat, x.view(6, 64), None, w, ws)
    assert torch.equal(out.view(6, 40), flat)
    one = torch.empty(40, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(one, x[1, 2], None, w, ws)
    assert torch.equal(one, flat[5])
    torch.ops._xpu_C.b200_int8_linear(torch.empty(0, 40, dtype=B16, device=DEV), x.view(6, 64)[:0], None, w, ws)
    torch.ops._xpu_C.b200_int8_linear(torch.empty(6, 0, dtype=B16, device=DEV), x.view(6, 64), None, w[:0], ws[:0])


# ---- by expert -----------------------------------------------------------------------

def _grouped(q, qs, w, ws, bias, rows, epilogue, dtype, clamp=0.0, f16=False):
    E, n, k = w.shape
    d = torch.full((q.shape[0], n // 2 if epilogue else n), float("nan"), dtype=dtype, device=DEV)
    torch.ops._xpu_C.b200_grouped_gemm(q, qs, w, ws, bias, d, rows, n, k, E, 0, epilogue, 1.702, 7.0, clamp, 0, 0, 0, None, f16)
    return d


@pytest.mark.parametrize("counts", [[1], [0, 3, 0, 1], [5, 0, 16, 2, 9], [33, 0, 17, 64], [300, 0, 1, 255, 257], [0, 0, 0]])
@pytest.mark.parametrize("n,k", [(8, 16), (104, 528), (520, 256)])
def test_grouped_product(native, counts, n, k):
    gen = torch.Generator().manual_seed(sum(counts) + n)
    M, E = sum(counts) + 3, len(counts)              # three rows behind the last segment
    q, qs = ref.weights(M, k, gen)
    w, ws = ref.weights(n, k, gen, E)
    bias = _rows((E, n), B16, gen).to(DEV)
    d = _grouped(q, qs, w, ws, bias, torch.tensor(counts, dtype=torch.int32, device=DEV), 0, B16)
    at = 0
    for e, c in enumerate(counts):
        if c:
            _check(d[at:at + c], q[at:at + c], qs[at:at + c], w[e], ws[e], bias[e])
        at += c
    assert torch.isnan(d[at:]).all()


@pytest.mark.parametrize("counts", [[1], [3, 0, 1, 16], [40, 0, 300]])
@pytest.mark.parametrize("inter,dtype,clamp", [(36, F32, 0.0), (128, B16, 0.0), (260, F32, 1.5)])
def test_grouped_gated_product(native, counts, inter, dtype, clamp):
    k = 272
    gen = torch.Generator().manual_seed(inter)
    M, E = sum(counts), len(counts)
    q, qs = ref.weights(M, k, gen)
    w, ws = ref.weights(2 * inter, k, gen, E)
    bias = _rows((E, 2 * inter), F16 if dtype == F32 else dtype, gen).to(DEV)
    d = _grouped(q, qs, w, ws * 0.2, bias, torch.tensor(counts, dtype=torch.int32, device=DEV), 1, dtype, clamp, dtype == F32)
    at = 0
    for e, c in enumerate(counts):
        if not c:
            continue
        y, p = ref.linear(q[at:at + c], qs[at:at + c], w[e], ws[e] * 0.2, bias[e])
        err = (3.01 * p.abs() + y.abs()) * 2.0 ** -24
        g, u, eg, eu = *y.chunk(2, dim=-1), *err.chunk(2, dim=-1)
        if clamp:
            g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
        s = ref.silu(g)
        # |silu'| < 1.1; the exponential's argument rounded twice (2^-23 |g|), the approximations and products 2^-20
        tol = 1.1 * u.abs() * eg + s.abs() * eu + (s * u).abs() * (2.0 ** -20 + g.abs() * 2.0 ** -23)
        if dtype != F32:
            tol = tol * 1.01 + (s * u).abs() * torch.finfo(dtype).eps / 2 * 1.01
        assert torch.all((d[at:at + c].double() - s * u).abs() <= tol + 1e-30)
        at += c


# ---- calls beside one another -------------------------------------------------------------

@pytest.mark.parametrize("rows", [4, 64])
def test_other_stream_and_graph(native, rows):
    gen = torch.Generator().manual_seed(1)
    n, k = 256, 512
    w, ws = ref.weights(n, k, gen)
    x = _rows((rows, k), B16, gen).to(DEV)
    want = torch.empty(rows, n, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(want, x, None, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.empty_like(want)
        torch.ops._xpu_C.b200_int8_linear(got, x, None, w, ws)
    side.synchronize()
    assert torch.equal(got, want)
    first, second = torch.empty_like(want), torch.empty_like(want)
    graphs = []
    for out in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            torch.ops._xpu_C.b200_int8_linear(out, x, None, w, ws)
        graphs.append(g)
    for _ in range(3):
        x.copy_(_rows((rows, k), B16, gen))
        torch.ops._xpu_C.b200_int8_linear(want, x, None, w, ws)
        for g in graphs:
            g.replay()
        assert torch.equal(first, want) and torch.equal(second, want)


def test_refusals(native):
    gen = torch.Generator().manual_seed(0)
    w, ws = ref.weights(24, 64, gen)
    x, out = torch.zeros(4, 64, dtype=B16, device=DEV), torch.zeros(4, 24, dtype=B16, device=DEV)
    q, qs = torch.zeros(4, 64, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    op = torch.ops._xpu_C.b200_int8_linear
    for args, message in [
        ((out, x, qs, w, ws), "int8 rows come with input_scales"), ((out, q, None, w, ws), "int8 rows come with input_scales"),
        ((out, x[:, :48], None, w, ws), "same K"), ((out[:, :20], x, None, w, ws), r"out must be \[\.\.\., N\]"),
        ((out, x[:, :40], None, w[:, :40].contiguous(), ws), "multiple of 16"), ((out, x, None, w.float(), ws), "int8"),
        ((out, x, None, w[:, ::2], ws), "same K"), ((out, x, None, w, ws[:20]), "weight_scales"), ((out, q, qs[:3], w, ws), "input_scales"),
        ((out, x, None, w, ws, torch.zeros(24, device=DEV)), "bias must be"), ((out, x, None, w, ws, out[0, :20]), "bias must be"),
        ((out.double(), x, None, w, ws), "float32, float16 and bfloat16"), ((out, x.double(), None, w, ws), "float32, float16 and bfloat16"),
        ((out, x, None, w.cpu(), ws), "device"), ((out[:1].expand(4, 24), x, None, w, ws), "overlap|expanded"),
        ((out, torch.zeros(4, 72, dtype=torch.int8, device=DEV)[:, :64], qs, w, ws), "16"),
        ((out, torch.zeros(4 * 80 + 8, dtype=torch.int8, device=DEV)[8:].view(4, 80)[:, :64], qs, w, ws), "aligned"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            op(*args)
    quant = torch.ops._C.b200_quant_int8_rows
    for args in [(x, q[:, :32], qs), (x, q, qs[:3]), (x, q.float(), qs), (x, q, qs.double()), (x, q[:1].expand(4, 64), qs),
                 (x.to(torch.int32), q, qs), (x.t(), q.t(), qs)]:
        with pytest.raises(RuntimeError):
            quant(*args)
    with pytest.raises(RuntimeError, match="int8 ptr_A"):
        _grouped(x, None, w[None], ws[None], None, torch.tensor([4], dtype=torch.int32, device=DEV), 0, B16)
