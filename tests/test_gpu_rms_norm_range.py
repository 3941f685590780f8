"""GPU: torch.ops._C.b200_add_rms_norm on rows whose squares fp32 does not hold: finite rows have finite results, within the bounds of
test_gpu_rms_norm (which leave the order of the sums open; what a power of two takes away before they are made is exact).
"""
import pytest
import torch

from test_gpu_rms_norm import call, check, fp32_bound, make, outputs, reference

pytestmark = pytest.mark.gpu
SIZES = [(3, 17, 0), (2, 32, 32), (4, 512, 128), (1, 7168, 128), (3, 1411, 0), (3, 1411, 83), (7, 2880, 0), (33, 2048, 32), (400, 1024, 0),
         (700, 1024, 64), (2, 5001, 0), (2, 9000, 0), (2, 65536, 128), (300, 264, 0), (3000, 99, 0)]
WIDE = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", WIDE, ids=str)
@pytest.mark.parametrize("rows,hidden,group", SIZES)
@pytest.mark.parametrize("power", [70, 120])
def test_large_rows_next_to_ordinary_ones(native, rows, hidden, group, dtype, power):
    for with_residual, weight_dtype in ((True, dtype), (False, None)):
        x, residual, weight = make(rows, hidden, dtype, with_residual, weight_dtype, power)
        for t in (x, residual):
            if t is not None:
                t[::2] = (t[::2].float() * 2.0 ** power).to(dtype)
        before = None if residual is None else residual.clone()
        out, q, scales = outputs(rows, hidden, dtype, group)
        call(x, residual, weight, out, q, scales, group)
        assert out.isfinite().all() and scales.isfinite().all()
        check(x, before, residual, weight, out, q, scales, group, False)


@pytest.mark.parametrize("dtype", WIDE, ids=str)
@pytest.mark.parametrize("rows,hidden,group", SIZES)
@pytest.mark.parametrize("power", [-110, -80, -45, 62, 64, 66, 110, 122])
def test_the_norm_does_not_change_with_a_power_of_two(native, rows, hidden, group, dtype, power):
    """Without an eps: the formula's results of the scaled rows are those of the rows as they were."""
    x, _, weight = make(rows, hidden, dtype, False, dtype)
    x = torch.where(x.abs() < 2.0 ** -12, torch.full_like(x, 2.0 ** -12), x)       # (no subnormals in what follows)
    scaled = (x.double() * 2.0 ** power).to(dtype)
    assert scaled.isfinite().all()
    fp, half, g = fp32_bound(hidden), torch.finfo(dtype).eps / 2, group or hidden
    for weights in (weight, None):
        out, q, scales = outputs(rows, hidden, dtype, group)
        call(scaled, None, weights, out, q, scales, group, eps=0.0)
        _, y = reference(x, None, weights, eps=0.0)
        assert ((out.double() - y).abs() <= y.abs() * (half + fp * (1 + half))).all()
        parts = y.view(-1, hidden // g, g)
        want, got = (parts.abs().amax(-1) / 448).clamp(min=1 / (448 * 512)), scales.double()
        assert ((got - want).abs() <= want * (fp + 3 * 2.0 ** -24)).all()
        real, slack = parts / got[..., None], 2.0 ** -4 + 2 * fp
        assert ((q.double().view_as(parts) - real).abs() <= real.abs() * slack + 2.0 ** -10 * (1 + slack)).all()


@pytest.mark.parametrize("dtype", WIDE, ids=str)
def test_a_single_large_value(native, dtype):
    """The largest finite value among ordinary ones: it gets sqrt(hidden), the others what is left of them."""
    hidden = 1024
    x, _, _ = make(2, hidden, dtype, False, None)
    x[0, 3] = -torch.finfo(dtype).max
    out, q, scales = outputs(2, hidden, dtype, 0)
    call(x, None, None, out, q, scales)
    _, y = reference(x, None, None)
    # (the mean square of row 0 is 2^246, its values of 1 come to 2^-123 and smaller ones into the subnormals, whose rounding is half of the
    # smallest one, 2^-133 or 2^-149, instead of half a step of the value)
    f = torch.finfo(dtype)
    half, smallest, fp = f.eps / 2, f.smallest_normal * f.eps, fp32_bound(hidden)
    assert ((out.double() - y).abs() <= y.abs() * (half + fp * (1 + half)) + smallest / 2 * (1 + fp)).all()
    check(x, None, None, None, None, q, scales, 0, False)
    assert abs(out[0, 3].item() + 32) <= 32 * torch.finfo(dtype).eps and q[0, 3].item() == -448


@pytest.mark.parametrize("dtype", WIDE, ids=str)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_that_are_not_finite_among_large_ones(native, dtype, value):
    x, _, weight = make(3, 512, dtype, False, dtype)
    x *= 2.0 ** 80
    x[1, 5] = value
    out, q, scales = outputs(3, 512, dtype, 128)
    call(x, None, weight, out, q, scales, 128)
    assert out[1, 5].isnan() and scales[1, 0].isnan() and q[1, 5].float().isnan()
    assert out[[0, 2]].isfinite().all() and scales[[0, 2]].isfinite().all()


@pytest.mark.parametrize("group", [0, 32])
def test_more_rows_than_a_block_has_turns_for(native, group):
    """Large rows among many short ones, the last ones too; in place."""
    rows, hidden = 200_003, 64
    x, _, weight = make(rows, hidden, torch.bfloat16, False, torch.bfloat16)
    large = torch.rand(rows, device=x.device) < 0.3
    large[-5:] = True
    x[large] = (x[large].float() * 2.0 ** 90).to(x.dtype)
    before = x.clone()
    _, q, scales = outputs(rows, hidden, x.dtype, group)
    call(x, None, weight, x, q, scales, group)
    check(before, None, None, weight, x, q, scales, group, False)
