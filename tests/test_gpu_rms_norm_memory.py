"""GPU: torch.ops._C.b200_add_rms_norm on tensors that are columns of one buffer, and on ones that share memory."""
import pytest
import torch

from test_gpu_rms_norm import DEV, call, check, make

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def columns(rows, *widths):
    """Slices of a buffer of bytes, one behind the other in each row."""
    buf = torch.zeros(rows, sum(widths), dtype=torch.uint8, device=DEV)
    return buf, torch.split(buf, widths, dim=1)


@pytest.mark.parametrize("hidden", [256, 248])
def test_all_of_a_call_in_the_rows_of_one_buffer(native, hidden):
    """Input, residual, output, 8-bit rows and scales side by side; the weight behind one of the rows."""
    rows, group = 9, hidden // 8
    x0, r0, w0 = make(rows, hidden, BF16, True, BF16)
    buf, parts = columns(rows, 2 * hidden, 2 * hidden, 2 * hidden, hidden, 4 * 8, 2 * hidden, 64)
    x, residual, out = (p.view(BF16) for p in parts[:3])
    q, scales, weight = parts[3].view(E4M3), parts[4].view(torch.float32), parts[5].view(BF16)[3]
    x.copy_(x0)
    residual.copy_(r0)
    weight.copy_(w0)
    parts[6].fill_(77)
    call(x, residual, weight, out, q, scales, group)
    assert torch.equal(x, x0) and torch.equal(weight, w0) and (parts[6] == 77).all()
    check(x0, r0, residual.contiguous(), w0, out.contiguous(), q.contiguous(), scales.contiguous(), group, False)


@pytest.mark.parametrize("first,second", [(0, 1), (1, 0)])
def test_input_and_residual_as_halves_of_a_buffer(native, first, second):
    x0, r0, w = make(300, 512, BF16, True, torch.float32)
    buf = torch.empty(300, 2, 512, dtype=BF16, device=DEV)
    buf[:, first], buf[:, second] = x0, r0
    x, residual = buf[:, first], buf[:, second]
    call(x, residual, w, x, None, None)
    check(x0, r0, residual.contiguous(), w, x.contiguous(), None, None, 0, False)


def test_rows_that_take_turns(native):
    """Every other row of a buffer each."""
    x0, r0, w = make(20, 512, BF16, True, BF16)
    buf = torch.empty(40, 512, dtype=BF16, device=DEV)
    buf[0::2], buf[1::2] = x0, r0
    out = torch.empty_like(x0)
    call(buf[0::2], buf[1::2], w, out, None, None)
    check(x0, r0, buf[1::2].contiguous(), w, out, None, None, 0, False)


def test_refusals(native):
    H, rows = 64, 6
    x, residual, weight = make(rows, H, BF16, True, BF16)
    buf = torch.zeros(rows, 4 * H, dtype=BF16, device=DEV)
    raw = torch.zeros(rows, 256, dtype=torch.uint8, device=DEV)
    out, q, scales = torch.empty_like(x), torch.empty(rows, H, dtype=E4M3, device=DEV), torch.empty(rows, 2, device=DEV)
    flat = torch.zeros(64, device=DEV)
    bad = [
        # a column shared, at either end
        (dict(x=buf[:, :H], residual=buf[:, H - 1:2 * H - 1]), "residual must not overlap the input"),
        (dict(x=buf[:, 8:8 + H], residual=buf[:, :H]), "residual must not overlap the input"),
        # a piece that goes over the end of a row into the next one's
        (dict(x=buf.view(-1)[:rows * 4 * H].view(rows, 4 * H)[:, :H], residual=buf.view(-1)[3 * H + 1:].as_strided((rows - 1, H), (4 * H, 1), 3 * H + 1),
              rows=rows - 1), "residual must not overlap the input"),
        (dict(out=buf[:, :H], residual=buf[:, H - 8:2 * H - 8]), "tensors that are written must not overlap"),
        (dict(q=raw[:, :H].view(E4M3), scales=raw[:, H - 4:H + 4].view(torch.float32)), "tensors that are written must not overlap"),
        (dict(x=buf[:, :H], out=buf[:, 1:H + 1]), "out must be the input or not overlap it"),
        (dict(x=buf[:, :H], q=buf[:, H // 2:H].view(E4M3)), "only out may be the input"),
        (dict(weight=buf[2, :H], residual=buf[:, H // 2:H // 2 + H]), "weight must not be written"),
        # other strides: whatever spans the same memory
        (dict(x=buf[:, :H], residual=buf.view(-1).as_strided((rows, H), (2 * H, 1), 2 * H)), "residual must not overlap the input"),
        (dict(scales=flat.as_strided((rows, 2), (1, 1))), "scales must not overlap themselves"),
        (dict(scales=flat.as_strided((rows, 2), (2, 3))), "scales must not overlap themselves"),
    ]
    for change, message in bad:
        n = change.pop("rows", rows)
        a = dict(x=x, residual=residual, weight=weight, out=out, q=q, scales=scales)
        a.update(change)
        a = {k: v if k == "weight" else v[:n] for k, v in a.items()}
        with pytest.raises(RuntimeError, match=message):
            call(a["x"], a["residual"], a["weight"], a["out"], a["q"], a["scales"], 32)
    # (the same with room between them)
    for change in (dict(scales=flat.as_strided((rows, 2), (1, 6))), dict(scales=flat.as_strided((rows, 2), (3, 2))),
                   dict(x=buf[:, :H], out=buf[:, H:2 * H], residual=buf[:, 2 * H:3 * H], weight=buf[4, 3 * H:])):
        a = dict(x=x, residual=residual, weight=weight, out=out, q=q, scales=scales)
        a.update(change)
        call(a["x"], a["residual"], a["weight"], a["out"], a["q"], a["scales"], 32)
