"""CPU: the checks that the dense products and the int8 quantiser make before any launch, struct layouts, op schemas."""
import ctypes as ct
import shutil
import subprocess

import pytest
import torch

from conftest import PKG_DIR, ROOT
from gemm_args import GemmArgs

P, I, L, Z = ct.c_void_p, ct.c_int, ct.c_int64, ct.c_size_t


class Int8LinearArgs(ct.Structure):
    """b200moe_int8_linear_args of include/b200moe.h."""
    _fields_ = [("x", P), ("x_scale", P), ("w", P), ("w_scale", P), ("bias", P), ("d", P), ("rows", L), ("x_stride", L), ("d_stride", L),
                ("n", I), ("k", I), ("x_dtype", I), ("d_dtype", I), ("bias_dtype", I), ("workspace", P), ("workspace_bytes", Z), ("status", P)]


class GatedLinearArgs(ct.Structure):
    """b200moe_gated_linear_args."""
    _fields_ = [("x", P), ("w", P), ("out", P), ("pre", P), ("grad", P), ("grad_x", P), ("grad_w", P), ("workspace", P),
                ("workspace_bytes", Z), ("rows", L), ("x_stride", L), ("out_stride", L), ("grad_stride", L), ("grad_x_stride", L),
                ("inter", I), ("hidden", I), ("dtype", I), ("status", P)]


@pytest.fixture(scope="module")
def lib():
    lib = ct.CDLL(str(PKG_DIR / "vllm_xpu_kernels" / "libb200moe.so"))
    lib.b200moe_last_error.restype = ct.c_char_p
    lib.b200moe_gated_linear_backward_workspace_bytes.restype = Z
    return lib


def _filled(cls, **values):
    a = cls()
    for k, v in values.items():
        setattr(a, k, v)
    return a


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
@pytest.mark.parametrize("cls,name", [(Int8LinearArgs, "b200moe_int8_linear_args"), (GatedLinearArgs, "b200moe_gated_linear_args")])
def test_struct_layout(tmp_path, cls, name):
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "b200moe.h"\nint main(void) {\n' +
                   "".join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_) +
                   f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(cls, f).offset for f, _ in cls._fields_] + [ct.sizeof(cls)]


LINEAR = dict(x=256, x_scale=256, w=256, w_scale=256, d=256, rows=4, x_stride=64, d_stride=8, n=8, k=64, x_dtype=10, d_dtype=2)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), b"negative or too large"), (dict(rows=1 << 31), b"negative or too large"), (dict(n=-1), b"negative or too large"),
    (dict(k=-16), b"negative or too large"), (dict(k=131072), b"at most 131071"), (dict(k=0), b"multiples of 16"), (dict(x_dtype=3), b"input must be"),
    (dict(k=24), b"multiples of 16"), (dict(x_stride=72), b"multiples of 16"), (dict(d_dtype=3), b"out must be"),
    (dict(bias=256, bias_dtype=0), b"bias must be"), (dict(x=None), b"null pointer"), (dict(w_scale=None), b"null pointer"),
    (dict(x=264), b"16-byte aligned"), (dict(w=264), b"16-byte aligned"),
])
def test_int8_linear_refused_before_any_launch(lib, change, message):
    assert lib.b200moe_int8_linear(ct.byref(_filled(Int8LinearArgs, **{**LINEAR, **change})), None) == -1
    assert message in lib.b200moe_last_error()


def test_int8_linear_workspace(lib):
    lib.b200moe_int8_linear_workspace_bytes.restype = Z
    assert lib.b200moe_int8_linear_workspace_bytes(L(300), 64) == 300 * 68
    assert lib.b200moe_int8_linear_workspace_bytes(L(0), 64) == 0
    for more in (dict(), dict(workspace=256, workspace_bytes=300 * 68 - 1), dict(workspace=264, workspace_bytes=300 * 68)):
        assert lib.b200moe_int8_linear(ct.byref(_filled(Int8LinearArgs, **{**LINEAR, "x_dtype": 2, "rows": 300, **more})), None) == -4
        assert b"workspace" in lib.b200moe_last_error()


def test_nothing_to_do_is_no_launch(lib):
    assert lib.b200moe_int8_linear(ct.byref(_filled(Int8LinearArgs, **{**LINEAR, "rows": 0})), None) == 0
    assert lib.b200moe_int8_linear(ct.byref(_filled(Int8LinearArgs, **{**LINEAR, "n": 0})), None) == 0
    assert lib.b200moe_int8_linear(None, None) == -1
    assert lib.b200moe_gated_linear(None, None) == -1
    assert lib.b200moe_gated_linear_backward(None, None) == -1
    assert lib.b200moe_gated_linear(ct.byref(_filled(GatedLinearArgs, **{**GATED, "rows": 0})), None) == 0
    assert lib.b200moe_gated_linear_backward(ct.byref(_filled(GatedLinearArgs, **GATED)), None) == 0      # (no gradient asked for)
    assert lib.b200moe_quant_int8_rows(None, 2, L(0), None, L(0), None, L(0), 16, 0, None, 0, None) == 0


GATED = dict(x=256, w=256, out=256, rows=4, x_stride=64, out_stride=8, inter=8, hidden=64, dtype=2)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), b"negative or too large"), (dict(rows=1 << 31), b"negative or too large"), (dict(inter=-1), b"negative or too large"),
    (dict(hidden=-8), b"negative or too large"), (dict(dtype=0), b"only float16 and bfloat16"), (dict(hidden=60), b"multiples of 16 bytes"),
    (dict(x_stride=68), b"multiples of 16 bytes"), (dict(x=264), b"16-byte aligned"), (dict(w=264), b"16-byte aligned"),
    (dict(out=None), b"null pointer"), (dict(hidden=0), b"null pointer or rows without values"),
])
def test_gated_linear_refused_before_any_launch(lib, change, message):
    assert lib.b200moe_gated_linear(ct.byref(_filled(GatedLinearArgs, **{**GATED, **change})), None) == -1
    assert message in lib.b200moe_last_error()


def test_gated_backward_refused_before_any_launch(lib):
    call = lambda **kw: lib.b200moe_gated_linear_backward(ct.byref(_filled(GatedLinearArgs, **{**GATED, **kw})), None)  # noqa: E731
    assert call(grad_x=256) == -1 and b"null pointer" in lib.b200moe_last_error()
    need = lib.b200moe_gated_linear_backward_workspace_bytes(L(4), 8)
    assert need == 4 * 16 * 2
    more = dict(grad=256, pre=256, grad_x=256, grad_stride=8, grad_x_stride=64)
    assert call(**more) == -4 and b"workspace" in lib.b200moe_last_error()
    assert call(**more, workspace=256, workspace_bytes=need - 1) == -4
    assert call(**more, workspace=264, workspace_bytes=need) == -4
    assert lib.b200moe_gated_linear_backward_workspace_bytes(L(3), 3) == 3 * 8 * 2      # rows of whole 16 bytes
    assert lib.b200moe_gated_linear_backward_workspace_bytes(L(0), 3) == 0


@pytest.mark.parametrize("change,message", [
    (dict(a_dtype=2), b"int8 weights need int8 rows"), (dict(a_scale=None), b"int8 weights need int8 rows"),
    (dict(w_scale=None), b"int8 weights need int8 rows"), (dict(k=24), b"divisible by 16"), (dict(k=131072), b"divisible by 16"),
    (dict(epilogue=2), b"SiLU epilogue or none"), (dict(d_dtype=3), b"float32, float16 or bfloat16"), (dict(d_dtype=0, bias=256), b"mid_dtype"),
    (dict(w_experts=2), b"share weight sets"), (dict(num_experts=1025), b"more than 1024"), (dict(n=12), b"divisible by 8"),
    (dict(rows_per_expert=None), b"null pointer"), (dict(a=264), b"aligned"),
])
def test_grouped_int8_refused_before_any_launch(lib, change, message):
    a = dict(a=256, a_dtype=10, a_scale=256, w=256, w_format=9, w_scale=256, d=256, d_dtype=2, rows_per_expert=256, m=4, n=16, k=64, num_experts=4)
    assert lib.b200moe_grouped_gemm(ct.byref(_filled(GemmArgs, **{**a, **change})), None) == -1
    assert message in lib.b200moe_last_error()


def test_grouped_int8_without_rows_is_no_launch(lib):
    a = dict(a_dtype=10, w=256, w_format=9, w_scale=256, d_dtype=2, rows_per_expert=256, m=0, n=16, k=64, num_experts=4)
    assert lib.b200moe_grouped_gemm(ct.byref(_filled(GemmArgs, **a)), None) == 0


def test_quantiser_refused_before_any_launch(lib):
    call = lambda rows=4, hidden=64, dtype=2, x=256, q=256, s=256, segments=None, n=0: lib.b200moe_quant_int8_rows(  # noqa: E731
        P(x), dtype, L(hidden), P(q), L(hidden), P(s), L(rows), hidden, 0, P(segments), n, None)
    for kw, message in ((dict(rows=-1), b"negative or too large"), (dict(rows=1 << 31), b"negative or too large"),
                        (dict(hidden=-1), b"negative or too large"), (dict(dtype=3), b"only float32, float16 and bfloat16"),
                        (dict(x=None), b"null pointer"), (dict(q=None), b"null pointer"), (dict(s=None), b"null pointer"),
                        (dict(segments=256, n=-1), b"negative number of segments")):
        assert call(**kw) == -1
        assert message in lib.b200moe_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(dtype=0), b"bfloat16 or float16"), (dict(hidden=44), b"multiple of 8"), (dict(hidden=0), b"multiple of 8"), (dict(x=264), b"16-byte aligned"),
    (dict(q=260), b"16-byte aligned"),
])
def test_permuting_quantiser_refused_before_any_launch(lib, change, message):
    v = {**dict(x=256, dtype=2, q=256, hidden=64), **change}
    assert lib.b200moe_remap_quant_int8(P(v["x"]), v["dtype"], P(v["q"]), P(256), None, P(256), P(256), P(256), 5, L(4), v["hidden"], 2, 8, 8,
                                        None, Z(0), None) == -1
    assert message in lib.b200moe_last_error()


def test_schemas_and_no_cpu_path(native):
    def schema(op):
        args = op.default._schema.arguments
        return [a.name for a in args], [a.name for a in args if a.is_write]
    C, X = torch.ops._C, torch.ops._xpu_C
    assert schema(C.b200_quant_int8_rows) == (["input", "out", "scales"], ["out", "scales"])
    assert schema(C.b200_silu_and_mul_quant_int8_rows) == (["out", "input", "scales"], ["out", "scales"])
    assert schema(X.b200_int8_linear) == (["out", "input", "input_scales", "weight", "weight_scales", "bias"], ["out"])
    assert schema(X.b200_gated_linear) == (["out", "input", "weight", "pre"], ["out", "pre"])
    assert schema(X.b200_gated_linear_backward) == (["grad_out", "pre", "input", "weight", "grad_input", "grad_weight"],
                                                    ["grad_input", "grad_weight"])
    assert schema(X.b200_gated_product) == (["input", "weight"], [])
    x, w = torch.ones(2, 16, dtype=torch.bfloat16), torch.ones(8, 16, dtype=torch.bfloat16)
    from vllm_xpu_kernels.gated_linear import gated_linear
    with pytest.raises(NotImplementedError):
        gated_linear(x, w)
    with pytest.raises(NotImplementedError):
        X.b200_int8_linear(torch.ones(2, 8, dtype=torch.bfloat16), x, None, w.to(torch.int8), torch.ones(8))
    with pytest.raises(NotImplementedError):
        C.b200_quant_int8_rows(x, x.to(torch.int8), torch.ones(2))


def test_int8_layers_are_told_apart(native):
    E, H, I = 2, 32, 16
    w13, w2 = torch.zeros(E, 2 * I, H, dtype=torch.int8), torch.zeros(E, H, I, dtype=torch.int8)
    s13, s2 = torch.ones(E, 2 * I), torch.ones(E, H)
    layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, 1, "silu", E)
    assert layer.recipe == "int8" and layer.inter_size == I and layer.fuses_activation(4) == "epilogue"
    assert native.XpuFusedMoe(w13, s13, None, w2, s2, None, 1, "silu", E, fuse_activation=False).fuses_activation(4) is None
    assert native.XpuFusedMoe(w13, s13, None, w2, s2, None, 1, "gelu", E).fuses_activation(4) is None
    for bad in (dict(few_tokens=True), dict(fuse_activation=True, activation="swigluoai")):
        with pytest.raises((NotImplementedError, ValueError)):
            native.XpuFusedMoe(w13, s13, None, w2, s2, None, 1, bad.pop("activation", "silu"), E, **bad)
    with pytest.raises(ValueError, match="both"):
        native.XpuFusedMoe(w13, s13, None, w2, None, None, 1, "silu", E)


@pytest.mark.parametrize("hidden", [(1 << 29) + 8, 1 << 30, (1 << 31) - 8])
def test_gated_rows_whose_bytes_32_bits_do_not_hold_are_refused(lib, hidden):
    """Rows are counted in bytes: of 2^30 values and more nothing was multiplied, and zeros came out."""
    a = {**GATED, "hidden": hidden, "x_stride": hidden, "grad_x_stride": hidden}
    assert lib.b200moe_gated_linear(ct.byref(_filled(GatedLinearArgs, **a)), None) == -1
    assert b"too large" in lib.b200moe_last_error()
    assert lib.b200moe_gated_linear_backward(ct.byref(_filled(GatedLinearArgs, **a, grad=256, pre=256, grad_x=256)), None) == -1
    assert b"too large" in lib.b200moe_last_error()


def test_weight_rows_that_32_bits_do_not_hold_with_a_tile_more_are_refused(lib):
    n = (1 << 31) - 8
    assert lib.b200moe_int8_linear(ct.byref(_filled(Int8LinearArgs, **{**LINEAR, "n": n, "d_stride": n})), None) == -1
    assert b"too large" in lib.b200moe_last_error()
    a = dict(a=256, a_dtype=10, a_scale=256, w=256, w_format=9, w_scale=256, d=256, d_dtype=2, rows_per_expert=256, m=4, n=n, k=64, num_experts=1)
    assert lib.b200moe_grouped_gemm(ct.byref(_filled(GemmArgs, **a)), None) == -1
    assert b"too many rows or features" in lib.b200moe_last_error()


@pytest.mark.parametrize("operand", [0, 1])
def test_forward_mode_derivatives_of_the_gated_product_are_refused(native, operand):
    """(On any device: below autograd the tangent would be lost, and the derivative come out as zero.)"""
    from vllm_xpu_kernels.gated_linear import gated_linear
    operands = [torch.ones(2, 16, dtype=torch.bfloat16), torch.ones(8, 16, dtype=torch.bfloat16)]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: gated_linear(*operands[:operand], t, *operands[operand + 1:]), (operands[operand],), (operands[operand],))
    with torch.autograd.forward_ad.dual_level():
        operands[operand] = torch.autograd.forward_ad.make_dual(operands[operand], torch.ones_like(operands[operand]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_linear(*operands)
