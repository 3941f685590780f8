"""CPU: the checks that b200moe_add_rms_norm makes before any launch, and the op's schema."""
import ctypes

import pytest
import torch

from conftest import PKG_DIR


class RmsNormArgs(ctypes.Structure):
    """b200moe_rms_norm_args of include/b200moe.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("input", "residual", "weight", "out", "q", "scales")] +
                [(n, ctypes.c_int64) for n in ("rows", "input_stride", "residual_stride", "out_stride", "q_stride",
                                               "s_stride_row", "s_stride_group")] +
                [("hidden", ctypes.c_int), ("group_size", ctypes.c_int), ("eps", ctypes.c_float),
                 ("scale_ue8m0", ctypes.c_int), ("dtype", ctypes.c_int), ("weight_dtype", ctypes.c_int)])


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), b"negative or too large size"),
    (dict(rows=1 << 31), b"negative or too large size"),
    (dict(hidden=-8), b"negative or too large size"),
    (dict(group_size=100), b"multiple of group_size"),
    (dict(group_size=-1), b"multiple of group_size"),
    (dict(q=256), b"go together"),
    (dict(weight=256, weight_dtype=1), b"weight must be float32 or"),
    (dict(input=None), b"null pointer"),
    (dict(out=None), b"nothing to write"),
    (dict(dtype=3, weight_dtype=3), b"only float32, float16 and bfloat16"),
])
def test_refused_before_any_launch(change, message):
    lib = ctypes.CDLL(str(PKG_DIR / "vllm_xpu_kernels" / "libb200moe.so"))
    lib.b200moe_last_error.restype = ctypes.c_char_p
    a = dict(input=256, out=256, rows=4, hidden=256, input_stride=256, out_stride=256, dtype=2, weight_dtype=2)
    a.update(change)
    args = RmsNormArgs()
    for name, value in a.items():
        setattr(args, name, value)
    assert lib.b200moe_add_rms_norm(ctypes.byref(args), None) == -1
    assert message in lib.b200moe_last_error()
    assert lib.b200moe_add_rms_norm(None, None) == -1


def test_schema(native):
    args = torch.ops._C.b200_add_rms_norm.default._schema.arguments
    assert [a.name for a in args] == ["input", "residual", "weight", "epsilon", "out", "out_q", "scales", "group_size",
                                      "scale_ue8m0"]
    assert [a.is_write for a in args] == [False, True, False, False, True, True, True, False, False]
    with pytest.raises(NotImplementedError):
        torch.ops._C.b200_add_rms_norm(torch.ones(2, 8), None, None, 1e-6, torch.empty(2, 8))
