# SPDX-License-Identifier: Apache-2.0
"""Both projections of a gated feed-forward block, its activation and the product, with gradients.

``gated_linear(input, weight)`` is ``silu(input @ weight[:I].T) * (input @ weight[I:].T)`` for ``weight`` ``[2 * I, H]`` (gate
rows first, the order of ``w13`` of a layer): the dense counterpart of what ``XpuFusedMoe`` does for its experts (a shared expert, a dense
layer between Mixture-of-Experts layers).  bfloat16 and float16; one kernel forward
(``torch.ops._xpu_C.b200_gated_linear``), three for the gradients (``b200_gated_linear_backward``).  (Not in the reference.)
"""
import torch

from .fused_moe_interface import _require_native


def _rows(t):
    """`t` as the kernels read it: rows that are dense, evenly spaced and on 16-byte boundaries (a copy where they are not)."""
    if t.numel() == 0:
        return t
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0:
        try:
            rows = t.view(-1, t.shape[-1])
        except RuntimeError:        # not evenly spaced
            return t.contiguous()
        if rows.shape[0] == 1 or rows.stride(0) % 8 == 0:
            return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(input, weight, keep):
    _require_native()
    inter = weight.shape[0] // 2
    out = torch.empty(*input.shape[:-1], inter, dtype=input.dtype, device=input.device)
    pre = torch.empty(*input.shape[:-1], 2 * inter, dtype=torch.float32, device=input.device) if keep else None
    torch.ops._xpu_C.b200_gated_linear(out, input, weight, pre)
    return out, pre


class _GatedLinear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, input, weight):
        out, pre = _forward(input, weight, True)
        ctx.save_for_backward(input, weight, pre)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        input, weight, pre = ctx.saved_tensors
        dx = torch.empty(input.shape, dtype=input.dtype, device=input.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        torch.ops._xpu_C.b200_gated_linear_backward(_rows(grad), pre, input, weight, dx, dw)
        return dx, dw


def gated_linear(input, weight):
    """``silu(input @ weight[:I].T) * (input @ weight[I:].T)``: ``input`` ``[..., H]``, ``weight`` ``[2 * I, H]`` of the same
    type (bfloat16 or float16), H divisible by 8; the result ``[..., I]``.

    With gradients enabled and asked for, the two products are kept in fp32 (8 bytes for each value of the result) and the gradients of
    either operand are computed from them; they are not differentiable again.  Weights that are not contiguous, and
    rows that are not evenly spaced on 16-byte boundaries, are copied first.  Under stream capture, as for any autograd function, the
    leaves must have no live graph from outside the capture."""
    input, weight = _rows(input), weight.contiguous()
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad):
        return _GatedLinear.apply(input, weight)
    return _forward(input, weight, False)[0]
