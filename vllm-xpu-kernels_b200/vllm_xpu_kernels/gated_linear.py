# SPDX-License-Identifier: Apache-2.0
"""Both projections of a gated feed-forward block, its activation and the product, with gradients.

``gated_linear(input, weight)`` is ``silu(input @ weight[:I].T) * (input @ weight[I:].T)`` for ``weight`` ``[2 * I, H]`` (gate
rows first, the order of ``w13`` of a layer): the dense counterpart of what ``XpuFusedMoe`` does for its experts (a shared expert, a dense
layer between Mixture-of-Experts layers).  bfloat16 and float16; one kernel forward
(``torch.ops._xpu_C.b200_gated_linear``), three for the gradients (``b200_gated_linear_backward``).  (Not in the reference.)
"""
import torch

from .fused_moe_interface import _require_native


def gated_linear(input, weight):
    """``silu(input @ weight[:I].T) * (input @ weight[I:].T)``: ``input`` ``[..., H]``, ``weight`` ``[2 * I, H]`` of the same
    type (bfloat16 or float16), H divisible by 8; the result ``[..., I]``.

    With gradients enabled and asked for, the two products are kept in fp32 (8 bytes for each value of the result) and the gradients of
    either operand are computed from them, those that a backward pass wants.  Derivatives of these gradients (``create_graph``) raise when they
    are asked for, forward-mode ones (``make_dual``, ``torch.func.jvp``) at the call.  Between the kernels the gradients of the two products
    are of the operands' type: in float16 what is beyond 65504 becomes an infinity, which the results show, and what is below 2^-25 zero.
    Weights that are not contiguous, and rows that are not evenly spaced on 16-byte boundaries, are copied first.  Under stream
    capture an operand that is, or is made of, a leaf that a live graph from outside the capture uses on the default stream
    is refused: let go of what was computed from it first."""
    _require_native()
    return torch.ops._xpu_C.b200_gated_product(input, weight)
