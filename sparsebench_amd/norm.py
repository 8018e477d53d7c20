"""Root-mean-square norms before and after a block, with the block's gate, its
scale and the residual sum in the same pass, forward and backward.

    norm_in(x, weight)                       the block's input:  weight n(x)
    norm_out(y, x, weight, gate, scale)      the residual stream after it:
                                             out = x + scale gate weight n(y)
    norm_out(..., next_weight=v)             (out, v n(out)): with the next block's input
    norm_in_backward, norm_out_backward      their gradients

n(v) = v / sqrt(mean(v^2) + eps) over each row. moe.moe_block_gated puts them
around the gated layer. No autograd graph is built and nothing syncs: forward
and backward calls can be captured in a graph.
"""

from __future__ import annotations

from typing import NamedTuple

import torch


class NormInGrads(NamedTuple):
    """Gradients of norm_in's operands."""

    x: torch.Tensor
    weight: torch.Tensor | None


class NormOutGrads(NamedTuple):
    """Gradients of norm_out's operands; None for those it was called without."""

    y: torch.Tensor
    x: torch.Tensor
    weight: torch.Tensor | None
    gate: torch.Tensor | None
    next_weight: torch.Tensor | None


def norm_in(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    valid_tokens: torch.Tensor | None = None,
) -> torch.Tensor:
    """weight n(x), of x's type. x [T, D] bf16 / fp16 / fp32 with contiguous rows (they may
    start any stride apart), D up to 32768; weight [D] of any of these types, or None for 1.
    valid_tokens (optional int32 CUDA scalar T'): rows t >= T' are left unwritten."""
    from sparsebench_amd import _C

    return _C.norm_in_cuda(x, weight, eps, valid_tokens)


def norm_in_backward(
    grad: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    grad_x: torch.Tensor | None = None,
    valid_tokens: torch.Tensor | None = None,
) -> NormInGrads:
    """The gradients of norm_in(x, weight), from the gradient of its result. grad_x: x's
    gradient from elsewhere (the residual stream), added to it. Rows t >= valid_tokens of
    x's gradient are left unwritten, and add nothing to the weight's."""
    from sparsebench_amd import _C

    return NormInGrads(*_C.norm_in_backward_cuda(grad, x, weight, eps, grad_x, valid_tokens))


def norm_out(
    y: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scale: float = 1.0,
    eps: float = 1e-6,
    next_weight: torch.Tensor | None = None,
    valid_tokens: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """out = x + scale gate weight n(y); with next_weight, (out, norm_in(out, next_weight)),
    bit for bit.

    y (the block's output) and x (the residual stream) [T, D] of one type, as in norm_in;
    weight, next_weight [D]; gate [D] (a layer's learned scale), [T, 1], [T, D], or None
    for 1. A gate [T, D] with T = 1 is one of rows."""
    from sparsebench_amd import _C

    return _C.norm_out_cuda(y, x, weight, gate, scale, eps, next_weight, valid_tokens)


def norm_out_backward(
    grad_out: torch.Tensor,
    y: torch.Tensor,
    weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scale: float = 1.0,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
    grad_next: torch.Tensor | None = None,
    next_weight: torch.Tensor | None = None,
    valid_tokens: torch.Tensor | None = None,
) -> NormOutGrads:
    """The gradients of a norm_out call with these operands, from the gradient of its out
    and, for a call with next_weight, of the next block's input (grad_next, with `out` as
    that call returned it). Without grad_next x's gradient is grad_out itself, the same
    tensor. Sums over tokens are fp32 and in a fixed order; each gradient has its operand's
    shape and type. Rows t >= valid_tokens are left unwritten, and add nothing to sums."""
    from sparsebench_amd import _C

    return NormOutGrads(*_C.norm_out_backward_cuda(grad_out, y, weight, gate, scale, eps, out, grad_next, next_weight,
                                                   valid_tokens))
