"""Updates: the AdamW step of a list of tensors in one kernel, with fp32 or 8-bit
states, and the orthogonalised step of matrices (Muon).

    adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, ...)   one step, in place
    new_step(device)                    the step counter that it advances
    new_state(param, bits)              (exp_avg, exp_avg_sq) of zeros
    dequantize(states, dtype)           the values that 8-bit states stand for
    AdamW(params, ...)                  states and counter kept together

    muon_step(params, grads, momenta, lr, ...)   one step of stacks of matrices, in place
    orthogonalize(matrices)                      its Newton-Schulz products alone
    Muon(params, ...)                            with its momenta

They update what moe.moe_gated_backward gives gradients of, and any other
tensors beside them. Nothing syncs: the step count lives on the GPU, and
learning rate and gradient scale may too, so that a captured step can be
replayed with other values. Expert weights are stacks of matrices, which Muon
takes as they are; the vectors beside them (norms, gates) and the router are AdamW's.
"""

from __future__ import annotations

from collections.abc import Iterable, Sequence
from typing import NamedTuple

import torch

BLOCK = 256  # values that share a scale


class Quantized(NamedTuple):
    """An 8-bit state: a code per value, a scale per BLOCK of them. int8 codes
    c stand for c |c| scale (the first moment), uint8 codes for c^2 scale (the
    second moment's square root)."""

    codes: torch.Tensor
    scales: torch.Tensor


State = torch.Tensor | Quantized


def new_step(device: torch.device | str = "cuda") -> torch.Tensor:
    """[steps done, scratch], int32. One for each sequence of steps."""
    return torch.zeros(2, dtype=torch.int32, device=device)


def new_state(param: torch.Tensor, bits: int = 32) -> tuple[State, State]:
    """(exp_avg, exp_avg_sq) of zeros for a parameter."""
    if bits == 32:
        return tuple(torch.zeros(param.shape, dtype=torch.float32, device=param.device) for _ in range(2))
    if bits != 8:
        raise ValueError(f"states have 32 or 8 bits, got {bits}")
    scales = -(-param.numel() // BLOCK)
    return tuple(Quantized(torch.zeros(param.shape, dtype=dtype, device=param.device),
                           torch.zeros(scales, dtype=torch.float32, device=param.device))
                 for dtype in (torch.int8, torch.uint8))


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[State],
    exp_avg_sqs: Sequence[State],
    step: torch.Tensor,
    lr: float | torch.Tensor,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.0,
    masters: Sequence[torch.Tensor] | None = None,
    grad_scale: float | torch.Tensor | None = None,
    seed: int = 0,
) -> None:
    """One AdamW step of every tensor, in place:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  g = grad * grad_scale
        w = w (1 - lr weight_decay) - lr / (1 - b1^s) m / (sqrt(v / (1 - b2^s)) + eps)

    params, grads: contiguous bf16 / fp16 / fp32 tensors, each gradient of its
    parameter's shape. exp_avgs, exp_avg_sqs: fp32 tensors, or all of them
    Quantized (8 bits: rounded at random with odds that keep small changes,
    from seed, step and position). masters: fp32 weights updated in the
    parameters' place and rounded into them; without them a bf16 parameter
    loses what its own rounding loses. step: new_step's tensor; the call reads
    s - 1 from it and advances it. lr and grad_scale may be one-element fp32
    tensors on the GPU. All on one GPU; tensors must not overlap. Parameters
    and masters count as modified in place: a backward pass through a graph that
    saved one of them raises. (A captured step's replays tell no graph.)
    """
    from sparsebench_amd import _C

    _C.adamw_cuda(params, grads, masters, exp_avgs, exp_avg_sqs, step, lr, *betas, eps, weight_decay, grad_scale, seed)


def dequantize(states: Sequence[Quantized], dtype: torch.dtype = torch.float32) -> list[torch.Tensor]:
    """The values that 8-bit states stand for, as views into one buffer."""
    from sparsebench_amd import _C

    return _C.dequantize_cuda(states, dtype)


class AdamW:
    """adamw_step with its states: step(grads) updates the parameters given here.

    state_bits: 32 or 8. master_weights: fp32 masters of all parameters, copied
    from them here (self.masters); each step writes the parameters from them."""

    def __init__(
        self,
        params: Iterable[torch.Tensor],
        lr: float | torch.Tensor = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0.0,
        state_bits: int = 32,
        master_weights: bool = False,
        seed: int = 0,
    ) -> None:
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        self.lr, self.betas, self.eps, self.weight_decay, self.seed = lr, betas, eps, weight_decay, seed
        states = [new_state(p, state_bits) for p in self.params]
        self.exp_avgs, self.exp_avg_sqs = [s[0] for s in states], [s[1] for s in states]
        self.masters = [p.detach().to(torch.float32, copy=True) for p in self.params] if master_weights else None
        self.step_count = new_step(self.params[0].device)

    def step(self, grads: Sequence[torch.Tensor], grad_scale: float | torch.Tensor | None = None) -> None:
        """One step; grads[i] is the gradient of the i-th parameter."""
        adamw_step(self.params, grads, self.exp_avgs, self.exp_avg_sqs, self.step_count, self.lr, self.betas, self.eps,
                   self.weight_decay, self.masters, grad_scale, self.seed)


# ---- orthogonalised updates ----


def orthogonalize(matrices: torch.Tensor, steps: int = 5) -> torch.Tensor:
    """Newton-Schulz products of each matrix of a stack [..., rows, columns]: with the
    smaller side as rows,

        X = M / (|M| + 1e-7),  steps times X = a X + (b A + c A^2) X,  A = X X^T

    (a, b, c) = (3.4445, -4.7750, 2.0315), which takes singular values from (0, 1] towards 1
    (to about [0.7, 1.2] in five steps). bf16 / fp16 / fp32, of any strides whose rows are
    contiguous, and of any size of under 2^30 values with sides padded to 64. The products
    take fp16 operands, sum in fp32, and keep X to twice fp16's bits: in up to five steps the
    result is within 0.5% of exact arithmetic's, in the matrix's norm, wherever its singular
    values lie (0.03 to 0.06% for noise with some strong directions), before it is rounded to
    the input's type; in eight within 1%. Each step raises weak directions up to 3.44-fold,
    and X's last bits (2^-23) with them: in twelve a matrix of nearly low rank is no longer
    told from its rounding, as in fp32. Matrices do not mix, but how many there are of a size
    chooses the kernels' tiles, and with them the last bits."""
    from sparsebench_amd import _C

    return _C.orthogonalize_cuda(matrices, steps)


def muon_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    momenta: Sequence[torch.Tensor],
    lr: float | torch.Tensor,
    momentum: float = 0.95,
    nesterov: bool = True,
    weight_decay: float = 0.0,
    update_rms: float = 0.2,
    steps: int = 5,
    masters: Sequence[torch.Tensor] | None = None,
    grad_scale: float | torch.Tensor | None = None,
) -> None:
    """One orthogonalised step of every matrix of every tensor, in place:

        m = momentum m + (1 - momentum) g,  g = grad * grad_scale
        u = (1 - momentum) g + momentum m  (nesterov), or m
        w = w (1 - lr weight_decay) - lr update_rms sqrt(max(rows, columns)) orthogonalize(u)

    so that an update's values have about the size update_rms (0.2: AdamW's, whose lr
    then fits). params, grads: bf16 / fp16 / fp32 tensors [..., rows, columns], each
    gradient of its parameter's shape; momenta: fp32, likewise, zeros at first. Their
    rows must be contiguous, and may lie any strides apart: w1[..., :F] and w1[..., F:] of
    the gated layer are two stacks, each expert's gate and up matrix orthogonalised by
    itself. masters: fp32 weights updated in the parameters' place and rounded into them.
    lr and grad_scale may be one-element fp32 tensors on the GPU. All on one GPU; tensors
    must not overlap (an fp32 parameter may be its own master, and a gradient its own parameter). Matrices of one size are
    taken together, those of 16 tensors at a time. A step takes a workspace for the most that
    are taken together: 8 to 14 bytes a value of theirs (the squarer, the more; sides are
    padded to 64, 128 or 256), up to 6 GiB where that holds a matrix. Parameters and masters
    count as modified in place, as in adamw_step; nothing syncs, and a step can be captured."""
    from sparsebench_amd import _C

    _C.muon_cuda(params, grads, momenta, masters, lr, momentum, nesterov, weight_decay, update_rms, steps, grad_scale)


class Muon:
    """muon_step with its momenta: step(grads) updates the matrices given here.

    master_weights: fp32 masters of all parameters, copied from them here (self.masters)."""

    def __init__(
        self,
        params: Iterable[torch.Tensor],
        lr: float | torch.Tensor = 1e-3,
        momentum: float = 0.95,
        nesterov: bool = True,
        weight_decay: float = 0.0,
        update_rms: float = 0.2,
        steps: int = 5,
        master_weights: bool = False,
    ) -> None:
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        self.lr, self.momentum, self.nesterov, self.weight_decay = lr, momentum, nesterov, weight_decay
        self.update_rms, self.steps = update_rms, steps
        self.momenta = [torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in self.params]
        # A view's copy keeps its strides; rows are all that the step needs contiguous.
        self.masters = [p.detach().to(torch.float32, copy=True) for p in self.params] if master_weights else None

    def step(self, grads: Sequence[torch.Tensor], grad_scale: float | torch.Tensor | None = None) -> None:
        """One step; grads[i] is the gradient of the i-th parameter."""
        muon_step(self.params, grads, self.momenta, self.lr, self.momentum, self.nesterov, self.weight_decay,
                  self.update_rms, self.steps, self.masters, grad_scale)
