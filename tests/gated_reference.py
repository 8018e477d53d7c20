"""The gated layer and its gradients in 64 bits, with a bound on how far the
kernels' results may lie from them.

Every product, rounding and approximation of the kernels' chain adds its own
worst case to the bound, carried through the rest of the chain with absolute
values:

    u = 2^-8     a rounding to bf16 (torch.finfo(torch.bfloat16).eps / 2)
    K 2^-24 |a||b|   an fp32 dot product of K terms in any order
    2^-20 |G|    an activation in fp32 (exp2 and a reciprocal to 1 ulp; erfc to
                 1.5e-7), 2^-20 its slope; slopes stay under 1.13, and their
                 own slopes under 0.8

Roundings (bf16): H, G and U as the backward pass reads them, y, [dG | dU],
w H, each row of dx before the sum over a token's copies, and every result.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

U = 2.0**-8
E32 = 2.0**-24


def act64(name: str, g: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


@dataclass
class Reference:
    value: dict[str, torch.Tensor]
    bound: dict[str, torch.Tensor]


def gated_reference(x, idx, gates, w1, w2, act="silu", grad_out=None) -> Reference:
    """CPU tensors; ids outside [0, E) route nowhere."""
    t, d = x.shape
    e, f, _ = w2.shape
    k = idx.shape[1]
    x64, g64 = x.double(), gates.double()
    out, out_b = torch.zeros(t, d).double(), torch.zeros(t, d).double()
    if grad_out is not None:
        go = grad_out.double()
        dx, dx_b = torch.zeros_like(out), torch.zeros_like(out)
        dg, dg_b = torch.zeros(t, k).double(), torch.zeros(t, k).double()
        dw1, dw1_b = torch.zeros(e, d, 2 * f).double(), torch.zeros(e, d, 2 * f).double()
        dw2, dw2_b = torch.zeros(e, f, d).double(), torch.zeros(e, f, d).double()
    for i in range(e):
        token, j = (idx == i).nonzero(as_tuple=True)
        n = len(token)
        if n == 0:
            continue
        a1, a2 = w1[i].double(), w2[i].double()
        xe, w = x64[token], g64[token, j][:, None]
        gu = xe @ a1
        gu_b = d * E32 * (xe.abs() @ a1.abs())
        g, u, g_b, u_b = gu[:, :f], gu[:, f:], gu_b[:, :f], gu_b[:, f:]
        a, slope = act64(act, g)
        h = a * u
        h_b = u.abs() * (1.13 * g_b + 2.0**-20 * g.abs()) + a.abs() * u_b + 2 * E32 * h.abs()
        h_b = h_b + U * (h.abs() + h_b)
        y = h @ a2
        y_b = h_b @ a2.abs() + f * E32 * ((h.abs() + h_b) @ a2.abs())
        y_b = y_b + U * (y.abs() + y_b)
        out.index_add_(0, token, w * y)
        out_b.index_add_(0, token, w.abs() * (y_b + (k + 1) * E32 * y.abs()))
        if grad_out is None:
            continue
        ge = go[token]
        dg[token, j] = (ge * y).sum(1)
        dg_b[token, j] = (ge.abs() * (y_b + d * E32 * y.abs())).sum(1)
        dh = w * (ge @ a2.t())
        dh_b = w.abs() * ((d + 2) * E32 * (ge.abs() @ a2.abs().t()))
        gr_b, ur_b = g_b + U * (g.abs() + g_b), u_b + U * (u.abs() + u_b)
        d_g = dh * u * slope
        d_g_b = ((u * slope).abs() * dh_b + (dh * slope).abs() * ur_b
                 + (dh * u).abs() * (0.8 * gr_b + 2.0**-20) + 3 * E32 * d_g.abs())
        d_u = dh * a
        d_u_b = a.abs() * dh_b + dh.abs() * (1.13 * gr_b + 2.0**-20 * g.abs()) + 2 * E32 * d_u.abs()
        dgu = torch.cat([d_g, d_u], 1)
        dgu_b = torch.cat([d_g_b, d_u_b], 1)
        dgu_b = dgu_b + U * (dgu.abs() + dgu_b)
        row = dgu @ a1.t()
        row_b = dgu_b @ a1.abs().t() + 2 * f * E32 * ((dgu.abs() + dgu_b) @ a1.abs().t())
        row_b = row_b + U * (row.abs() + row_b)
        dx.index_add_(0, token, row)
        dx_b.index_add_(0, token, row_b + k * E32 * row.abs())
        wh = w * h
        wh_b = w.abs() * (u.abs() * (1.13 * gr_b + 2.0**-20 * g.abs()) + a.abs() * ur_b + 3 * E32 * h.abs())
        wh_b = wh_b + U * (wh.abs() + wh_b)
        dw1[i] = xe.t() @ dgu
        dw1_b[i] = xe.abs().t() @ (dgu_b + n * E32 * (dgu.abs() + dgu_b))
        dw2[i] = wh.t() @ ge
        dw2_b[i] = (wh_b + n * E32 * (wh.abs() + wh_b)).t() @ ge.abs()
    value, bound = {"out": out}, {"out": out_b}
    if grad_out is not None:
        value |= {"x": dx, "gates": dg, "w1": dw1, "w2": dw2}
        bound |= {"x": dx_b, "gates": dg_b, "w1": dw1_b, "w2": dw2_b}
    for name in bound:
        half = torch.finfo(gates.dtype).eps / 2 if name == "gates" else U
        bound[name] = bound[name] * (1 + half) + half * value[name].abs() + 1e-30
    return Reference(value, bound)


# Roundings in each result's chain. Independent ones of at most U each, spread
# evenly, add up to about U sqrt(count / 3) of the result's 2-norm, where it
# holds enough values: a single one may cancel (a gate's gradient <grad_out, y>
# can be as near 0 as it likes, its error stays U |grad_out * y|'s 2-norm), so
# the norm says something from MANY values on.
MANY = 64
CHAIN = {"out": 3, "gates": 3, "x": 6, "w1": 5, "w2": 4}


def assert_close(name: str, got: torch.Tensor, ref: Reference) -> None:
    """Element by element within the bound, and in the 2-norm within twice what
    the roundings of the chain amount to."""
    got, want, bound = got.double().cpu(), ref.value[name], ref.bound[name]
    assert got.shape == want.shape
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{name}: {int((off > bound).sum())} of {off.numel()} values out of bounds, " \
                                       f"the worst by {float((off / bound).max()):.2f} times"
    norm = float(want.norm())
    if norm and want.numel() >= MANY:
        rel = float((got - want).norm()) / norm
        assert rel <= 2 * U * math.sqrt(CHAIN[name] / 3), f"{name}: off by {rel:.2e} in the 2-norm"
