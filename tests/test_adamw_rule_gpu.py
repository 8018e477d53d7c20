"""The 8-bit AdamW step over several steps against its rule, in numpy: fp32
operations one by one, each rounded to nearest, with nothing read back in
between. Codes and scales have to be the same bits.

    m = b1 m + a1 g,  v = b2 v + (a2 g) g      a = fp32(1 - b)
    scale_m = max |m| fp32(1 / 127^2),         scale_v = max sqrt(v) fp32(1 / 255^2)
    code = floor(sqrt(|m| / scale_m) + r / 2^16),   likewise of sqrt(v), at least 1 where v > 0

A weight follows in 64 bits from the moments before they are rounded to codes:
each step adds up to 16 roundings of its update (coefficients, square root,
reciprocal, products), up to 3 of the weight itself and up to 6 of the moments."""

import numpy as np
import pytest
import torch

from tests.test_adamw_gpu import BETAS, E, EPS, LR, SIZES, WD, mix, quantized, tensors

pytestmark = pytest.mark.gpu

F = np.float32


def bits_of(n: int, seed: int, step: int, tensor: int) -> np.ndarray:
    key = mix(mix(np.array([step * 0x9E3779B9 + seed])) ^ np.uint64(tensor))
    return mix(np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B9) + key)


def in_blocks(a: np.ndarray) -> np.ndarray:
    return np.pad(a, (0, -len(a) % 256)).reshape(-1, 256)


def encode(values: np.ndarray, most: int, part: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) of values >= 0."""
    b = in_blocks(values)
    scale = b.max(1) * (F(1) / F(most**2))
    root = np.sqrt(b / np.where(scale > 0, scale, F(1))[:, None]).reshape(-1)[: len(values)]
    return np.minimum(np.floor(root + part.astype(F) / F(65536)), F(most)), scale


def spread(scale: np.ndarray, n: int) -> np.ndarray:
    return np.repeat(scale, 256)[:n]


class Rule:
    """One tensor's states and, in 64 bits, its weights."""

    def __init__(self, w, m, v) -> None:
        self.w, self.off = w.double().cpu().numpy(), np.zeros(w.numel())
        self.m, self.ms = m.codes.cpu().numpy().astype(F), m.scales.cpu().numpy()
        self.v, self.vs = v.codes.cpu().numpy().astype(F), v.scales.cpu().numpy()

    def step(self, g: np.ndarray, s: int, seed: int, tensor: int, betas, eps: float) -> None:
        n = len(g)
        (b1, b2), (a1, a2) = (F(b) for b in betas), (F(1 - b) for b in betas)
        old_m = self.m * np.abs(self.m) * spread(self.ms, n)
        root = self.v * self.v * spread(self.vs, n)
        m, v = b1 * old_m + a1 * g, b2 * (root * root) + a2 * g * g
        size, under = LR / (1 - betas[0] ** s), np.sqrt(v.astype(float)) / (1 - betas[1] ** s) ** 0.5 + eps
        delta = size * m.astype(float) / under
        grow = np.abs(b1 * old_m) + np.abs(a1 * g)
        self.off += 16 * E * np.abs(delta) + 3 * E * np.abs(self.w) + 6 * E * size * grow / under
        self.w = self.w * (1 - LR * WD) - delta
        rand = bits_of(n, seed, s, tensor)
        code, self.ms = encode(np.abs(m), 127, rand & np.uint64(0xFFFF))
        self.m = np.where(m < 0, -code, code)
        code, self.vs = encode(np.sqrt(v), 255, rand >> np.uint64(16))
        self.v = np.where(v > 0, np.maximum(code, F(1)), code)


def follow(sizes, p_type, g_type, master=False, offset=0, steps=4, grad_size=1e-2, betas=BETAS, seed=77, fresh=False,
           eps=EPS):
    from sparsebench_amd import optim

    params = tensors(sizes, p_type, 1, 0.5, offset)
    masters = [p.float() for p in params] if master else None
    if fresh:
        states = [optim.new_state(p, 8) for p in params]
    else:
        m = tensors(sizes, torch.float32, 3, 0.3 * grad_size)
        v = tensors(sizes, torch.float32, 4, grad_size)
        states = [(quantized(a, True, offset), quantized(b.abs(), False, offset)) for a, b in zip(m, v)]
    at = 0 if fresh else 20
    step = torch.tensor([at, 0], dtype=torch.int32, device="cuda")
    rules = [Rule(p, *s) for p, s in zip(masters or params, states)]
    for s in range(at + 1, at + 1 + steps):
        grads = tensors(sizes, g_type, 10 + s, grad_size, offset)
        optim.adamw_step(params, grads, [a for a, _ in states], [b for _, b in states], step, LR, betas, eps, WD,
                         masters, None, seed)
        for i, (rule, g) in enumerate(zip(rules, grads)):
            rule.step(g.float().cpu().numpy(), s, seed, i, betas, eps)
    for i, (rule, (m, v)) in enumerate(zip(rules, states)):
        for name, want, got in (("exp_avg scales", rule.ms, m.scales), ("exp_avg_sq scales", rule.vs, v.scales),
                                ("exp_avg codes", rule.m, m.codes), ("exp_avg_sq codes", rule.v, v.codes)):
            differ = int((want != got.cpu().numpy().astype(F)).sum())
            assert differ == 0, f"tensor {i}, {name}: {differ} of {got.numel()} differ"
        if master or p_type == torch.float32:
            got = (masters or params)[i].double().cpu().numpy()
            assert (np.abs(got - rule.w) <= rule.off + 1e-30).all()


MANY = [1_500_000, 257, 2048 * 300 + 19]


def test_many_values() -> None:
    follow(MANY, torch.float32, torch.float32)


def test_many_values_with_masters_of_bf16() -> None:
    follow(MANY, torch.bfloat16, torch.bfloat16, master=True)


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("fresh", [False, True])
def test_odd_lengths_and_offsets(offset, fresh) -> None:
    follow(SIZES * 3, torch.float32, torch.bfloat16, offset=offset, fresh=fresh, steps=6)


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.5), (0.8, 0.0)])
def test_other_betas(betas) -> None:
    follow([300_000], torch.float32, torch.float32, betas=betas)


@pytest.mark.parametrize("grad_size", [1e-12, 1e-18, 1e-20, 3e-23, 1e-30, 1e4, 1e12])
def test_small_and_large_gradients(grad_size) -> None:
    """Second moments and scales down to fp32's subnormals, and zero where they end."""
    follow([100_000], torch.float32, torch.float32, grad_size=grad_size)
