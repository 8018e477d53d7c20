"""AdamW steps whose second moments are fp32 subnormals, against 64 bits: the
root under the step is theirs, however small eps is."""

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0**-24


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [5, 4096])
@pytest.mark.parametrize(("g", "eps"), [(1e-16, 1e-30), (1e-18, 1e-30), (1e-20, 1e-30), (1e-20, 1e-20), (2e-21, 1e-24)])
def test_steps_from_subnormal_second_moments(bits, n, g, eps) -> None:
    """The first step of a zero state goes by g / (|g| + eps), whatever |g| is. v is a
    subnormal of steps 2^-149: its root is off by half of that over 2 v, at most."""
    from sparsebench_amd import optim

    lr, betas = 1e-3, (0.9, 0.999)
    p, grad = torch.ones(n, device="cuda"), torch.full((n,), g, device="cuda")
    grad[1] = 0
    m, v = optim.new_state(p, bits)
    optim.adamw_step([p], [grad], [m], [v], optim.new_step(), lr, betas, eps)
    exact = grad.double()
    want = 1 - lr * exact / (exact.abs() + eps)
    v1 = (1 - betas[1]) * g * g
    # Products, two roundings of v, root, coefficients, reciprocal: 16 E; the weight's own 2 E.
    off = lr * (16 * E + 2 * 2.0**-149 / v1) + 2 * E
    assert ((p.double() - want).abs() <= off).all()
