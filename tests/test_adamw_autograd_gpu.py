"""AdamW steps and autograd: what a live graph has saved must not change under it unnoticed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_that_saved_a_parameter_notices_the_step(bits) -> None:
    from sparsebench_amd import optim

    w = torch.ones(300, device="cuda", requires_grad=True)
    other = torch.ones(300, device="cuda", requires_grad=True)
    opt = optim.AdamW([w], state_bits=bits)
    loss, untouched = (w * w).sum(), (other * other).sum()
    opt.step([torch.ones_like(w)])
    untouched.backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (w * w).sum().backward()  # a graph of the new values
    assert torch.equal(w.grad, 2 * w.detach())


def test_masters_move_on_too_and_refused_calls_nothing() -> None:
    from sparsebench_amd import optim

    w = torch.ones(300, dtype=torch.bfloat16, device="cuda")
    opt = optim.AdamW([w], master_weights=True)
    before = w._version, opt.masters[0]._version
    with pytest.raises(RuntimeError, match="shape"):
        opt.step([torch.ones(299, device="cuda")])
    assert (w._version, opt.masters[0]._version) == before
    opt.step([torch.ones_like(w)])
    assert w._version > before[0] and opt.masters[0]._version > before[1]
