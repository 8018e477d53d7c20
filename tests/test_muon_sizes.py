"""Long matrices: what is accepted and refused (by the C calls, on the CPU), and their results."""

import pytest
import torch

from sparsebench_amd import optim
from tests.test_muon_refusals import lib, muon, orthogonalize, words  # noqa: F401


@pytest.mark.parametrize(("rows", "columns", "taken"), [
    (1, 2**22, True), (2**22, 1, True), (8, 2**22, True), (1, 2**24 - 64, True), (100, 2**22, True), (32704, 32768, True),
    (1, 2**24 - 63, False), (65, 2**23, False), (32768, 32705, False),
])
def test_bound_of_sizes(lib, rows, columns, taken) -> None:  # noqa: F811
    """Of values, sides padded to 64. A list that is taken fails at most for want of a GPU: the
    workspace here is too small for any."""
    w = words(rows=rows, columns=columns)
    for call in (lambda: lib.sb_muon(w.buffer_info()[0], 1, 0.1, None, 0.9, 1, 0.0, 0.2, 5, None, 4096, 1, None),
                 lambda: lib.sb_muon_sizes(w.buffer_info()[0], 1, None)):
        failed = call() != 0
        assert ("2^30" in lib.sb_last_error().decode()) == (not taken) if failed else taken


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 2**22), (2**22, 1), (8, 2**21 + 3), (2**21 + 5, 3), (70, 2**20 + 1)])
def test_long_matrices(size) -> None:
    """fp32 sums of n squares: off by 2^-24 sqrt(n) at most where roundings do not conspire, 0.012%
    for 2^22; the polynomial's five steps and the products' roundings as for short ones (0.4%)."""
    from tests.test_muon_gpu import PRODUCTS, newton_schulz

    u = torch.randn(*size, generator=torch.Generator("cuda").manual_seed(7), device="cuda")
    got, want = optim.orthogonalize(u), newton_schulz(u)
    assert (got.double() - want).norm() <= (PRODUCTS + 5 * 2.0**-24 * max(size) ** 0.5) * want.norm()
    assert torch.equal(u, torch.randn(*size, generator=torch.Generator("cuda").manual_seed(7), device="cuda"))
