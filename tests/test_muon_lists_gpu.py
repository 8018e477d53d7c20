"""Lists of many separate matrices: each launch's matrices choose its kernels, and the workspace
holds one launch's; a list that is refused leaves everything as it was."""

import ctypes

import pytest
import torch

from sparsebench_amd import _C, _lib, optim
from tests.test_muon_gpu import gradient

pytestmark = pytest.mark.gpu

DEV = "cuda"
A_LAUNCH = 16  # tensors of one size that go together


def make(count, rows, columns, dtype=torch.bfloat16):
    params = [gradient(rows, columns, seed=300 + i, scale=0.05, dtype=dtype) for i in range(count)]
    grads = [gradient(rows, columns, seed=700 + i, dtype=dtype) for i in range(count)]
    return params, grads, [torch.zeros(rows, columns, device=DEV) for _ in range(count)]


def workspace_bytes(params, grads, momenta):
    words = _C._muon_words(params, grads, momenta, None)
    size = ctypes.c_int64()
    _lib.check(_lib.lib().sb_muon_sizes(words.buffer_info()[0], len(params), ctypes.byref(size)))
    return size.value


@pytest.mark.parametrize(("count", "rows", "columns"), [(64, 768, 1024), (70, 520, 1100), (33, 300, 200), (18, 2048, 1024)])
def test_launches_take_what_they_hold(count, rows, columns) -> None:
    """All together the matrices would fill wide tiles, a launch's sixteen do not."""
    params, grads, momenta = make(count, rows, columns)
    assert workspace_bytes(params, grads, momenta) == workspace_bytes(*(t[:A_LAUNCH] for t in (params, grads, momenta)))
    want = [p.clone() for p in params]
    for i in range(0, count, A_LAUNCH):
        some = slice(i, i + A_LAUNCH)
        optim.muon_step(want[some], grads[some], [m.clone() for m in momenta[some]], 0.1)
    optim.muon_step(params, grads, momenta, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(params, want))


def test_a_refused_list_is_left_as_it_was() -> None:
    """A workspace that holds the first size's matrices and not the second's."""
    params = [gradient(2, 24, 40, seed=1), gradient(2, 300, 400, seed=2)]
    grads = [gradient(*p.shape, seed=3 + i) for i, p in enumerate(params)]
    momenta = [torch.zeros_like(p) for p in params]
    before = [t.clone() for t in (*params, *momenta)]
    small = workspace_bytes(params[:1], grads[:1], momenta[:1])
    workspace = torch.empty(small, dtype=torch.uint8, device=DEV)
    words = _C._muon_words(params, grads, momenta, None)
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        rc = _lib.lib().sb_muon(words.buffer_info()[0], 2, 0.1, None, 0.9, 1, 0.0, 0.2, 5, None, workspace.data_ptr(), small,
                                stream)
        assert rc != 0 and "needed" in _lib.lib().sb_last_error().decode()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (*params, *momenta)))
    words = _C._muon_words(params, grads, momenta, None)
    assert _lib.lib().sb_muon(words.buffer_info()[0], 1, 0.1, None, 0.9, 1, 0.0, 0.2, 5, None, workspace.data_ptr(), small,
                              stream) == 0
    assert not torch.equal(before[0], params[0])
