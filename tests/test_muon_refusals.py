"""What the orthogonalised updates' entry points refuse, on the CPU: by their C calls
(before anything is launched) and by their Python functions."""

import array
import re

import pytest
import torch

from sparsebench_amd import _lib, optim


@pytest.fixture(scope="module")
def lib():
    try:
        return _lib.lib()
    except _lib.LibraryNotBuilt as e:
        pytest.skip(str(e))


P = 4096  # an aligned address that is never read


def words(param=P, grad=P, momentum=P, master=0, matrices=1, rows=8, columns=8, stride=8, types=0):
    return array.array("q", (param, grad, momentum, master, matrices, rows, columns, *(64, stride) * 4, types))


def muon(lib, w, count=1, momentum=0.9, steps=5):
    return lib.sb_muon(w.buffer_info()[0] if w is not None else None, count, 0.1, None, momentum, 1, 0.0, 0.2, steps,
                       None, P, 1 << 40, None)


def orthogonalize(lib, w, count=1, steps=5):
    return lib.sb_orthogonalize(w.buffer_info()[0] if w is not None else None, count, steps, P, 1 << 40, None)


@pytest.mark.parametrize(("change", "match"), [
    ({"param": 0}, "null buffer"),
    ({"grad": 0}, "null buffer"),
    ({"matrices": -1}, "negative size"),
    ({"rows": -1}, "negative size"),
    ({"columns": -3}, "negative size"),
    ({"rows": 2**31}, "2\\^30"),
    ({"rows": 2**15, "columns": 2**15 + 1}, "2\\^30"),
    ({"rows": 2**20, "columns": 2**20}, "2\\^30"),
    ({"matrices": 2**31}, "2\\^30"),
    ({"stride": -8}, "negative stride"),
    ({"types": 3}, "unsupported dtype"),
    ({"types": 5 << 32}, "unsupported dtype"),
])
def test_lists_are_refused(lib, change, match) -> None:
    w = words(**change)
    for call in (muon, orthogonalize, lambda lib, w: lib.sb_muon_sizes(w.buffer_info()[0], 1, None)):
        assert call(lib, w) == 1
        assert re.search(match, lib.sb_last_error().decode())


def test_other_arguments_are_refused(lib) -> None:
    def error():
        return lib.sb_last_error().decode()

    assert muon(lib, words(momentum=0)) == 1 and "null buffer" in error()
    assert muon(lib, None) == 1 and "null buffer" in error()
    assert muon(lib, words(), count=-1) == 1 and "null buffer" in error()
    for beta in (1.0, -0.1, float("nan")):
        assert muon(lib, words(), momentum=beta) == 1 and "momentum must be" in error()
    for steps in (0, 33, -1):
        assert muon(lib, words(), steps=steps) == 1 and "steps" in error()
        assert orthogonalize(lib, words(momentum=0), steps=steps) == 1 and "steps" in error()
    assert orthogonalize(lib, words()) == 1 and "neither momentum" in error()
    assert orthogonalize(lib, words(momentum=0, master=P)) == 1 and "neither momentum" in error()


def test_python_calls_refuse_cpu_tensors() -> None:
    w = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        optim.orthogonalize(w)
    with pytest.raises(RuntimeError, match="on one GPU"):
        optim.muon_step([w], [w], [w], 0.1)


def test_python_calls_refuse_lists_and_numbers() -> None:
    w = torch.zeros(4, 4)
    for args in (([w], [], [w]), ([w], [w], []), ([], [w], [])):
        with pytest.raises(RuntimeError, match="one length"):
            optim.muon_step(*args, 0.1)
    with pytest.raises(RuntimeError, match="one length"):
        optim.muon_step([w], [w], [w], 0.1, masters=[])
    with pytest.raises(RuntimeError, match="steps"):
        optim.muon_step([w], [w], [w], 0.1, steps=0)
    with pytest.raises(RuntimeError, match="steps"):
        optim.orthogonalize(w, steps=33)
    with pytest.raises(RuntimeError, match="momentum"):
        optim.muon_step([w], [w], [w], 0.1, momentum=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize(("make", "match"), [
    (lambda w: ([w[0, 0]], [w[0, 0]], [w[0, 0]]), "must be matrices"),
    (lambda w: ([w.double()], [w], [w]), "parameters must be of"),
    (lambda w: ([w], [w.int()], [w]), "gradients must be of"),
    (lambda w: ([w], [w], [w.bfloat16()]), "momenta must be of"),
    (lambda w: ([w], [w[:1]], [w]), "gradients must have the parameters' shapes"),
    (lambda w: ([w], [w], [w[:, :3]]), "momenta must have the parameters' shapes"),
    (lambda w: ([w.transpose(1, 2)], [w.transpose(1, 2)], [w.transpose(1, 2)]), "contiguous rows"),
    (lambda w: ([w[:1].expand(2, 4, 4)], [w], [w]), "overlap themselves"),
    (lambda w: ([w], [w], [w[:, :1].expand(2, 4, 4)]), "overlap themselves"),
    (lambda w: ([torch.zeros(2, 3, 4, 4, device="cuda").transpose(0, 1)],) * 3, "leading dimensions"),
    (lambda w: ([w], [w.cpu()], [w]), "on one GPU"),
])
def test_python_step_refuses(make, match) -> None:
    with pytest.raises(RuntimeError, match=match):
        optim.muon_step(*make(torch.zeros(2, 4, 4, device="cuda")), 0.1)


@pytest.mark.gpu
def test_python_step_refuses_masters_and_scalars() -> None:
    w = torch.zeros(2, 4, 4, device="cuda")
    with pytest.raises(RuntimeError, match="masters must be of"):
        optim.muon_step([w], [w], [w.clone()], 0.1, masters=[w.half()])
    with pytest.raises(RuntimeError, match="lr must be"):
        optim.muon_step([w], [w], [w.clone()], torch.zeros(1))
    with pytest.raises(RuntimeError, match="grad_scale must be"):
        optim.muon_step([w], [w], [w.clone()], 0.1, grad_scale=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="2\\^30"):
        optim.orthogonalize(torch.zeros(2**16, dtype=torch.float16, device="cuda").expand(2**15, 2**16))
