"""Which lists of tensors the orthogonalised step refuses for overlapping, on the CPU: against the
addresses of all their values."""

import array
import random

import pytest
import torch

from sparsebench_amd import _C, optim
from tests.test_muon_refusals import lib  # noqa: F401


def view(flat, g):
    """A stack of matrices somewhere in flat, with the strides of one of a few layouts."""
    kind = g.choice(["columns", "rows", "matrices", "one"])
    e, r, c = g.randint(1, 3), g.randint(1, 4), g.randint(1, 6)
    whole = flat[g.randint(0, 40):]
    if kind == "columns":  # of a wider weight
        wide, r = g.choice([6, 12]), g.choice([r, 4])
        at = g.randint(0, wide - c)
        return whole[:e * r * wide].view(e, r, wide)[:, :, at:at + c]
    if kind == "rows":
        tall, c = 4, g.choice([6, 12])
        return whole[:e * tall * c].view(e, tall, c)[:, tall - r:]
    if kind == "matrices":  # matrices nearer to each other than rows
        return whole[:e * r * c].view(r, e, c).transpose(0, 1)
    return whole[:r * c].view(r, c)


def bytes_of(t):
    at = torch.zeros((), dtype=torch.int64)
    for size, stride in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(size) * stride
    return {t.data_ptr() + int(i) * t.element_size() + b for i in at.flatten() for b in range(t.element_size())}


APART = 1 << 40  # where no view is
FAR = iter(range(APART, 1 << 46, 1 << 20))


def refused(lib, tensors):  # noqa: F811
    """Of (param, grad, momentum, master) tensors or None, which then lie apart from all others.
    The workspace is too small for any list, so nothing is launched."""
    words = array.array("q")
    for p, g, m, w in tensors:
        shape = p if p is not None else next(t for t in (g, m, w) if t is not None)
        stacks = [None if t is None else _C._stack_of(t, "tensor", False) for t in (p, g, m, w)]
        e, r, c = next(s for s in stacks if s is not None)[:3]
        at = [next(FAR) if t is None else t.data_ptr() for t in (p, g, m)] + [0 if w is None else w.data_ptr()]
        strides = [s[3:] if s is not None else (r * c, c) for s in stacks]
        types = [2 if t is None or t.dtype is torch.float32 else 0 for t in (p, g)]
        assert shape.numel() == e * r * c
        words.extend((*at, e, r, c, *(v for s in strides for v in s), types[0] | types[1] << 32))
    assert lib.sb_muon(words.buffer_info()[0], len(tensors), 0.1, None, 0.9, 1, 0.0, 0.2, 5, None, 4096, 1, None) != 0
    return "must not overlap" in lib.sb_last_error().decode()


def lattice(t):
    """Strides in bytes by size of those that count: lists of the same are told apart for certain."""
    dims = [(s * t.element_size(), n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1]
    return sorted(dims, reverse=True)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_against_all_addresses(lib, types) -> None:  # noqa: F811
    g, flat = random.Random(5), torch.zeros(600)
    found = {True: 0, False: 0}
    for i in range(8000):
        a, b = (view(flat.view(t), g) for t in types)
        share = bool(bytes_of(a) & bytes_of(b))
        others = [(a, None, None, None), (b, None, None, None)] if i % 2 else [(a, None, b, None)]
        if i % 2 == 0 and a.shape != b.shape:
            continue
        got = refused(lib, others)
        assert not got or share
        if [s for s, _ in lattice(a)] == [s for s, _ in lattice(b)]:
            assert got == share
            found[got] += 1
    assert min(found.values()) > 50, found


def test_lists(lib) -> None:  # noqa: F811
    w = torch.zeros(4, 6, 10)
    m, g = torch.zeros(4, 6, 5), torch.ones(4, 6, 5)
    n, h = m.clone(), g.clone()
    a, b = w[..., :5], w[..., 5:]
    half = torch.zeros(4, 6, 10, dtype=torch.bfloat16)
    for taken in (
        [(a, g, m, None), (b, h, n, None)],
        [(a, g, m, a), (b, g, n, b)],  # their own masters, one gradient for both
        [(a, a, m, None), (b, b, n, b)],  # gradients that are read before weights are written
        [(half[..., :5], a, m, a), (half[..., 5:], b, n, b)],
        [(w[:2], w[:2], None, None), (w[2:], w[2:], None, None)],
        [(w[:, ::2], torch.ones(1, 3, 10).expand(4, 3, 10), None, None), (w[:, 1::2], None, None, None)],
        [],
    ):
        assert not (taken and refused(lib, taken))
    for overlapping in (
        [(w[..., :6], None, None, None), (w[..., 4:], None, None, None)],
        [(a, g, m, None), (b, h, m, None)],
        [(a, g, m, None), (b, h, g, None)],
        [(a, g, m, b), (b, h, n, a)],
        [(a, b, m, None), (b, a, n, None)],
        [(a, m, m, None)],
        [(a, g, a, None)],
        [(a, g, m, m)],
        [(w[:3], None, None, None), (w[2:], None, None, None)],
        [(w[:, :4], None, None, None), (w[:, 3:], None, None, None)],
        [(a, w[..., 1:6], m, None)],
        [(a, g, m, None), (a, g, n, None)],
    ):
        assert refused(lib, overlapping)


@pytest.mark.gpu
def test_step_refuses_values_in_two_places() -> None:
    w = torch.zeros(2, 32, 48, device="cuda")
    a, b = w[..., :30], w[..., 20:]
    grads, momenta = [torch.ones_like(a), torch.ones_like(b)], [torch.zeros_like(a), torch.zeros_like(b)]
    with pytest.raises(RuntimeError, match="must not overlap"):
        optim.muon_step([a, b], grads, momenta, 0.1)
    with pytest.raises(RuntimeError, match="must not overlap"):
        optim.muon_step([a], [momenta[0]], [momenta[0]], 0.1)
    assert not w.any() and not momenta[0].any()
    optim.muon_step([w[..., :24], w[..., 24:]], [g[..., :24] for g in grads], [m[..., :24] for m in momenta], 0.1)
    assert w.all()
