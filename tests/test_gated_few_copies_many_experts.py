"""The gated layer where there are fewer copies than experts: rows, workspaces
and grids go by the row blocks that can hold a copy, not by every expert's padding."""

import pytest

from sparsebench_amd import _C, _lib

SHAPES = [(3, 1, 256, 4096, 2048), (3, 2, 200, 2048, 4096), (24, 2, 64, 1024, 4096), (1, 8, 1024, 1024, 512)]


@pytest.mark.parametrize(("t", "k", "e", "d", "f"), SHAPES)
def test_workspaces_hold_the_rows_that_copies_can_have(t, k, e, d, f) -> None:
    try:
        _lib.lib()
    except _lib.LibraryNotBuilt as error:
        pytest.skip(str(error))
    layer, saved, train, backward = _C.gated_bytes(t, k, e, d, f)
    rows = 128 * min(t * k, (t * k + 127 * e) // 128)
    # The routing's layout: a word a padded row, two a row block and one a block of H, a few an expert or copy.
    routing = 4 * ((128 + f // 128 + 2) * (t * k + e) + 4 * (t * k + e)) + 4096
    parts = 16 * rows * d * 4  # of a split product
    assert saved <= rows * (2 * f + d) * 2 + routing
    assert train <= rows * f * 2 + parts + routing
    assert layer <= max(rows * (f + d) * 2 + parts + routing, 4 * t * k * (16 * f + 16 * d) + 4096)
    assert backward <= rows * (3 * f + 3 * d) * 2 + parts + routing


# Split and unsplit products, row blocks and chunks, ids of one expert or out of range; more than 127 copies.
@pytest.mark.gpu
@pytest.mark.parametrize(("t", "k", "e", "d", "f", "ids"), [
    (3, 1, 160, 128, 1152, "random"), (5, 2, 200, 128, 1664, "random"), (3, 2, 64, 384, 2944, "one"),
    (9, 1, 60, 256, 2944, "bad"), (150, 1, 250, 256, 128, "random"), (170, 1, 180, 128, 1280, "random"),
    (60, 3, 256, 128, 512, "bad"), (300, 1, 301, 512, 128, "random"), (40, 8, 330, 128, 256, "random"),
    (1, 66, 256, 128, 256, "random")])
def test_matches_64_bits(t, k, e, d, f, ids) -> None:
    from tests.test_gated_gpu import check_all, make

    check_all(make(t, k, e, d, f, seed=t + e, ids=ids), valid=None if t % 2 else t - 1)


@pytest.mark.gpu
def test_rows_of_neighbours_stay_as_they_were() -> None:
    """Training through the C calls in workspaces of exactly the bytes asked for, with a pattern behind them."""
    import torch

    from sparsebench_amd._lib import check, lib, stream_of
    from tests.test_gated_gpu import make

    t, k, e, d, f = 5, 2, 200, 256, 1664
    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(t, k, e, d, f, seed=3))
    _, saved_size, train_size, backward_size = _C.gated_bytes(t, k, e, d, f)
    buffers = [torch.full((n + 4096,), 85, dtype=torch.uint8, device="cuda")
               for n in (saved_size, train_size, backward_size)]
    out, grads = torch.empty_like(x), [torch.empty_like(v) for v in (x, gates, w1, w2)]
    stream = stream_of(x.device)
    check(lib().sb_gated_train(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                               out.data_ptr(), 0, buffers[0].data_ptr(), saved_size, buffers[1].data_ptr(), train_size,
                               t, k, e, d, f, None, stream))
    check(lib().sb_gated_backward(grad.data_ptr(), x.data_ptr(), gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                                  buffers[0].data_ptr(), saved_size, *(g.data_ptr() for g in grads), 0,
                                  buffers[2].data_ptr(), backward_size, t, k, e, d, f, None, stream))
    torch.cuda.synchronize()
    for buffer, size in zip(buffers, (saved_size, train_size, backward_size)):
        assert bool((buffer[size:] == 85).all())
    from sparsebench_amd import moe

    want, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(grads, moe.moe_gated_backward(saved, grad)))


@pytest.mark.gpu
def test_every_copy_on_an_expert_of_its_own(hooks) -> None:
    """240 copies over 250 experts: the second product's tiles by expert, by row block and
    as it chooses, in a workspace of NaN, which a tile that no workgroup takes would leave."""
    import torch

    from sparsebench_amd._lib import check, lib, stream_of
    from tests.test_gated_gpu import make

    t, e, d, f = 240, 250, 2048, 128
    x, idx, gates, w1, w2, _ = (v.cuda() for v in make(t, 1, e, d, f, seed=6))
    idx.copy_(torch.randperm(e, generator=torch.Generator().manual_seed(1))[:t, None])
    workspace = torch.empty(_C.gated_bytes(t, 1, e, d, f)[0] // 2, dtype=torch.bfloat16, device="cuda")
    outs = []
    for gate in (0, 1, 2):
        hooks.expert_gate(gate)
        workspace.fill_(float("nan"))
        outs.append(torch.zeros_like(x))
        check(lib().sb_gated_layer(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                                   outs[-1].data_ptr(), 0, workspace.data_ptr(), 2 * workspace.numel(), t, 1, e, d, f,
                                   None, stream_of(x.device)))
    assert torch.isfinite(outs[0].float()).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
