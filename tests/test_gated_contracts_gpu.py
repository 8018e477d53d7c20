"""What the gated layer's documents promise beyond its results: training's
forward pass gives serving's bits, and rows behind the valid tokens stay as they
were in every result; and its second product where H passes 2 GiB."""

import pytest
import torch

from tests.gated_reference import assert_close, gated_reference
from tests.test_gated_gpu import GATES, make

pytestmark = pytest.mark.gpu


def by_counts(counts, d, f, seed):
    """One copy a token, `counts` of them for each expert, shuffled."""
    counts = torch.tensor(counts)
    x, _, gates, w1, w2, grad = make(int(counts.sum()), 1, len(counts), d, f, seed=seed)
    idx = torch.repeat_interleave(torch.arange(len(counts)), counts)
    return x, idx[torch.randperm(len(idx), generator=torch.Generator().manual_seed(seed))][:, None], gates, w1, w2, grad


# Row blocks; chunks of each height with the three staged at once (up to 192
# rows) and one after another; split and unsplit second products, their own and the layer's.
FORMS = {
    "row blocks": lambda: make(250, 2, 8, 256, 512, seed=1),
    "row blocks, bad ids": lambda: make(77, 3, 5, 128, 384, seed=2, ids="bad"),
    "short chunks": lambda: by_counts([64, 65, 128, 129, 191, 192, 1, 0] * 10, 256, 640, 3),
    "tall chunks": lambda: by_counts([193, 256, 257, 320, 321, 542, 255, 30] * 6, 640, 640, 4),
    "one expert": lambda: make(2200, 8, 9, 128, 1280, seed=5, ids="one"),
    "split": lambda: make(18, 3, 3, 384, 6400, seed=6),
    "split chunks": lambda: make(2300, 8, 8, 256, 640, seed=7),
    "three tokens": lambda: make(3, 2, 64, 256, 256, seed=8),
}


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("form", FORMS)
def test_training_s_forward_pass_gives_serving_s_bits(form, act) -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, _ = (v.cuda() for v in FORMS[form]())
    assert torch.equal(moe.moe_forward_gated(x, idx, gates, w1, w2, act),
                       moe.moe_gated_train(x, idx, gates, w1, w2, act)[0])


@pytest.mark.parametrize("gate_dtype", GATES)
@pytest.mark.parametrize(("t", "k", "valid"), [(700, 2, 300), (200, 3, 199), (64, 4, 0), (65, 1, 1), (2, 2, 1)])
def test_training_leaves_rows_behind_the_valid_tokens(t, k, valid, gate_dtype) -> None:
    """Results that hold a pattern before the C calls, ids out of range on both sides of the border."""
    from sparsebench_amd import _C, moe
    from sparsebench_amd._lib import check, lib, stream_of

    e, d, f = 4, 256, 256
    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(t, k, e, d, f, seed=t, ids="bad", gate_dtype=gate_dtype))
    vt = torch.tensor([valid], dtype=torch.int32, device="cuda")
    _, saved_size, train_size, backward_size = _C.gated_bytes(t, k, e, d, f)
    saved, train, backward = (torch.empty(n, dtype=torch.uint8, device="cuda")
                              for n in (saved_size, train_size, backward_size))
    out, grad_x, grad_gates = (torch.full_like(v, 7.0) for v in (x, x, gates))
    grad_w1, grad_w2 = torch.full_like(w1, 7.0), torch.full_like(w2, 7.0)
    code, stream = _C._GATE_DTYPES[gate_dtype], stream_of(x.device)
    check(lib().sb_gated_train(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), code, w1.data_ptr(), w2.data_ptr(),
                               out.data_ptr(), 0, saved.data_ptr(), saved_size, train.data_ptr(), train_size, t, k, e, d,
                               f, vt.data_ptr(), stream))
    check(lib().sb_gated_backward(grad.data_ptr(), x.data_ptr(), gates.data_ptr(), code, w1.data_ptr(), w2.data_ptr(),
                                  saved.data_ptr(), saved_size, grad_x.data_ptr(), grad_gates.data_ptr(),
                                  grad_w1.data_ptr(), grad_w2.data_ptr(), 0, backward.data_ptr(), backward_size, t, k, e,
                                  d, f, vt.data_ptr(), stream))
    for v in (out, grad_x, grad_gates):
        assert torch.all(v[valid:] == 7.0)
    ref = gated_reference(*(v[:valid].cpu() for v in (x, idx, gates)), w1.cpu(), w2.cpu(), "silu", grad[:valid].cpu())
    for name, got in (("out", out[:valid]), ("x", grad_x[:valid]), ("gates", grad_gates[:valid]), ("w1", grad_w1),
                      ("w2", grad_w2)):
        assert_close(name, got, ref)


def test_h_of_more_than_two_gigabytes() -> None:
    """D a multiple of 256, where smaller layouts take the layer's own second product."""
    from sparsebench_amd import moe

    t, k, e, d, f = 33_000, 2, 2, 256, 16_384
    g = torch.Generator(device="cuda").manual_seed(1)
    x, grad = (torch.randn(t, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    idx = torch.randint(0, e, (t, k), generator=g, device="cuda")
    gates = torch.rand(t, k, generator=g, device="cuda") + 0.5
    w1 = (torch.randn(e, d, 2 * f, generator=g, device="cuda") / d**0.5).bfloat16()
    w2 = (torch.randn(e, f, d, generator=g, device="cuda") / f**0.5).bfloat16()
    served = moe.moe_forward_gated(x, idx, gates, w1, w2)
    out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    grads = moe.moe_gated_backward(saved, grad)
    assert torch.equal(served, out)
    some = torch.cat([torch.arange(40), torch.arange(t // 2, t // 2 + 40), torch.arange(t - 40, t)]).cuda()
    ref = gated_reference(*(v[some].cpu() for v in (x, idx, gates)), w1.cpu(), w2.cpu(), "silu", grad[some].cpu())
    assert_close("out", out[some], ref)
    assert_close("x", grads.x[some], ref)
    assert_close("gates", grads.expert_weight[some], ref)
