"""What the gated layer's and the update's entry points refuse, on the CPU: by
their C calls (before anything is launched) and by their Python functions."""

import ctypes

import pytest
import torch

from sparsebench_amd import _C, _lib, moe, optim


@pytest.fixture(scope="module")
def lib():
    try:
        return _lib.lib()
    except _lib.LibraryNotBuilt as e:
        pytest.skip(str(e))


def error(lib) -> str:
    return lib.sb_last_error().decode()


@pytest.mark.parametrize(("args", "match"), [
    ((0, 2, 4, 128, 128), "T, k > 0"),
    ((4, 0, 4, 128, 128), "T, k > 0"),
    ((2**31, 1, 4, 128, 128), "T, k > 0"),
    ((4, 2, 0, 128, 128), "expert count"),
    ((4, 2, 2000, 128, 128), "num_experts"),
    ((4, 2, 4, 64, 128), "multiples of 128"),
    ((4, 2, 4, 128, 192), "multiples of 128"),
    ((4, 2, 4, 128, 0), "multiples of 128"),
    ((4, 2, 4, 32768, 32768), "too large"),
    ((2**26, 8, 4, 128, 128), "too large"),
])
def test_gated_sizes_refuse(lib, args, match) -> None:
    assert lib.sb_gated_sizes(*args, None, None, None, None) == 1
    assert match in error(lib)


@pytest.mark.parametrize(("d", "f"), [(128, 2**21), (2**22, 128)])
def test_rows_too_long_for_32_bit_offsets(lib, d, f) -> None:
    assert lib.sb_gated_sizes(4, 2, 4, d, f, None, None, None, None) == 1
    assert "32-bit" in error(lib)


def test_gated_sizes(lib) -> None:
    layer, saved, train, backward = _C.gated_bytes(100, 2, 4, 256, 384)
    rows = (200 + 4 * 127) // 128 * 128
    assert saved >= rows * (2 * 384 + 256) * 2 and layer >= rows * (384 + 256) * 2
    assert train >= rows * 384 * 2 and backward >= rows * (3 * 384 + 3 * 256) * 2


def test_gated_calls_refuse_null_misaligned_and_short(lib) -> None:
    shape = (4, 2, 4, 128, 128)
    layer, saved, train, backward = _C.gated_bytes(*shape)
    ok, ws = 4096, 1 << 20

    def forward(x=ok, act=0, gate=0, workspace=ws, size=layer):
        return lib.sb_gated_layer(x, ok, 0, ok, gate, ok, ok, ok, act, workspace, size, *shape, None, None)

    def run_train(kept=ws, kept_size=saved, size=train):
        return lib.sb_gated_train(ok, ok, 0, ok, 0, ok, ok, ok, 0, kept, kept_size, ws, size, *shape, None, None)

    def run_backward(grad=ok, kept_size=saved, size=backward, gates=ok):
        return lib.sb_gated_backward(grad, ok, ok, 0, ok, ok, ws, kept_size, ok, gates, ok, ok, 0, ws, size, *shape, None,
                                     None)

    for rc, match in [(lambda: forward(x=None), "null"), (lambda: forward(x=ok + 2), "16-byte"),
                      (lambda: forward(act=2), "activation"), (lambda: forward(gate=7), "dtype"),
                      (lambda: forward(workspace=ws + 16), "256-byte"), (lambda: forward(workspace=None), "256-byte"),
                      (lambda: forward(size=layer - 1), "workspace of"), (lambda: run_train(kept=None), "256-byte"),
                      (lambda: run_train(kept_size=saved - 1), "workspace of"),
                      (lambda: run_train(size=train - 1), "workspace of"),
                      (lambda: run_backward(grad=ok + 8), "16-byte"), (lambda: run_backward(gates=None), "null"),
                      (lambda: run_backward(kept_size=saved - 1), "workspace of"),
                      (lambda: run_backward(size=backward - 1), "workspace of")]:
        assert rc() == 1
        assert match in error(lib)


def test_adamw_and_dequantize_refuse(lib) -> None:
    import array

    def call(words=(4096, 4096, 0, 4096, 4096, 0, 0, 8, 0), count=1, bits=32, step=4096, betas=(0.9, 0.99)):
        a = array.array("q", words)
        return lib.sb_adamw(a.buffer_info()[0], count, bits, step, 0.1, None, *betas, 1e-8, 0.0, None, 0, None)

    for rc, match in [(lambda: call(bits=16), "32 or 8"), (lambda: call(step=None), "null"),
                      (lambda: call(count=-1), "null"), (lambda: call(betas=(1.0, 0.9)), "betas"),
                      (lambda: call(betas=(0.9, float("nan"))), "betas"), (lambda: call(bits=8), "null"),
                      (lambda: call(words=(0, 4096, 0, 4096, 4096, 0, 0, 8, 0)), "null"),
                      (lambda: call(words=(4096, 4096, 0, 4096, 4096, 0, 0, -1, 0)), "negative"),
                      (lambda: call(words=(4096, 4096, 0, 4096, 4096, 0, 0, 8, 5)), "dtype"),
                      (lambda: call(words=(4096, 4096, 0, 4096, 4096, 0, 0, 8, 9 << 32)), "dtype"),
                      (lambda: lib.sb_dequantize(None, 1, 0, None), "null"),
                      (lambda: lib.sb_dequantize(None, 0, 4, None), "dtype")]:
        assert rc() == 1
        assert match in error(lib)


def operands(t=4, k=2, e=4, d=128, f=128):
    return (torch.zeros(t, d, dtype=torch.bfloat16), torch.zeros(t, k, dtype=torch.int64),
            torch.zeros(t, k, dtype=torch.bfloat16), torch.zeros(e, d, 2 * f, dtype=torch.bfloat16),
            torch.zeros(e, f, d, dtype=torch.bfloat16))


def test_cpu_tensors_are_refused() -> None:
    with pytest.raises(RuntimeError, match="same GPU"):
        moe.moe_forward_gated(*operands())
    with pytest.raises(RuntimeError, match="same GPU"):
        moe.moe_gated_train(*operands())
    p = torch.zeros(4)
    with pytest.raises(RuntimeError, match="step must be"):
        optim.adamw_step([p], [p], [p], [p], optim.new_step("cpu"), 1e-3)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.dequantize([optim.new_state(p, 8)[0]])
    with pytest.raises(ValueError, match="32 or 8"):
        optim.new_state(p, 16)
    with pytest.raises(ValueError, match="no parameters"):
        optim.AdamW([])


def test_states_have_their_shapes() -> None:
    m, v = optim.new_state(torch.zeros(3, 171), 8)
    assert m.codes.dtype == torch.int8 and v.codes.dtype == torch.uint8 and m.codes.shape == (3, 171)
    assert m.scales.shape == v.scales.shape == (3,) and m.scales.dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize(("change", "match"), [
    (lambda a: a.update(x=a["x"].float()), "bfloat16"),
    (lambda a: a.update(w1=a["w1"].transpose(0, 1).contiguous()), "must be"),
    (lambda a: a.update(w1=a["w1"][:, :, ::2]), "must be"),
    (lambda a: a.update(w2=a["w2"].transpose(1, 2)), "contiguous"),
    (lambda a: a.update(x=torch.cat([a["x"], a["x"]], 1)[:, :128]), "contiguous"),
    (lambda a: a.update(x=torch.zeros(4 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 128)), "aligned"),
    (lambda a: a.update(expert_weight=a["expert_weight"].double()), "expert_weight"),
    (lambda a: a.update(expert_weight=a["expert_weight"][:, :1]), "expert_idx"),
    (lambda a: a.update(expert_idx=a["expert_idx"].float()), "expert_idx"),
    (lambda a: a.update(expert_idx=a["expert_idx"].cpu()), "same GPU"),
    (lambda a: a.update(activation="relu"), "activation"),
    (lambda a: a.update(valid_tokens=torch.tensor([3], device="cuda")), "valid_tokens"),
    (lambda a: a.update(valid_tokens=torch.tensor([3], dtype=torch.int32)), "valid_tokens"),
])
def test_gated_operands_are_refused(change, match) -> None:
    names = ("x", "expert_idx", "expert_weight", "w1", "w2")
    args = dict(zip(names, (v.cuda() for v in operands())))
    change(args)
    for call in (moe.moe_forward_gated, moe.moe_gated_train):
        with pytest.raises(RuntimeError, match=match):
            call(**args)


@pytest.mark.gpu
def test_backward_refuses() -> None:
    args = [v.cuda() for v in operands()]
    _, saved = moe.moe_gated_train(*args)
    for grad in (torch.zeros(4, 128, device="cuda"), torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"),
                 torch.zeros(4, 128, dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError, match="grad_out"):
            moe.moe_gated_backward(saved, grad)
    other = moe.GatedSaved(*(getattr(saved, n) for n in ("x", "expert_weight", "w1", "w2", "activation",
                                                         "valid_tokens")), saved.kept[:-256])
    with pytest.raises(RuntimeError, match="saved is not"):
        moe.moe_gated_backward(other, torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.gpu
def test_adamw_operands_are_refused() -> None:
    p = torch.zeros(512, device="cuda")
    step = optim.new_step()
    m, v = optim.new_state(p)
    m8, v8 = optim.new_state(p, 8)
    bad = [
        (([p], [p[:5]], [m], [v], step, 0.1), "shape"),
        (([p], [p, p], [m], [v], step, 0.1), "one length"),
        (([p], [p.double()], [m], [v], step, 0.1), "bfloat16"),
        (([p[::2]], [p[::2]], [m[:256]], [v[:256]], step, 0.1), "contiguous"),
        (([p], [p], [m.bfloat16()], [v], step, 0.1), "float32 states"),
        (([p], [p], [m], [v8], step, 0.1), "one kind"),
        (([p], [p], [v8], [m8], step, 0.1), "codes"),
        (([p], [p], [optim.Quantized(m8.codes, m8.scales[:1])], [v8], step, 0.1), "scales"),
        (([p], [p], [m], [v], step[:1], 0.1), "step"),
        (([p], [p], [m], [v], step, torch.tensor([0.1])), "lr"),
    ]
    for args, match in bad:
        with pytest.raises(RuntimeError, match=match):
            optim.adamw_step(*args)
    with pytest.raises(RuntimeError, match="master"):
        optim.adamw_step([p], [p], [m], [v], step, 0.1, masters=[p.bfloat16()])
    assert step.tolist() == [0, 0]


def test_ctypes_sizes_match_the_header(lib) -> None:
    """The tables that the Python side packs: nine and five 64-bit words an entry."""
    class Entry(ctypes.Structure):
        _fields_ = [(f"p{i}", ctypes.c_void_p) for i in range(7)] + [("numel", ctypes.c_int64),
                                                                    ("param_dtype", ctypes.c_int32),
                                                                    ("grad_dtype", ctypes.c_int32)]

    assert ctypes.sizeof(Entry) == 9 * 8
