"""What the 4-bit experts' entry points refuse, on the CPU: by their C calls (before
anything is launched) and by their Python functions."""

import pytest
import torch

from sparsebench_amd import _lib, moe


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
    ((2049, 1, 4, 128, 128), "2048 copies"),
    ((1025, 2, 4, 128, 128), "2048 copies"),
    ((2**40, 2, 4, 128, 128), "2048 copies"),
    ((4, 2, 0, 128, 128), "num_experts"),
    ((4, 2, 1025, 128, 128), "num_experts"),
    ((4, 2, 4, 64, 128), "multiples of 128"),
    ((4, 2, 4, 128, 192), "multiples of 128"),
    ((4, 2, 4, 128, 0), "multiples of 128"),
    ((4, 2, 4, 2**21, 128), "multiples of 128, up to"),
])
def test_layer_refuses_sizes(lib, args, match) -> None:
    assert lib.sb_experts4_sizes(*args, None) == 1
    assert match in error(lib)
    p = 4096
    assert lib.sb_experts4_layer(p, p, 0, p, 0, p, p, p, p, p, 0, p, 1 << 30, *args, None, None) == 1
    assert match in error(lib)


def test_layer_refuses_operands(lib) -> None:
    def call(x=4096, idx=4096, gates=4096, gate=0, c1=4096, s1=4096, c2=4096, s2=4096, out=4096, act=0):
        return lib.sb_experts4_layer(x, idx, 0, gates, gate, c1, s1, c2, s2, out, act, 4096, 1 << 30, 4, 2, 4, 128, 128,
                                     None, None)

    for name in ("x", "idx", "gates", "c1", "s1", "c2", "s2", "out"):
        assert call(**{name: None}) == 1 and "null buffer" in error(lib)
    for name in ("x", "c1", "c2", "out"):
        assert call(**{name: 4104}) == 1 and "16-byte aligned" in error(lib)
    assert call(gate=3) == 1 and "gate dtype" in error(lib)
    assert call(act=2) == 1 and "activation" in error(lib)


@pytest.mark.parametrize(("args", "match"), [
    ((0, 32, 32), "multiples of 32"),
    ((1, 33, 32), "multiples of 32"),
    ((1, 32, 48), "multiples of 32"),
    ((1, 0, 32), "multiples of 32"),
    ((2**40, 32, 32), "multiples of 32"),
    ((1, 2**25, 32), "multiples of 32"),
])
def test_codes_refuse(lib, args, match) -> None:
    assert lib.sb_quantize4(4096, 0, 4096, 4096, *args, None) == 1 and match in error(lib)
    assert lib.sb_dequantize4(4096, 4096, 4096, *args, None) == 1 and match in error(lib)


def test_codes_refuse_operands(lib) -> None:
    assert lib.sb_quantize4(4096, 5, 4096, 4096, 1, 32, 32, None) == 1 and "dtype" in error(lib)
    assert lib.sb_quantize4(4096, 0, 4104, 4096, 1, 32, 32, None) == 1 and "aligned" in error(lib)
    assert lib.sb_dequantize4(4104, 4096, 4096, 1, 32, 32, None) == 1 and "aligned" in error(lib)
    for args in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert lib.sb_quantize4(args[0], 0, *args[1:], 1, 32, 32, None) == 1 and "null buffer" in error(lib)
        assert lib.sb_dequantize4(*args, 1, 32, 32, None) == 1 and "null buffer" in error(lib)


def test_python_calls_refuse_cpu_tensors() -> None:
    w = torch.zeros(1, 32, 32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        moe.quantize_experts(w)
    w4 = moe.Experts4(torch.zeros(1, 1, 1, 32, 16, dtype=torch.uint8), torch.zeros(1, 1, 1, 32, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="on one GPU"):
        moe.dequantize_experts(w4)
    with pytest.raises(RuntimeError, match="on one GPU"):
        moe.moe_forward_gated_4bit(torch.zeros(2, 128), torch.zeros(2, 2), torch.zeros(2, 2), w4, w4)


def gpu_operands():
    def codes(e, k, n):
        return moe.Experts4(torch.zeros(e, n // 32, k // 32, 32, 16, dtype=torch.uint8, device="cuda"),
                            torch.full((e, n // 32, k // 32, 32), 127, dtype=torch.uint8, device="cuda"))

    return {"x": torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"),
            "idx": torch.zeros(3, 2, dtype=torch.int32, device="cuda"), "gates": torch.zeros(3, 2, device="cuda"),
            "w1": codes(4, 128, 512), "w2": codes(4, 256, 128), "act": "silu", "valid": None}


@pytest.mark.gpu
@pytest.mark.parametrize(("change", "match"), [
    (lambda o: o.update(x=o["x"][:2]), r"x must be \[T, D\]"),
    (lambda o: o.update(x=o["x"][0]), r"x must be \[T, D\]"),
    (lambda o: o.update(x=o["x"].float()), "bfloat16"),
    (lambda o: o.update(x=torch.zeros(128, 3, dtype=torch.bfloat16, device="cuda").t()), "contiguous"),
    (lambda o: o.update(x=torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")), r"w1 of \[E, D, 2F\]"),
    (lambda o: o.update(w1=o["w2"]), r"w1 of \[E, D, 2F\]"),
    (lambda o: o.update(w2=moe.Experts4(o["w2"].codes[:3], o["w2"].scales[:3])), r"w1 of \[E, D, 2F\]"),
    (lambda o: o.update(w1=moe.Experts4(o["w1"].codes, o["w2"].scales)), "codes"),
    (lambda o: o.update(w1=moe.Experts4(o["w1"].codes.int(), o["w1"].scales)), "codes"),
    (lambda o: o.update(w1=moe.Experts4(o["w1"].codes.flip(0)[:, :, :, :, ::2], o["w1"].scales)), "codes"),
    (lambda o: o.update(w1=moe.Experts4(o["w1"].codes.transpose(0, 1).contiguous().transpose(0, 1), o["w1"].scales)),
     "contiguous"),
    (lambda o: o.update(idx=o["idx"].short()), "int32 or int64"),
    (lambda o: o.update(idx=o["idx"].cpu()), "same GPU"),
    (lambda o: o.update(gates=o["gates"].double()), "expert_weight must be"),
    (lambda o: o.update(gates=o["gates"][:, :1]), r"\[T, k\]"),
    (lambda o: o.update(gates=o["gates"][:, :0], idx=o["idx"][:, :0]), "k > 0"),
    (lambda o: o.update(act="relu"), "activation"),
    (lambda o: o.update(valid=torch.zeros(1, device="cuda")), "valid_tokens"),
    (lambda o: o.update(x=torch.zeros(1025, 128, dtype=torch.bfloat16, device="cuda"),
                        idx=torch.zeros(1025, 2, dtype=torch.int32, device="cuda"),
                        gates=torch.zeros(1025, 2, device="cuda")), "2048 copies"),
])
def test_python_layer_refuses(change, match) -> None:
    o = gpu_operands()
    change(o)
    with pytest.raises(RuntimeError, match=match):
        moe.moe_forward_gated_4bit(o["x"], o["idx"], o["gates"], o["w1"], o["w2"], o["act"], o["valid"])


@pytest.mark.gpu
def test_no_tokens_and_bad_weights() -> None:
    o = gpu_operands()
    out = moe.moe_forward_gated_4bit(o["x"][:0], o["idx"][:0], o["gates"][:0], o["w1"], o["w2"])
    assert out.shape == (0, 128)
    for w in (torch.zeros(1, 33, 32, device="cuda"), torch.zeros(32, 32, device="cuda"),
              torch.zeros(1, 32, 32, dtype=torch.int32, device="cuda"), torch.zeros(0, 32, 32, device="cuda")):
        with pytest.raises(RuntimeError, match="multiples of 32|must be an"):
            moe.quantize_experts(w)
