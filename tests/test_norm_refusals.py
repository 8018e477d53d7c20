"""What the norms' entry points refuse, on the CPU: by their C calls (before anything is
launched) and by their Python functions."""

import ctypes

import pytest
import torch

from sparsebench_amd import _lib, norm


@pytest.fixture(scope="module")
def lib():
    try:
        return _lib.lib()
    except _lib.LibraryNotBuilt as e:
        pytest.skip(str(e))


P = 4096  # an aligned address that is never read


def norm_in(lib, x=P, weight=None, wd=0, out=P, dtype=0, t=4, d=64, stride=64, eps=1e-6):
    return lib.sb_norm_in(x, stride, weight, wd, out, dtype, t, d, eps, None, None)


@pytest.mark.parametrize(("args", "match"), [
    ({"x": None}, "null buffer"),
    ({"out": None}, "null buffer"),
    ({"dtype": 3}, "unsupported dtype"),
    ({"wd": 7}, "unsupported dtype"),
    ({"d": 0}, "0 < D"),
    ({"d": 32769}, "0 < D"),
    ({"t": -1}, "0 <= T"),
    ({"t": 2**31}, "0 <= T"),
    ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"),
    ({"stride": -64}, "negative stride"),
])
def test_norm_in_refuses(lib, args, match) -> None:
    assert norm_in(lib, **args) == 1
    assert match in lib.sb_last_error().decode()


def norm_out(lib, y=P, x=P, out=P, gate=None, gd=0, kind=0, gate_stride=0, dtype=0, nd=0, t=4, d=64):
    return lib.sb_norm_out(y, d, x, d, None, 0, gate, gd, kind, gate_stride, 1.0, None, nd, out, None, dtype, t, d,
                           1e-6, None, None)


@pytest.mark.parametrize(("args", "match"), [
    ({"y": None}, "null buffer"),
    ({"x": None}, "null buffer"),
    ({"out": None}, "null buffer"),
    ({"kind": 4, "gate": P}, "gate kind"),
    ({"kind": -1, "gate": P}, "gate kind"),
    ({"kind": 1}, "gate kind"),
    ({"gd": 3}, "unsupported dtype"),
    ({"nd": 3}, "unsupported dtype"),
    ({"gate_stride": -1}, "negative stride"),
])
def test_norm_out_refuses(lib, args, match) -> None:
    assert norm_out(lib, **args) == 1
    assert match in lib.sb_last_error().decode()


def test_sizes_refuse(lib) -> None:
    size = ctypes.c_int64()
    for t, d in ((-1, 64), (4, 0), (4, 40000)):
        assert lib.sb_norm_sizes(t, d, ctypes.byref(size)) == 1
        assert "norm: 0 <= T" in lib.sb_last_error().decode()


def test_backward_refuses_null_buffers(lib) -> None:
    def out_backward(grad_out=P, grad_next=P, y=P, out=P, gate=None, kind=0, dy=P, dx=P, dgate=None):
        return lib.sb_norm_out_backward(grad_out, 64, grad_next, 64, y, 64, out, 64, None, 0, gate, 0, kind, 0, 1.0,
                                        None, 0, dy, dx, None, dgate, None, 0, 4, 64, 1e-6, None, P, 1 << 20, None)

    for args in ({"grad_out": None}, {"y": None}, {"out": None}, {"dy": None}, {"dx": None}):
        assert out_backward(**args) == 1 and "null buffer" in lib.sb_last_error().decode()
    assert out_backward(gate=P, kind=1) == 1 and "gate kind" in lib.sb_last_error().decode()  # no place for its gradient
    for grad, x, dx in ((None, P, P), (P, None, P), (P, P, None)):
        assert lib.sb_norm_in_backward(grad, 64, x, 64, None, 0, None, 0, dx, None, 0, 4, 64, 1e-6, None, P, 1 << 20,
                                       None) == 1
        assert "null buffer" in lib.sb_last_error().decode()


def test_python_calls_refuse_cpu_tensors() -> None:
    x = torch.zeros(4, 64)
    for call in (lambda: norm.norm_in(x), lambda: norm.norm_out(x, x), lambda: norm.norm_in_backward(x, x),
                 lambda: norm.norm_out_backward(x, x)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize(("make", "match"), [
    (lambda x, w: norm.norm_in(x[0]), r"\[T, D\]"),
    (lambda x, w: norm.norm_in(x.double()), "bfloat16, float16 or float32"),
    (lambda x, w: norm.norm_in(x.t()), "contiguous rows"),
    (lambda x, w: norm.norm_in(x[:, :0]), "1 to 32768"),
    (lambda x, w: norm.norm_in(x, w[:-1]), "weight must be"),
    (lambda x, w: norm.norm_in(x, w.cpu()), "weight must be"),
    (lambda x, w: norm.norm_in(x, w.int()), "weight must be"),
    (lambda x, w: norm.norm_in(x, eps=-1.0), "eps"),
    (lambda x, w: norm.norm_in(x, valid_tokens=torch.tensor([1])), "valid_tokens"),
    (lambda x, w: norm.norm_out(x, x[:2]), "y must be"),
    (lambda x, w: norm.norm_out(x.half(), x), "y must be"),
    (lambda x, w: norm.norm_out(x, x, gate=w[:3]), "gate must be"),
    (lambda x, w: norm.norm_out(x, x, gate=x.t()), "gate must be"),
    (lambda x, w: norm.norm_out(x, x, gate=w.int()), "gate must be"),
    (lambda x, w: norm.norm_out(x, x, next_weight=w[1:]), "next_weight must be"),
    (lambda x, w: norm.norm_out_backward(x, x, grad_next=x), "needs grad_next"),
    (lambda x, w: norm.norm_out_backward(x, x, next_weight=w), "needs grad_next"),
    (lambda x, w: norm.norm_out_backward(x, x, grad_next=x, next_weight=w), "needs grad_next"),
    (lambda x, w: norm.norm_out_backward(x[:1], x), "grad_out must be"),
    (lambda x, w: norm.norm_in_backward(x[:1], x), "grad must be"),
    (lambda x, w: norm.norm_in_backward(x, x, grad_x=x[:1]), "grad_x must be"),
])
def test_python_calls_refuse(make, match) -> None:
    with pytest.raises(RuntimeError, match=match):
        make(torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda"))


def test_both_import_paths() -> None:
    import sparsebench.norm

    assert sparsebench.norm is norm
