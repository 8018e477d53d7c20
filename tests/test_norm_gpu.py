"""The norms before and after a block, forward and backward, against their
formulas in 64 bits, and the backward pass against differences.

Tolerances count roundings. Elementwise results are rounded once to their type:
half a step, eps / 2 relative. Before that everything is fp32: products of at
most 6 factors, and sums over a row that are short of D 2^-24 relative (the
adders work in parallel parts, so the factor is far smaller); 64 steps of 2^-24
cover them, relative to the sum of the terms' sizes, which the tests compute
beside the result. Sums over tokens likewise.
"""

import pytest
import torch

from sparsebench_amd import norm

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32_STEPS = 64 * 2.0**-24


def tensor(*shape, dtype=torch.float32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def check(got, want, size):
    """got: rounded once to its type; size: the sum of the sizes of the terms that made each value."""
    assert got.shape == want.shape
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + F32_STEPS * size.abs() + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs() - tol
    assert not (off > 0).any(), f"{(off > 0).sum()} of {off.numel()} off, worst by {off.max():.3g}"
    assert not got.isnan().any()


def forward(y, x, w, gate, scale, eps, v):
    """(out unrounded, its terms' sizes, next of the rounded out)."""
    y, x, d = y.double(), x.double(), x.shape[1]
    g = 1.0 if gate is None else gate.double()
    w = 1.0 if w is None else w.double()
    branch = scale * g * w * y / torch.sqrt((y * y).sum(1, keepdim=True) / d + eps)
    return x + branch, x.abs() + branch.abs()


def normed(o, v, eps):
    o = o.double()
    return v.double() * o / torch.sqrt((o * o).mean(1, keepdim=True) + eps)


GATES = {"none": lambda t, d: None, "channel": lambda t, d: (d,), "token": lambda t, d: (t, 1), "full": lambda t, d: (t, d)}
SHAPES = [(1, 1), (1, 1024), (3, 7), (5, 64), (4, 511), (2, 513), (9, 1024), (33, 1001), (6, 2048), (5, 2049), (3, 4096),
          (2, 4100), (2, 8192), (3, 10000), (1, 32768), (2, 32767), (5000, 48)]


def operands(t, d, gate, dtype, weights, seed=0):
    shape = GATES[gate](t, d)
    return (tensor(t, d, dtype=dtype, seed=seed, scale=2.0), tensor(t, d, dtype=dtype, seed=seed + 1),
            tensor(d, dtype=weights, seed=seed + 2, scale=0.3, shift=1.0),
            None if shape is None else tensor(*shape, dtype=weights, seed=seed + 3, scale=0.5, shift=0.5),
            tensor(d, dtype=weights, seed=seed + 4, scale=0.3, shift=1.0))


@pytest.mark.parametrize(("t", "d"), SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_in(t, d, dtype) -> None:
    x = tensor(t, d, dtype=dtype, seed=5, scale=3.0)
    w = tensor(d, seed=6, shift=1.0)
    want = normed(x, w, 1e-6)
    check(norm.norm_in(x, w), want, want)
    want = normed(x, torch.ones(d, device=DEV), 1e-3)
    check(norm.norm_in(x, eps=1e-3), want, want)


@pytest.mark.parametrize(("t", "d"), SHAPES)
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_out(t, d, gate, dtype) -> None:
    y, x, w, g, v = operands(t, d, gate, dtype, torch.bfloat16 if t % 2 else torch.float32)
    out, after = norm.norm_out(y, x, w, g, 0.25, 1e-5, next_weight=v)
    want, size = forward(y, x, w, g, 0.25, 1e-5, v)
    check(out, want, size)
    assert torch.equal(after, norm.norm_in(out, v, 1e-5))
    assert torch.equal(out, norm.norm_out(y, x, w, g, 0.25, 1e-5))
    want, size = forward(y, x, None, g, 1.0, 1e-6, v)
    check(norm.norm_out(y, x, gate=g), want, size)


def gradients(do, dn, y, out, w, g, scale, eps, v):
    """(dy, dx, dw, dg, dv), each with the sum of its terms' sizes, by the formulas in 64 bits."""
    do, y = do.double(), y.double()
    d = y.shape[1]
    wd = torch.ones(d, dtype=torch.float64, device=DEV) if w is None else w.double()
    gd = torch.ones(1, 1, dtype=torch.float64, device=DEV) if g is None else g.double()
    dx, dx_size, dv = do, do.abs(), None
    if dn is not None:
        o, dn, vd = out.double(), dn.double(), v.double()
        rn = 1 / torch.sqrt((o * o).mean(1, keepdim=True) + eps)
        on = o * rn
        dx = do + rn * (vd * dn - on * (vd * dn * on).mean(1, keepdim=True))
        dx_size = do.abs() + rn * ((vd * dn).abs() + on.abs() * (vd * dn * on).abs().mean(1, keepdim=True))
        dv = ((dn * on).sum(0), (dn * on).abs().sum(0))
    r = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    yn = y * r
    e, es = scale * gd * wd * dx, abs(scale) * gd.abs() * wd.abs() * dx_size
    dy = (r * (e - yn * (e * yn).mean(1, keepdim=True)), r * (es + yn.abs() * (es * yn.abs()).mean(1, keepdim=True)))
    p, ps = scale * yn * dx, abs(scale) * yn.abs() * dx_size
    dw = None if w is None else ((gd * p).sum(0), (gd.abs() * ps).sum(0))
    dg = None
    if g is not None:
        over = (lambda a: a.sum(0)) if g.dim() == 1 else (lambda a: a.sum(1, keepdim=True)) if g.shape[1] == 1 < d else (
            lambda a: a)
        dg = over(wd * p), over(wd.abs() * ps)
    return dy, (dx, dx_size), dw, dg, dv


@pytest.mark.parametrize(("t", "d"), SHAPES)
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_out_backward(t, d, gate, dtype) -> None:
    y, x, w, g, v = operands(t, d, gate, dtype, torch.float32 if t % 2 else torch.bfloat16, seed=20)
    do, dn = tensor(t, d, dtype=dtype, seed=30), tensor(t, d, dtype=dtype, seed=31)
    out, _ = norm.norm_out(y, x, w, g, 0.25, 1e-5, next_weight=v)
    got = norm.norm_out_backward(do, y, w, g, 0.25, 1e-5, out=out, grad_next=dn, next_weight=v)
    for have, want in zip(got, gradients(do, dn, y, out, w, g, 0.25, 1e-5, v)):
        assert (have is None) == (want is None)
        if have is not None:
            check(have, *want)
    alone = norm.norm_out_backward(do, y, None, g, 0.25, 1e-5)
    assert alone.x is do and alone.weight is None and alone.next_weight is None
    want = gradients(do, None, y, None, None, g, 0.25, 1e-5, None)
    check(alone.y, *want[0])
    if g is not None:
        check(alone.gate, *want[3])


@pytest.mark.parametrize(("t", "d"), SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_in_backward(t, d, dtype) -> None:
    x, dn, do = (tensor(t, d, dtype=dtype, seed=s) for s in (40, 41, 42))
    v = tensor(d, seed=43, shift=1.0)
    zero = torch.zeros_like(do)
    want = gradients(do, dn, zero, x, None, None, 1.0, 1e-5, v)
    got = norm.norm_in_backward(dn, x, v, 1e-5, grad_x=do)
    check(got.x, *want[1])
    check(got.weight, *want[4])
    want = gradients(zero, dn, zero, x, None, None, 1.0, 1e-5, torch.ones_like(v))
    got = norm.norm_in_backward(dn, x, eps=1e-5)
    check(got.x, *want[1])
    assert got.weight is None


def test_gradients_against_differences() -> None:
    """The directional derivative of a smooth function of (out, next), in 64 bits by the
    formulas' forward pass, against the gradients in fp32."""
    t, d, eps, scale = 6, 40, 1e-3, 0.5
    y, x, w, g, v = (a.double() for a in operands(t, d, "channel", torch.float32, torch.float32, seed=50))
    a, b = tensor(t, d, seed=60).double(), tensor(t, d, seed=61).double()

    def value(y, x, w, g, v):
        o, _ = forward(y, x, w, g, scale, eps, v)
        return (a * o).sum() + (b * normed(o, v, eps)).sum()

    args = [p.float() for p in (y, x, w, g, v)]
    out, _ = norm.norm_out(*args[:4], scale, eps, next_weight=args[4])
    grads = norm.norm_out_backward(a.float(), args[0], args[2], args[3], scale, eps, out=out, grad_next=b.float(),
                                   next_weight=args[4])
    for i, grad in enumerate(grads):  # y, x, weight, gate, next_weight, as the operands
        step = tensor(*grad.shape, seed=70 + i).double()
        h = 1e-5
        up, down = [y, x, w, g, v], [y, x, w, g, v]
        up[i], down[i] = up[i] + h * step, down[i] - h * step
        want = (value(*up) - value(*down)) / (2 * h)
        # Central differences are off by h^2 times third derivatives; the fp32 terms by 64 steps each.
        size = (grad.double() * step).abs().sum()
        assert abs((grad.double() * step).sum() - want) < 1e-4 * size


@pytest.mark.parametrize("d", [96, 1024, 2500])
def test_strides_and_offsets(d) -> None:
    """Rows inside wider rows, at addresses that no vector divides."""
    t = 7
    wide = tensor(4, t, d + 13, dtype=torch.bfloat16, seed=80)
    y, x, do, dn = (wide[i, :, 3:3 + d] for i in range(4))
    w = tensor(d + 1, dtype=torch.bfloat16, seed=81, shift=1.0)[1:]
    gate = tensor(t, d + 5, dtype=torch.bfloat16, seed=82)[:, 2:2 + d]
    out, after = norm.norm_out(y, x, w, gate, 0.5, next_weight=w)
    want, size = forward(y, x, w, gate, 0.5, 1e-6, w)
    check(out, want, size)
    check(after, normed(out, w, 1e-6), normed(out, w, 1e-6))
    got = norm.norm_out_backward(do, y, w, gate, 0.5, out=out, grad_next=dn, next_weight=w)
    for have, (want, size) in zip(got, gradients(do, dn, y, out, w, gate, 0.5, 1e-6, w)):
        check(have, want, size)
    one = x[:1].expand(t, d)  # a stride of 0
    assert torch.equal(norm.norm_in(one, w), norm.norm_in(x[:1], w).expand(t, d))
    tokens = gate[:, :1]
    want, size = forward(y, x, w, tokens, 0.5, 1e-6, w)
    check(norm.norm_out(y, x, w, tokens, 0.5), want, size)


@pytest.mark.parametrize("valid", [0, 1, 5, 9])
@pytest.mark.parametrize("d", [64, 1001])
def test_rows_behind_the_valid_tokens(d, valid) -> None:
    """They are neither read into sums nor written: a graph's later rows may hold anything."""
    t = 9
    y, x, w, g, v = operands(t, d, "channel", torch.float32, torch.float32)
    do, dn = tensor(t, d, seed=1), tensor(t, d, seed=2)
    limit = torch.tensor([valid], dtype=torch.int32, device=DEV)
    for a in (y, x, do, dn):
        a[valid:] = float("nan")
    torch.full((64, t, d), 7.0, device=DEV)  # what a new tensor's memory may hold
    out, after = norm.norm_out(y, x, w, g, 0.5, next_weight=v, valid_tokens=limit)
    want = norm.norm_out(y[:valid], x[:valid], w, g, 0.5, next_weight=v)
    assert torch.equal(out[:valid], want[0]) and torch.equal(after[:valid], want[1])
    out[valid:] = float("nan")
    got = norm.norm_out_backward(do, y, w, g, 0.5, out=out, grad_next=dn, next_weight=v, valid_tokens=limit)
    if valid:
        short = norm.norm_out_backward(do[:valid], y[:valid], w, g, 0.5, out=out[:valid], grad_next=dn[:valid],
                                       next_weight=v)
        assert torch.equal(got.y[:valid], short.y) and torch.equal(got.x[:valid], short.x)
        for a, b in zip(got[2:], short[2:]):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    else:
        assert not got.weight.any() and not got.gate.any() and not got.next_weight.any()


def test_no_tokens() -> None:
    y, w = torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV)
    out, after = norm.norm_out(y, y, w, w, next_weight=w)
    assert out.shape == after.shape == (0, 64)
    got = norm.norm_out_backward(y, y, w, w, out=out, grad_next=y, next_weight=w)
    assert got.y.shape == (0, 64) and not got.weight.any() and not got.gate.any() and not got.next_weight.any()


def test_zero_rows_infinities_and_nan() -> None:
    """A row of zeros gives zeros, and a row that is not finite does not leave its row."""
    x = tensor(4, 256, dtype=torch.bfloat16, seed=3)
    y = tensor(4, 256, dtype=torch.bfloat16, seed=4)
    y[1] = 0
    clean = norm.norm_out(y, x, next_weight=torch.ones(256, device=DEV))
    assert torch.equal(clean[0][1], x[1])
    y[2, 5], y[3, 7] = float("inf"), float("nan")
    out, after = norm.norm_out(y, x, next_weight=torch.ones(256, device=DEV))
    assert torch.equal(out[:2], clean[0][:2]) and torch.equal(after[:2], clean[1][:2])
    assert out[2].isnan()[5] and out[3].isnan().all() and after[2:].isnan().all()


def test_many_rows_beyond_32_bit_offsets() -> None:
    """2^31 values and more: the last rows are found."""
    t, d = 66_000, 32768
    x = torch.zeros(t, d, dtype=torch.bfloat16, device=DEV)
    x[-2:] = tensor(2, d, dtype=torch.bfloat16, seed=9)
    out = norm.norm_in(x)
    assert torch.equal(out[-2:], norm.norm_in(x[-2:])) and not out[:2].any() and not out[t // 2].any()


def test_same_bits_every_time_and_in_a_graph() -> None:
    t, d = 3000, 768
    y, x, w, g, v = operands(t, d, "channel", torch.bfloat16, torch.bfloat16)
    do, dn = tensor(t, d, dtype=torch.bfloat16, seed=1), tensor(t, d, dtype=torch.bfloat16, seed=2)

    def both():
        out, after = norm.norm_out(y, x, w, g, 0.5, next_weight=v)
        return out, after, *norm.norm_out_backward(do, y, w, g, 0.5, out=out, grad_next=dn, next_weight=v)

    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for seed in (3, 4, 5):
        y.copy_(tensor(t, d, dtype=torch.bfloat16, seed=seed))
        do.copy_(tensor(t, d, dtype=torch.bfloat16, seed=seed + 100))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, both()))
