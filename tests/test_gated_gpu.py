"""The layer with gated experts and its gradients against 64 bits
(gated_reference.py: element-wise bounds and 2-norms derived from the
kernels' roundings)."""

import pytest
import torch

from tests.gated_reference import assert_close, gated_reference

pytestmark = pytest.mark.gpu

GATES = [torch.bfloat16, torch.float16, torch.float32]


def make(t, k, e, d, f, seed=0, gate_dtype=torch.bfloat16, ids="random", index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, d, generator=g).bfloat16()
    w1 = (torch.randn(e, d, 2 * f, generator=g) / d**0.5).bfloat16()
    w2 = (torch.randn(e, f, d, generator=g) / f**0.5).bfloat16()
    if ids == "random":
        idx = torch.rand(t, e, generator=g).topk(min(k, e), dim=-1).indices
        idx = torch.cat([idx, idx[:, : k - idx.shape[1]]], 1)
    elif ids == "one":  # every copy on the last expert: the same expert twice for a token too
        idx = torch.full((t, k), e - 1)
    else:  # "bad": some ids out of range, on both sides
        idx = torch.randint(-2, e + 2, (t, k), generator=g)
    gates = torch.softmax(torch.randn(t, k, generator=g), -1).to(gate_dtype)
    grad = torch.randn(t, d, generator=g).bfloat16()
    return x, idx.to(index), gates, w1, w2, grad


def check_all(args, act="silu", valid=None):
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = args
    t = x.shape[0] if valid is None else valid
    ref = gated_reference(x[:t], idx[:t], gates[:t], w1, w2, act, grad[:t])
    vt = None if valid is None else torch.tensor([valid], dtype=torch.int32, device="cuda")
    dev = [v.cuda() for v in (x, idx, gates, w1, w2)]
    out = moe.moe_forward_gated(*dev, act, vt)
    out_train, saved = moe.moe_gated_train(*dev, act, vt)
    grads = moe.moe_gated_backward(saved, grad.cuda())
    assert out.dtype == torch.bfloat16 and grads.expert_weight.dtype == gates.dtype
    assert_close("out", out[:t], ref)
    assert_close("out", out_train[:t], ref)
    assert_close("gates", grads.expert_weight[:t], ref)
    assert_close("x", grads.x[:t], ref)
    assert_close("w1", grads.w1, ref)
    assert_close("w2", grads.w2, ref)
    return out, grads


SHAPES = [(1, 1, 1, 128, 128), (1, 2, 8, 256, 512), (7, 3, 5, 128, 384), (250, 2, 8, 256, 512), (130, 1, 2, 384, 128),
          (300, 8, 16, 256, 256), (520, 3, 4, 512, 768), (513, 2, 3, 640, 256), (129, 4, 130, 128, 128), (1100, 2, 2, 256, 640)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_64_bits(shape, act) -> None:
    check_all(make(*shape, seed=sum(shape)), act)


# D and F that 256 do not divide, with enough row blocks for the chunk form:
# short and tall experts (chunks of 64 to 320 rows, several an expert).
EDGES = [(64, 2, 64, 640, 128), (40, 1, 70, 128, 896), (900, 3, 9, 384, 640), (2500, 2, 6, 896, 384)]


@pytest.mark.parametrize("shape", EDGES)
def test_half_slices(shape) -> None:
    check_all(make(*shape, seed=sum(shape)))


def test_chunk_lengths() -> None:
    """48 experts of up to three chunks: full, joined and short last pieces, one
    row, none; enough of them that every product runs in chunks, with half slices."""
    counts = torch.tensor([257, 320, 321, 64, 542, 1, 0, 255] * 6)
    x, _, gates, w1, w2, grad = make(int(counts.sum()), 1, 48, 640, 640, seed=11)
    idx = torch.repeat_interleave(torch.arange(48), counts)
    idx = idx[torch.randperm(len(idx), generator=torch.Generator().manual_seed(2))][:, None]
    check_all((x, idx, gates, w1, w2, grad), "gelu")


# Few tiles and a long reduction, split over workgroups: y = H W2 alone or dX
# too, in row blocks or chunks, D that 256 divide or not, several parts of
# unequal lengths, rows of one expert only.
SPLITS = [(18, 3, 3, 384, 6400, "random"), (5, 2, 4, 256, 2944, "random"), (700, 2, 3, 128, 1664, "random"),
          (2300, 8, 8, 256, 640, "random"), (2200, 8, 9, 128, 1280, "one"), (30, 2, 2, 256, 1152, "bad")]


@pytest.mark.parametrize("shape", SPLITS)
def test_split_reductions(shape) -> None:
    check_all(make(*shape[:5], seed=sum(shape[:5]), ids=shape[5]))


@pytest.mark.parametrize("gate_dtype", GATES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_gate_and_index_types(gate_dtype, index) -> None:
    check_all(make(77, 2, 6, 128, 256, gate_dtype=gate_dtype, index=index))


@pytest.mark.parametrize("ids", ["one", "bad"])
@pytest.mark.parametrize(("t", "k"), [(1, 1), (3, 2), (200, 2), (65, 17)])
def test_unusual_ids(ids, t, k) -> None:
    check_all(make(t, k, 4, 256, 128, ids=ids, seed=t))


def test_no_copy_routed_anywhere() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(20, 2, 4, 128, 128))
    idx.fill_(99)
    out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    grads = moe.moe_gated_backward(saved, grad)
    for v in (moe.moe_forward_gated(x, idx, gates, w1, w2), out, *grads):
        assert torch.all(v == 0)


@pytest.mark.parametrize("valid", [0, 1, 33, 64])
def test_valid_tokens(valid) -> None:
    check_all(make(64, 2, 4, 128, 256, seed=valid), valid=valid)


def test_rows_behind_the_valid_tokens_stay_as_they_were() -> None:
    """The allocator hands out the block that held a known pattern."""
    from sparsebench_amd import _C

    t, valid = 700, 300
    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(t, 2, 4, 256, 256))
    vt = torch.tensor([valid], dtype=torch.int32, device="cuda")
    ref = _C.gated_layer_cuda(x[:valid].clone(), idx[:valid], gates[:valid], w1, w2, "silu")
    pattern = torch.full_like(x, 7.0)
    size = _C.gated_bytes(t, 2, 4, 256, 256)[0]
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    from sparsebench_amd._lib import check, lib, stream_of

    check(lib().sb_gated_layer(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                               pattern.data_ptr(), 0, workspace.data_ptr(), size, t, 2, 4, 256, 256, vt.data_ptr(),
                               stream_of(x.device)))
    assert torch.all(pattern[valid:] == 7.0) and torch.equal(pattern[:valid], ref)


def test_gradient_against_differences() -> None:
    """<grad, direction> against the change of <grad_out, out> along it, in 64 bits
    (central differences of the definition), for each operand."""
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = make(40, 2, 4, 128, 128, seed=9, gate_dtype=torch.float32)
    _, saved = moe.moe_gated_train(*(v.cuda() for v in (x, idx, gates, w1, w2)))
    grads = moe.moe_gated_backward(saved, grad.cuda())
    operands = {"x": x.double(), "expert_weight": gates.double(), "w1": w1.double(), "w2": w2.double()}
    g = torch.Generator().manual_seed(3)
    for name, got in grads._asdict().items():
        direction = torch.randn(operands[name].shape, generator=g).double()

        def value(h):
            o = {n: v + h * direction if n == name else v for n, v in operands.items()}
            out = gated_reference(o["x"], idx, o["expert_weight"], o["w1"], o["w2"]).value["out"]
            return float((out * grad.double()).sum())

        h = 1e-4
        slope = (value(h) - value(-h)) / (2 * h)
        got = got.double().cpu()
        # The gradient's own error (2-norm, as in assert_close) along the direction.
        scale = float(got.norm()) * float(direction.norm()) * 2 * 2.0**-8 * 2**0.5 / got.numel()**0.5
        assert abs(float((got * direction).sum()) - slope) <= 4 * scale + 1e-6 * abs(slope)


def test_backward_may_run_twice_and_forward_forms_agree() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(333, 2, 8, 256, 256))
    out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    first = moe.moe_gated_backward(saved, grad)
    second = moe.moe_gated_backward(saved, grad)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    again, _ = moe.moe_gated_train(x, idx, gates, w1, w2)
    assert torch.equal(out, again)


def test_strided_ids_gates_and_gradient() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(50, 3, 5, 128, 128))
    wide_idx, wide_gates = idx.repeat_interleave(2, 1)[:, ::2], gates.repeat_interleave(2, 1)[:, ::2]
    one = grad[:1].expand(50, 128)
    out, saved = moe.moe_gated_train(x, wide_idx, wide_gates, w1, w2)
    grads = moe.moe_gated_backward(saved, one)
    want, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    assert torch.equal(out, want)
    for a, b in zip(grads, moe.moe_gated_backward(saved, one.contiguous())):
        assert torch.equal(a, b)
    odd = torch.empty(50 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(50, 128).copy_(grad)
    for a, b in zip(moe.moe_gated_backward(saved, odd), moe.moe_gated_backward(saved, grad)):
        assert torch.equal(a, b)


def test_no_tokens() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, grad = (v.cuda() for v in make(3, 2, 4, 128, 128))
    out, saved = moe.moe_gated_train(x[:0], idx[:0], gates[:0], w1, w2)
    grads = moe.moe_gated_backward(saved, grad[:0])
    assert out.shape == (0, 128) and moe.moe_forward_gated(x[:0], idx[:0], gates[:0], w1, w2).shape == (0, 128)
    assert grads.x.shape == (0, 128) and grads.expert_weight.shape == (0, 2)
    assert torch.all(grads.w1 == 0) and torch.all(grads.w2 == 0)


def test_non_finite_values_stay_in_their_tokens() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, _ = (v.cuda() for v in make(64, 2, 4, 128, 128))
    clean = moe.moe_forward_gated(x, idx, gates, w1, w2)
    x[5, 3], x[40, 0] = float("nan"), float("inf")
    out = moe.moe_forward_gated(x, idx, gates, w1, w2)
    rest = [i for i in range(64) if i not in (5, 40)]
    assert torch.equal(out[rest], clean[rest]) and not torch.isfinite(out[[5, 40]].float()).any()


def test_captured_and_replayed_with_new_values() -> None:
    """Forward, forward and backward, and serving of one token, in graphs that
    share a memory pool, replayed with other inputs and eager work in between."""
    from sparsebench_amd import moe

    static = [v.cuda() for v in make(120, 2, 6, 256, 256, seed=1)]
    x, idx, gates, w1, w2, grad = static
    one = [x[:1].clone(), idx[:1].clone(), gates[:1].clone()]

    def step():
        out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
        return (out, *moe.moe_gated_backward(saved, grad), moe.moe_forward_gated(x, idx, gates, w1, w2, "gelu"),
                moe.moe_forward_gated(*one, w1, w2))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (2, 3, 4):
        for a, b in zip(static, make(120, 2, 6, 256, 256, seed=seed)):
            a.copy_(b)
        for a, b in zip(one, (x, idx, gates)):
            a.copy_(b[seed:seed + 1])
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed


def test_two_streams_at_once() -> None:
    from sparsebench_amd import moe

    sets = [[v.cuda() for v in make(400, 2, 8, 256, 256, seed=s)] for s in (5, 6)]

    def step(args):
        out, saved = moe.moe_gated_train(*args[:5])
        return (out, *moe.moe_gated_backward(saved, args[5]))

    want = [step(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, (s, a) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(step(a))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(r, w))


@pytest.mark.parametrize("shape", [(30, 2, 2, 256, 1152), (18, 3, 3, 384, 6400), (2, 2, 4, 256, 512)])
def test_two_graphs_of_one_pool(shape) -> None:
    """Split reductions and two tokens, forward and backward in one graph and
    serving in another of the same pool, replayed in turn with other inputs."""
    from sparsebench_amd import moe

    static = [v.cuda() for v in make(*shape, seed=1)]

    def train():
        out, saved = moe.moe_gated_train(*static[:5])
        return (out, *moe.moe_gated_backward(saved, static[5]))

    def serve():
        return (moe.moe_forward_gated(*static[:5]),)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train(), serve()
    torch.cuda.synchronize()
    graphs, captured = [], []
    for step in (train, serve):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            captured.append(step())
    for seed in (2, 3, 4):
        for a, b in zip(static, make(*shape, seed=seed)):
            a.copy_(b)
        for graph, step, got in zip(graphs, (train, serve), captured):
            graph.replay()
            torch.cuda.synchronize()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (seed, step)


# ---- one or two tokens -------------------------------------------------

# (T, k, E, D, F, ids): copies of one expert or spread, up to the 64 that run
# without a routing layout and one past them; sums by the last workgroup (up to
# 32 of them) and by a launch of their own; F in several ranges of 2048 a workgroup.
FEW = [(1, 1, 1, 128, 128, "one"), (1, 64, 4, 128, 256, "bad"), (1, 65, 4, 128, 256, "bad"), (2, 32, 3, 128, 128, "one"),
       (2, 33, 3, 128, 128, "bad"), (2, 17, 4, 256, 384, "bad"), (1, 2, 8, 2048, 256, "random"),
       (2, 1, 2, 128, 4352, "random"), (1, 64, 3, 1024, 2304, "one"), (2, 16, 16, 384, 640, "random")]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape", FEW)
def test_one_or_two_tokens(shape, act) -> None:
    check_all(make(*shape[:5], seed=sum(shape[:5]), ids=shape[5]), act)


@pytest.mark.parametrize("gate_dtype", GATES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_one_or_two_tokens_gate_and_index_types(gate_dtype, index) -> None:
    check_all(make(2, 2, 6, 128, 256, gate_dtype=gate_dtype, index=index))


@pytest.mark.parametrize("d", [128, 2048])
@pytest.mark.parametrize("valid", [0, 1, 2, 3])
def test_two_tokens_valid_ones(valid, d) -> None:
    from sparsebench_amd import _C
    from sparsebench_amd._lib import check, lib, stream_of

    args = make(2, 3, 4, d, 256, seed=valid)
    check_all(args, valid=min(valid, 2))
    x, idx, gates, w1, w2, _ = (v.cuda() for v in args)
    whole = _C.gated_layer_cuda(x, idx, gates, w1, w2, "silu")
    vt = torch.tensor([valid], dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 7.0)
    size = _C.gated_bytes(2, 3, 4, d, 256)[0]
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    check(lib().sb_gated_layer(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                               out.data_ptr(), 0, workspace.data_ptr(), size, 2, 3, 4, d, 256, vt.data_ptr(),
                               stream_of(x.device)))
    assert torch.all(out[valid:] == 7.0) and torch.equal(out[:valid], whole[:valid])


def test_two_tokens_non_finite_values_stay_in_theirs() -> None:
    from sparsebench_amd import moe

    x, idx, gates, w1, w2, _ = (v.cuda() for v in make(2, 2, 2, 256, 128))
    clean = moe.moe_forward_gated(x, idx, gates, w1, w2)
    x[0, 3] = float("nan")
    out = moe.moe_forward_gated(x, idx, gates, w1, w2)
    assert torch.equal(out[1], clean[1]) and torch.isnan(out[0].float()).all()


# ---- sizes past the kernels' windows ------------------------------------


def relative(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.float() - b.float()).norm() / b.float().norm())


# Two runs of the same values, each with bf16 roundings (u = 2^-8 at most) of
# its own: of H or wH, G, U, dG | dU, y or a row of dX, and the result, fewer
# than 6 in a chain; the 2-norm of their difference is 2 * 6 u at the very most.
TWO_RUNS = 12 * 2.0**-8


def test_many_experts_without_rows() -> None:
    """1024 experts of 44 gradient tiles each, more than 128 of them a CU, 30
    experts with rows: against the layer of those 30."""
    from sparsebench_amd import moe

    t, k, e, d, f, few = 400, 2, 1024, 896, 896, 30
    x, idx, gates, v1, v2, grad = (v.cuda() for v in make(t, k, few, d, f, seed=4))
    w1, w2 = torch.zeros(e, d, 2 * f, dtype=x.dtype, device="cuda"), torch.zeros(e, f, d, dtype=x.dtype, device="cuda")
    at = torch.arange(few, device="cuda") * 35 + 1
    w1[at], w2[at] = v1, v2
    out, saved = moe.moe_gated_train(x, at[idx], gates, w1, w2)
    grads = moe.moe_gated_backward(saved, grad)
    want, want_saved = moe.moe_gated_train(x, idx, gates, v1, v2)
    want_grads = moe.moe_gated_backward(want_saved, grad)
    assert relative(out, want) <= TWO_RUNS and relative(grads.x, want_grads.x) <= TWO_RUNS
    assert relative(grads.expert_weight, want_grads.expert_weight) <= TWO_RUNS
    for got, ref in ((grads.w1, want_grads.w1), (grads.w2, want_grads.w2)):
        for i in range(few):
            assert relative(got[at[i]], ref[i]) <= TWO_RUNS
        got[at] = 0
        assert not got.any()


def test_x_of_more_than_two_gigabytes() -> None:
    """Each token's results against those of a layer of a few of the tokens, and
    the weights' gradients against the sum of two halves'."""
    from sparsebench_amd import moe

    t, d, f, e = 270_000, 4096, 128, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(t, d, generator=g, device="cuda", dtype=torch.bfloat16)
    grad = torch.randn(t, d, generator=g, device="cuda", dtype=torch.bfloat16)
    idx = torch.randint(0, e, (t, 1), generator=g, device="cuda")
    gates = torch.rand(t, 1, generator=g, device="cuda") + 0.5
    w1 = (torch.randn(e, d, 2 * f, generator=g, device="cuda") / d**0.5).bfloat16()
    w2 = (torch.randn(e, f, d, generator=g, device="cuda") / f**0.5).bfloat16()
    some = torch.cat([torch.arange(50), torch.arange(262_100, 262_200), torch.arange(t - 50, t)]).cuda()
    served = moe.moe_forward_gated(x, idx, gates, w1, w2)
    out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
    grads = moe.moe_gated_backward(saved, grad)
    ref = gated_reference(*(v[some].cpu() for v in (x, idx, gates)), w1.cpu(), w2.cpu(), "silu", grad[some].cpu())
    assert_close("out", served[some], ref)
    assert_close("out", out[some], ref)
    assert_close("x", grads.x[some], ref)
    assert_close("gates", grads.expert_weight[some], ref)
    sums = [torch.zeros_like(w, dtype=torch.float32) for w in (w1, w2)]
    for half in (slice(0, t // 2), slice(t // 2, t)):
        _, saved = moe.moe_gated_train(x[half], idx[half], gates[half], w1, w2)
        part = moe.moe_gated_backward(saved, grad[half])
        for total, p in zip(sums, (part.w1, part.w2)):
            total += p.float()
    assert relative(grads.w1, sums[0]) <= TWO_RUNS and relative(grads.w2, sums[1]) <= TWO_RUNS
