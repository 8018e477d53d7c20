"""The gated layer between its norms: the block's call against its parts, a training step
of it from the forward pass to the orthogonalised update, and the trained block served with
4-bit weights.

Tolerance of the training step, in each gradient's norm: between the operands and a gradient
lie at most 14 roundings to bf16 (the layer's input; H, G, U, y; the layer's output; the norm's
result; the gradients of the norm's operands, [dG | dU], w H, rows of dx, dx, its sum with the
residual's, and the result), each of relative size 2^-8 / sqrt(3) at most and independent.
Where a rounding passes the activation it may grow by the ratio of |g a'(g)| to |a(g)|, 1.6 in
quadratic mean over a normal distribution's g; 2 covers it: 2 sqrt(14 / 3) 2^-8 = 1.7%.
"""

import math

import pytest
import torch

from sparsebench_amd import moe, norm, optim
from tests.test_muon_gpu import check_weights, step_reference

pytestmark = pytest.mark.gpu

DEV = "cuda"
CHAIN = 2 * math.sqrt(14 / 3) * 2.0**-8


def block(t, d, f, e, k, seed=0):
    """x, w1, w2, the norms' weights, gate and next weight, the router's ids and weights."""
    g = torch.Generator().manual_seed(seed)

    def some(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g) * scale + shift).bfloat16().to(DEV)

    ids = torch.rand(t, e, generator=g).topk(k, dim=1).indices.to(DEV)
    weights = torch.softmax(torch.randn(t, k, generator=g), 1).to(DEV)
    return (some(t, d), some(e, d, 2 * f, scale=d**-0.5), some(e, f, d, scale=f**-0.5),
            [some(d, scale=0.2, shift=1.0) for _ in range(2)] + [some(d, scale=0.1, shift=0.5), some(d, shift=1.0)],
            (ids, weights))


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("t", [1, 3, 70, 300])
def test_the_call_is_its_parts(t, four) -> None:
    x, w1, w2, (wi, wo, gate, wn), routed = block(t, 256, 384, 6, 2, seed=t)
    if four:
        w1, w2 = moe.quantize_experts(w1), moe.quantize_experts(w2)
    layer = moe.moe_forward_gated_4bit if four else moe.moe_forward_gated
    seen = []

    def route(n):
        seen.append(n)
        return routed

    out, after = moe.moe_block_gated(x, route, w1, w2, wi, wo, gate, 0.5, wn, activation="gelu")
    n = norm.norm_in(x, wi)
    assert torch.equal(seen[0], n)
    want = norm.norm_out(layer(n, *routed, w1, w2, "gelu"), x, wo, gate, 0.5)
    assert torch.equal(out, want) and torch.equal(after, norm.norm_in(want, wn))
    # The next block takes its input as it comes.
    second = moe.moe_block_gated(out, route, w1, w2, normed=after, out_weight=wo)
    assert torch.equal(second, moe.moe_block_gated(out, route, w1, w2, wn, wo))
    plain = moe.moe_block_gated(x, route, w1, w2)
    assert torch.equal(plain, norm.norm_out(layer(norm.norm_in(x), *routed, w1, w2), x))


@pytest.mark.parametrize("four", [False, True])
def test_padded_batch(four) -> None:
    """Rows behind the last token: whatever they hold, the others keep their bits."""
    x, w1, w2, (wi, wo, gate, wn), (ids, weights) = block(90, 128, 256, 5, 2, seed=9)
    if four:
        w1, w2 = moe.quantize_experts(w1), moe.quantize_experts(w2)
    want = moe.moe_block_gated(x, lambda n: (ids, weights), w1, w2, wi, wo, gate, next_weight=wn)
    valid = torch.tensor([33], dtype=torch.int32, device=DEV)
    x[33:], ids[33:] = float("nan"), 4
    got = moe.moe_block_gated(x, lambda n: (ids, weights), w1, w2, wi, wo, gate, next_weight=wn, valid_tokens=valid)
    # An expert's copies are counted without the padding: other tiles, the same sums.
    for have, full in zip(got, want):
        assert torch.equal(have[:33], full[:33])


def test_refusals() -> None:
    x, w1, w2, (wi, _, _, _), routed = block(4, 128, 128, 2, 1)
    four = moe.quantize_experts(w1)
    with pytest.raises(ValueError, match="both of them"):
        moe.moe_block_gated(x, lambda n: routed, four, w2)
    with pytest.raises(ValueError, match="in_weight must be None"):
        moe.moe_block_gated(x, lambda n: routed, w1, w2, wi, normed=x)


def train(x, w1, w2, vectors, routed, a, b):
    """Gradients of sum(a out + b next): of x, w1, w2, the norms' vectors, the router's weights."""
    wi, wo, gate, wn = vectors
    n = norm.norm_in(x, wi)
    y, saved = moe.moe_gated_train(n, *routed, w1, w2)
    out, after = norm.norm_out(y, x, wo, gate, 0.5, next_weight=wn)
    after_layer = norm.norm_out_backward(a, y, wo, gate, 0.5, out=out, grad_next=b, next_weight=wn)
    layer = moe.moe_gated_backward(saved, after_layer.y)
    first = norm.norm_in_backward(layer.x, x, wi, grad_x=after_layer.x)
    return (out, after), [first.x, layer.w1, layer.w2, first.weight, after_layer.weight, after_layer.gate,
                          after_layer.next_weight, layer.expert_weight]


def formula(x, w1, w2, vectors, routed, a, b):
    """The same in 64 bits, gradients by autograd, on the CPU."""
    ids = routed[0].cpu()
    leaves = [p.cpu().double().requires_grad_() for p in (x, w1, w2, *vectors, routed[1])]
    x, w1, w2, wi, wo, gate, wn, weights = leaves

    def n(v, w):
        return w * v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)

    h, y, f = n(x, wi), torch.zeros_like(x), w2.shape[1]
    for i in range(len(w2)):
        token, j = (ids == i).nonzero(as_tuple=True)
        g, u = (h[token] @ w1[i]).split(f, 1)
        y = y.index_add(0, token, weights[token, j][:, None] * ((torch.nn.functional.silu(g) * u) @ w2[i]))
    out = x + 0.5 * gate * n(y, wo)
    after = n(out, wn)
    ((a.cpu().double() * out).sum() + (b.cpu().double() * after).sum()).backward()
    return (out, after), [p.grad for p in leaves]


@pytest.mark.parametrize("t", [1, 70, 513])
def test_training_step(t) -> None:
    x, w1, w2, vectors, routed = block(t, 256, 384, 6, 2, seed=t + 100)
    a, b = (torch.randn(t, 256, generator=torch.Generator().manual_seed(s)).bfloat16().to(DEV) for s in (1, 2))
    outs, grads = train(x, w1, w2, vectors, routed, a, b)
    want_outs, want = formula(x, w1, w2, vectors, routed, a, b)
    for have, exact in zip([*outs, *grads], [*want_outs, *want]):
        exact = exact.to(DEV)
        assert have.shape == exact.shape
        assert (have.double() - exact).norm() <= CHAIN * exact.norm(), ((have.double() - exact).norm() / exact.norm()).item()


def test_steps_in_a_graph_then_served() -> None:
    """Forward, backward and update, captured once and replayed on new data beside the same
    eager steps; the weights that come of it in 4 bits through the block."""
    t, d, f = 70, 256, 384
    x, w1, w2, vectors, routed = block(t, d, f, 6, 2, seed=7)
    a, b = torch.empty_like(x), torch.empty_like(x)
    rate = torch.tensor([0.02], device=DEV)

    def trainer(w1, w2, vectors):
        views = [w1[..., :f], w1[..., f:], w2]
        muon = optim.Muon(views, lr=rate, weight_decay=0.1, master_weights=True)
        adam = optim.AdamW(vectors, lr=1e-3, master_weights=True)

        def step():
            _, (_, g1, g2, *others) = train(x, w1, w2, vectors, routed, a, b)
            muon.step([g1[..., :f], g1[..., f:], g2])
            adam.step(others[:4])
            return g1, g2

        return muon, step

    mine = [w1.clone(), w2.clone(), [v.clone() for v in vectors]]
    _, captured = trainer(w1, w2, vectors)
    muon, eager = trainer(*mine)
    a.normal_(), b.normal_()
    # The first calls, outside of the graph: workspaces.
    trainer(w1.clone(), w2.clone(), [v.clone() for v in vectors])[1]()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    for i in range(4):
        a.normal_(), b.normal_(), x.normal_(), rate.fill_(0.01 * (i + 1))
        graph.replay()
        before = [m.clone() for m in muon.masters], [m.clone() for m in muon.momenta]
        g1, g2 = eager()
        torch.cuda.synchronize()
        for have, same in zip([w1, w2, *vectors], [mine[0], mine[1], *mine[2]]):
            assert torch.equal(have, same)
        for j, g in enumerate((g1[..., :f], g1[..., f:], g2)):
            kept, update, _ = step_reference(before[0][j], g, before[1][j], 0.01 * (i + 1), 0.95, True, 0.1, 0.2, 1.0)
            check_weights(muon.masters[j], kept, update)

    four = moe.quantize_experts(w1), moe.quantize_experts(w2)
    wide = [moe.dequantize_experts(w) for w in four]
    wi, wo, gate, wn = vectors
    for rows in (1, 5, t):
        part = x[:rows].contiguous()
        route = tuple(r[:rows].contiguous() for r in routed)
        got = moe.moe_block_gated(part, lambda n: route, *four, wi, wo, gate, 0.5, wn)
        want = moe.moe_block_gated(part, lambda n: route, *wide, wi, wo, gate, 0.5, wn)
        # Both round H and the layer's output, the bf16 layer its copies' outputs too, then out.
        for have, other in zip(got, want):
            assert (have.double() - other.double()).norm() <= CHAIN * other.double().norm()
