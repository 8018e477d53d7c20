"""The AdamW step against 64 bits, value by value, with bounds from fp32
arithmetic (E = 2^-24 a rounding): coefficients, products and sums each add
one, the square root, division and reciprocal one or two. 8-bit codes have to
be the ones that the exact root falls on, for the same random bits, unless
the root lies within its own error of a border."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0**-24
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.95), 1e-8, 0.1
SIZES = [1, 7, 255, 256, 257, 2048, 5001]


def mix(h: np.ndarray) -> np.ndarray:
    h = h.astype(np.uint64) & 0xFFFFFFFF
    h ^= h >> 16
    h = h * 0x6A09E667 & 0xFFFFFFFF
    h ^= h >> 15
    h = h * 0xBB67AE85 & 0xFFFFFFFF
    return h ^ h >> 16


def random_bits(n: int, seed: int, step: int, tensor: int) -> torch.Tensor:
    key = mix(mix(np.array([step * 0x9E3779B9 + seed])) ^ np.uint64(tensor))
    i = np.arange(n, dtype=np.uint64)
    return torch.from_numpy(mix(i * np.uint64(0x9E3779B9) + key).astype(np.int64))


def tensors(sizes, dtype, seed, scale=1.0, offset=0):
    """Odd offsets: addresses that are multiples of the element alone."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        flat = (torch.randn(n + offset, generator=g) * scale).to(dtype).cuda()
        out.append(flat[offset:])
    return out


def quantized(values: torch.Tensor, signed: bool, offset=0):
    from sparsebench_amd import optim

    n, most = values.numel(), 127 if signed else 255
    b = torch.nn.functional.pad(values.abs().float(), (0, -n % 256)).view(-1, 256)
    scale = b.amax(1) / most**2
    root = torch.sqrt(b / torch.where(scale > 0, scale, 1)[:, None]).view(-1)[:n].round()
    codes = torch.where(values < 0, -root, root).to(torch.int8 if signed else torch.uint8)
    flat = torch.zeros(n + offset, dtype=codes.dtype, device=codes.device)
    flat[offset:] = codes
    return optim.Quantized(flat[offset:], scale)


def value64(q, root_only=False):
    c = q.codes.double().cpu()
    r = c * c.abs() * q.scales.double().cpu().repeat_interleave(256)[: c.numel()]
    return r if q.codes.dtype == torch.int8 or root_only else r * r


def check_step(sizes, p_type, g_type, bits, master, offset=0, seed=11, steps=1, scale=None, lr=LR):
    from sparsebench_amd import optim

    params, grads = tensors(sizes, p_type, 1, 0.5, offset), tensors(sizes, g_type, 2, 1e-2, offset)
    masters = [p.float().add_(1e-4) for p in params] if master else None
    m, v = tensors(sizes, torch.float32, 3, 3e-3, offset), tensors(sizes, torch.float32, 4, 1e-2, offset)
    v = [t.square_() for t in v]
    if bits == 8:
        m, v = [quantized(t, True, offset) for t in m], [quantized(t.sqrt(), False, offset) for t in v]
    step = torch.tensor([20, 0], dtype=torch.int32, device="cuda")
    for s in range(21, 21 + steps):
        before = []
        for i in range(len(sizes)):
            w = (masters[i] if master else params[i]).double().cpu()
            mv = (value64(m[i]), value64(v[i])) if bits == 8 else (m[i].double().cpu(), v[i].double().cpu())
            before.append((w, *mv))
        optim.adamw_step(params, grads, m, v, step, lr, BETAS, EPS, WD, masters, scale, seed)
        assert step.tolist() == [s, 0]
        lr_value, by = float(lr), 1.0 if scale is None else float(scale)
        for i, n in enumerate(sizes):
            w0, m0, v0 = before[i]
            g = grads[i].double().cpu() * by
            m1, v1 = BETAS[0] * m0 + (1 - BETAS[0]) * g, BETAS[1] * v0 + (1 - BETAS[1]) * g * g
            # Old 8-bit moments come out of fp32 products: two and three roundings more.
            m_b = (4 if bits == 32 else 6) * E * (BETAS[0] * m0.abs() + (1 - BETAS[0]) * g.abs()) + 1e-43
            v_b = (6 if bits == 32 else 10) * E * v1 + 1e-43
            size = lr_value / (1 - BETAS[0]**s)
            under = v1.sqrt() / (1 - BETAS[1]**s) ** 0.5 + EPS
            delta = size * m1 / under
            w1 = w0 * (1 - lr_value * WD) - delta
            w_b = 3 * E * w0.abs() + size * m_b / under + 16 * E * delta.abs() + 1e-30
            if master:
                got = masters[i].double().cpu()
                assert ((got - w1).abs() <= w_b).all()
                assert torch.equal(params[i].cpu(), masters[i].to(p_type).cpu())
            else:
                half = torch.finfo(p_type).eps / 2
                tiny = torch.finfo(p_type).smallest_normal * half
                got = params[i].double().cpu()
                assert ((got - w1).abs() <= w_b + half * (w1.abs() + w_b) + tiny).all()
            if bits == 32:
                assert ((m[i].double().cpu() - m1).abs() <= m_b).all()
                assert ((v[i].double().cpu() - v1).abs() <= v_b).all()
                continue
            rand = random_bits(n, seed, s, i)
            for q, exact, off, low16, most in ((m[i], m1.abs(), m_b, True, 127),
                                               (v[i], v1.sqrt(), v_b / v1.sqrt().clamp_min(1e-30), False, 255)):
                b = torch.nn.functional.pad(exact, (0, -n % 256)).view(-1, 256)
                ob = torch.nn.functional.pad(off, (0, -n % 256)).view(-1, 256)
                scale64 = b.amax(1) / most**2
                found = q.scales.double().cpu()
                assert ((found - scale64).abs() <= ob.amax(1) / most**2 + 8 * E * scale64).all()
                spread = found.repeat_interleave(256)[:n].clamp_min(1e-300)
                part = (rand & 0xFFFF if low16 else rand >> 16).double() / 65536
                low = ((exact - off).clamp_min(0) / spread).sqrt() * (1 - 4 * E) + part - 4 * E * most
                high = ((exact + off) / spread).sqrt() * (1 + 4 * E) + part + 4 * E * most
                low, high = low.floor().clamp(0, most), high.floor().clamp(0, most)
                if not low16:
                    low, high = (torch.where(exact > 0, t.clamp_min(1), t) for t in (low, high))
                codes = q.codes.double().cpu()
                assert ((codes.abs() >= low) & (codes.abs() <= high)).all()
                if low16:
                    sure = m1.abs() > m_b
                    assert (codes * m1 >= 0)[sure].all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize(("p_type", "g_type"), [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                                (torch.float16, torch.float16), (torch.float32, torch.float32),
                                                (torch.float32, torch.bfloat16)])
def test_matches_64_bits(p_type, g_type, bits, master) -> None:
    check_step(SIZES, p_type, g_type, bits, master, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_any_alignment(bits, offset) -> None:
    check_step(SIZES, torch.bfloat16, torch.float32, bits, True, offset=offset)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits) -> None:
    check_step([i * 37 % 700 + (i % 3 == 0) for i in range(101)], torch.float32, torch.float32, bits, False)


def test_more_values_than_workgroups_take_at_once() -> None:
    check_step([2048 * 8 * 256 + 12345, 3], torch.bfloat16, torch.bfloat16, 8, False)


def test_device_rate_and_gradient_scale() -> None:
    one = {"dtype": torch.float32, "device": "cuda"}
    check_step(SIZES, torch.float32, torch.float32, 32, False, lr=torch.tensor([LR], **one),
               scale=torch.tensor(0.25, **one))
    check_step(SIZES, torch.bfloat16, torch.bfloat16, 8, True, scale=0.5)


@pytest.mark.parametrize("sizes", [[], [0], [0, 5, 0]])
def test_empty_tensors_and_lists(sizes) -> None:
    check_step(sizes, torch.float32, torch.float32, 32, False)


def test_mixed_types_in_one_list() -> None:
    from sparsebench_amd import optim

    def run(order):
        a, b = tensors([300], torch.bfloat16, 1)[0], tensors([500], torch.float32, 2)[0]
        ga, gb = tensors([300], torch.bfloat16, 3)[0], tensors([500], torch.float32, 4)[0]
        step = optim.new_step()
        ps, gs = [(a, b)[i] for i in order], [(ga, gb)[i] for i in order]
        states = [optim.new_state(p) for p in ps]
        optim.adamw_step(ps, gs, [s[0] for s in states], [s[1] for s in states], step, LR)
        return a, b

    for x, y in zip(run([0, 1]), run([1, 0])):
        assert torch.equal(x, y)


def test_a_nan_takes_its_block_and_nothing_else() -> None:
    from sparsebench_amd import optim

    p = tensors([1024], torch.float32, 1)[0]
    states, step = optim.new_state(p, 8), optim.new_step()
    g = torch.ones_like(p)
    g[300] = float("nan")
    g[600] = float("inf")
    optim.adamw_step([p], [g], [states[0]], [states[1]], step, LR)
    values = optim.dequantize(states)
    for v in values:
        assert torch.isfinite(v[:256]).all() and torch.isfinite(v[768:]).all()
        assert not torch.isfinite(v[256:768]).any()


def test_small_changes_of_the_second_moment_are_kept() -> None:
    """sqrt(v) from 1 towards 0.5 at 1 - b2 = 0.001 for 1500 steps: rounded to
    nearest it would stay at 1 (a step's change is 0.04% of it, half a code 0.4%).
    exact: v = 0.25 + 0.75 b2^1500 = 0.417. At random the root's mean is exact to
    first order; what stays of its spread (a code is 0.8%, 65536 values) is far
    under the 10% allowed."""
    from sparsebench_amd import optim

    n = 65536
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    m = optim.new_state(p, 8)[0]
    g[::256] = 1.0  # holds each block's largest value at 1
    v = quantized(torch.ones(n, device="cuda"), False)
    step = optim.new_step()
    for _ in range(1500):
        optim.adamw_step([p], [g], [m], [v], step, 0.0, (0.9, 0.999))
    root = optim.dequantize([v])[0].view(-1, 256)[:, 1:]
    assert abs(float(root.mean()) - 0.417**0.5) < 0.1 * 0.417**0.5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequantize(dtype) -> None:
    from sparsebench_amd import optim

    states = []
    for i, n in enumerate([1, 255, 4096, 777, 0] * 15):
        values = tensors([n], torch.float32, i)[0] if n else torch.empty(0, device="cuda")
        states.append(quantized(values if i % 2 else values.abs(), bool(i % 2), offset=i % 4))
    for q, got in zip(states, optim.dequantize(states, dtype)):
        want = value64(q, root_only=True)
        half = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).smallest_normal * half
        assert got.dtype == dtype
        assert ((got.double().cpu() - want).abs() <= (half + 2 * E) * want.abs() * (1 + 4 * E) + tiny).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_with_their_own_counts(bits) -> None:
    """A replay takes the next step each time, with a learning rate set in between."""
    from sparsebench_amd import optim

    def fresh():
        ps = tensors(SIZES, torch.bfloat16, 1)
        opt = optim.AdamW(ps, torch.tensor([LR], device="cuda"), BETAS, EPS, WD, bits, True, seed=5)
        return opt, tensors(SIZES, torch.bfloat16, 2)

    opt, grads = fresh()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fresh()[0].step(grads)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step(grads)
    eager, eager_grads = fresh()
    for s in range(1, 5):
        for o in (opt, eager):
            o.lr.fill_(LR / s)
        for a, b in zip(grads, eager_grads):
            a.mul_(0.9)
            b.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        eager.step(eager_grads)
        assert opt.step_count.tolist() == [s, 0]
        for a, b in zip(opt.params + opt.masters, eager.params + eager.masters):
            assert torch.equal(a, b)


def test_a_training_step_of_a_gated_layer() -> None:
    """Forward, backward and update together, eager and captured: the same bits."""
    from sparsebench_amd import moe, optim
    from tests.test_gated_gpu import make

    def run(steps, captured):
        x, idx, gates, w1, w2, grad = (v.cuda() for v in make(100, 2, 4, 256, 256, seed=8))
        opt = optim.AdamW([w1, w2], LR, BETAS, EPS, WD, 8, True, seed=3)

        def step():
            out, saved = moe.moe_gated_train(x, idx, gates, w1, w2)
            g = moe.moe_gated_backward(saved, grad)
            opt.step([g.w1, g.w2])
            return out

        if captured:
            graph = torch.cuda.CUDAGraph()
            moe.moe_forward_gated(x, idx, gates, w1, w2)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                out = step()
            for _ in range(steps):
                graph.replay()
            torch.cuda.synchronize()
        else:
            for _ in range(steps):
                out = step()
        return out, w1, w2, *opt.masters, opt.exp_avgs[0].codes, opt.exp_avg_sqs[1].scales

    for a, b in zip(run(4, False), run(4, True)):
        assert torch.equal(a, b)


def test_masters_of_fp32_parameters_are_copies() -> None:
    from sparsebench_amd import optim

    p = tensors([600], torch.float32, 1)[0]
    g = tensors([600], torch.float32, 2)[0]
    q = p.clone()
    with_masters, without = optim.AdamW([p], LR, master_weights=True), optim.AdamW([q], LR)
    assert with_masters.masters[0].data_ptr() != p.data_ptr()
    for _ in range(2):
        with_masters.step([g])
        without.step([g])
    assert torch.equal(p, q) and torch.equal(with_masters.masters[0], p)


def test_more_values_than_32_bits_count() -> None:
    """Slices of a tensor of 2^31 + 4099 values against steps of copies of them:
    the same bits with fp32 states; with 8-bit ones the same scales, and codes
    that the random bits (of another position) put at most one apart."""
    from sparsebench_amd import optim

    n = 2**31 + 4099
    g = torch.Generator(device="cuda").manual_seed(7)
    grad = torch.randn(n, generator=g, device="cuda", dtype=torch.bfloat16)
    slices = [slice(0, 4096), slice(2**31 - 2048, 2**31 + 2048), slice(2**31, n)]
    for bits in (32, 8):
        p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
        states, step = optim.new_state(p, bits), optim.new_step()
        optim.adamw_step([p], [grad], [states[0]], [states[1]], step, LR, weight_decay=0.1)
        for s in slices:
            q = torch.ones_like(p[s])
            small = optim.new_state(q, bits)
            optim.adamw_step([q], [grad[s].clone()], [small[0]], [small[1]], optim.new_step(), LR, weight_decay=0.1)
            assert torch.equal(p[s], q)
            for big, little in zip(states, small):
                if bits == 32:
                    assert torch.equal(big[s], little)
                    continue
                blocks = slice(s.start // 256, -(-s.stop // 256))
                assert torch.equal(big.scales[blocks], little.scales)
                assert ((big.codes[s].int() - little.codes.int()).abs() <= 1).all()
        del p, states
