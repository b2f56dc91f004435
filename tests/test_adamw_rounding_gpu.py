"""Stochastic rounding of 8-bit optimiser states on the GPU.

Bounds.  A code is one of the two values next to the exact quotient: the difference is below one step of e4m3 (2^-3 of
the lower value, 2^-9 below 2^-6) and the float error of the quotient (2^-22 of it).  The mean of S such codes is off by
at most half a step / sqrt(S) as standard deviation; the probabilities are multiples of 2^-16.  With 4,096 steps and
4,096 elements, six standard deviations are exceeded once in 10^5 runs.

Drift: a step moves the root by |d| = 0.0005 |g^2 / v - 1| of itself; rounding it stochastically adds a variance of
|d| * 0.125 of the root squared at most, 6e-5 on average for normal gradients (|g^2 / v - 1| has the mean 0.97), to the square, against which the
average pulls with 1e-3: the stored square settles at most 6 % above, the root 3 %.  The median over 4,096 elements
with a spread of 0.17 is off by 1.25 * 0.17 / 64 = 0.0033; four and a half of them: 1.5 %.  Together 4.5 %.
"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 256


def decode(codes, scales):
    return codes.view(torch.float8_e4m3fn).double() * scales.double().repeat_interleave(BLOCK)[:codes.numel()]


def make(sizes, dtype=torch.float32, seed=1, misalign=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def place(t):
        raw = torch.zeros(t.numel() + misalign, dtype=t.dtype, device="cuda")
        raw[misalign:] = t
        return raw[misalign:]

    p = [place((torch.randn(n, generator=gen, device="cuda") * 0.1).to(dtype)) for n in sizes]
    g = [place((torch.randn(n, generator=gen, device="cuda") * torch.randn(n, generator=gen, device="cuda").exp() * 1e-3).to(dtype))
         for n in sizes]
    codes = [[place(torch.randint(1, 127, (n,), generator=gen, device="cuda").to(torch.uint8)) for n in sizes] for _ in range(2)]
    scales = [[torch.rand(-(-n // BLOCK), generator=gen, device="cuda") * 1e-5 + 1e-6 for n in sizes] for _ in range(2)]
    return p, g, *codes, *scales


def copies(state):
    return [[t.clone() for t in x] for x in state]


def one(ops, handle, state, step=1, rounding="stochastic", **kw):
    p, g, m, v, ms, vs = state
    ops.MultiTensorAdamW(p, m, v, ms, vs).step(handle, g, 1e-3, step=step, rounding=rounding, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_codes_are_next_to_the_exact_values(ops, gpu_handle, dtype):
    sizes = [1, 255, 256, 257, 2047, 2048, 2049, 0, 100003]
    state = make(sizes, dtype)
    before, nearest = copies(state), copies(state)
    one(ops, gpu_handle, state, step=7)
    one(ops, gpu_handle, nearest, step=7, rounding="nearest")
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        # parameters and scales do not depend on the rounding
        assert torch.equal(state[0][i], nearest[0][i])
        assert torch.equal(state[4][i], nearest[4][i]) and torch.equal(state[5][i], nearest[5][i])
        g = before[1][i].double()
        m = 0.9 * decode(before[2][i], before[4][i]) + 0.1 * g
        root = (0.999 * decode(before[3][i], before[5][i]) ** 2 + 0.001 * g * g).sqrt()
        for codes, scales, want in ((state[2][i], state[4][i], m), (state[3][i], state[5][i], root)):
            per = scales.double().repeat_interleave(BLOCK)[:n]
            x = want / per
            off = (codes.view(torch.float8_e4m3fn).double() - x).abs()
            step = torch.maximum(2.0 ** -3 * x.abs(), torch.full_like(x, 2.0 ** -9))
            # (float: constants, products and the scale's two roundings; 16 of 2^-24, of the terms where they cancel)
            slack = 2.0 ** -20 * (x.abs() + (0.1 * g).abs() / per + 448)
            assert (off <= step + slack).all()
        assert (decode(state[3][i], state[5][i]) > 0).all()


def test_right_on_average_and_independent_between_steps(ops, gpu_handle):
    n, steps = 4096, 4096
    state = make([n])
    total, both, last = [torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2)], 0.0, None
    for step in range(1, steps + 1):
        now = copies(state)
        one(ops, gpu_handle, now, step=step)
        x = [now[2][0].view(torch.float8_e4m3fn).double(), now[3][0].view(torch.float8_e4m3fn).double()]
        for t, v in zip(total, x):
            t += v
    p, g, mc, vc, ms, vs = (t[0] for t in state)
    m = 0.9 * decode(mc, ms) + 0.1 * g.double()
    root = (0.999 * decode(vc, vs) ** 2 + 0.001 * g.double() ** 2).sqrt()
    for t, want, scales in zip(total, (m, root), (now[4][0], now[5][0])):
        x = want / scales.double().repeat_interleave(BLOCK)
        step = torch.maximum(torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -9))).clamp(min=-6) - 3), torch.tensor(2.0 ** -9, device="cuda"))
        low = torch.floor(x.abs() / step)
        f = x.abs() / step - low
        deviation = step * (f * (1 - f)).clamp(min=2.0 ** -16).sqrt() / steps ** 0.5
        raised = (x > 0) & (x < 2.0 ** -9) if want is root else torch.zeros_like(x, dtype=torch.bool)
        slack = 2.0 ** -16 * step + 2.0 ** -20 * (x.abs() + 0.1 * g.double().abs() / scales.double().repeat_interleave(BLOCK) + 448 * 2.0 ** -3)
        off = (t / steps - x).abs()
        assert ((off <= 6 * deviation + slack) | raised).all(), float((off / (6 * deviation + slack)).max())
        z = (t / steps - x)[~raised] / deviation[~raised]
        # spread of the means: independent choices from step to step (a choice that stayed would make it 64 times larger)
        keep = (f[~raised] > 0.05) & (f[~raised] < 0.95)
        spread = float(z[keep].square().mean())
        assert abs(spread - 1) <= 6 * (2.0 / int(keep.sum())) ** 0.5 + 0.02, spread


def test_paths_calls_and_devices_agree(ops, gpu_handle):
    """Aligned and misaligned tensors, one call or several, the step from the host or the device: the same codes."""
    sizes = [5000, 300, 2048]
    base = make(sizes)
    off = make(sizes, misalign=1)
    split = copies(base)
    counted = copies(base)
    one(ops, gpu_handle, base, step=3)
    one(ops, gpu_handle, off, step=3)
    for i in (2, 0, 1):
        one(ops, gpu_handle, [x[i:i + 1] for x in split], step=3)
    one(ops, gpu_handle, counted, step=3, step_count=torch.full((), 3, dtype=torch.int64, device="cuda"))
    for other in (off, split, counted):
        assert all(torch.equal(a, b) for x, y in zip(base, other) for a, b in zip(x, y))
    far = make(sizes)
    one(ops, gpu_handle, far, step=4)
    assert any(not torch.equal(a, b) for a, b in zip(base[2] + base[3], far[2] + far[3]))
    high, low = make(sizes), make(sizes)  # a step above 32 bits is another step
    one(ops, gpu_handle, high, step=3 + 2 ** 40, step_count=torch.full((), 3 + 2 ** 40, dtype=torch.int64, device="cuda"))
    one(ops, gpu_handle, low, step=3)
    assert any(not torch.equal(a, b) for a, b in zip(high[2] + high[3], low[2] + low[3]))


def test_captured_steps_choose_anew(ops, gpu_handle):
    state = make([5000])
    eager = copies(state)
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    schedule = torch.tensor([1e-3, 0.5, 0.5], device="cuda")
    opt, ref = [ops.MultiTensorAdamW(s[0], *s[2:]) for s in (state, eager)]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
        count += 1
        opt.step(gpu_handle, state[1], 0.0, schedule=schedule, rounding="stochastic", step_count=count)
    gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
    for step in range(1, 5):
        graph.replay()
        ref.step(gpu_handle, eager[1], 0.0, schedule=schedule, step=1, rounding="stochastic",
                 step_count=torch.full((), step, dtype=torch.int64, device="cuda"))
        assert all(torch.equal(a, b) for x, y in zip(state, eager) for a, b in zip(x, y))


def test_not_a_number_and_infinity_stay_in_their_block(ops, gpu_handle):
    for bad in (float("nan"), float("inf"), float("-inf")):
        for misalign in (0, 1):
            state = make([2048 + 300], misalign=misalign)
            state[1][0][700] = bad
            one(ops, gpu_handle, state, step=2)
            wrong = ~torch.isfinite(state[0][0])
            assert wrong[700] and int(wrong.sum()) == 1
            for x in (decode(state[2][0], state[4][0]), decode(state[3][0], state[5][0])):
                wrong = ~torch.isfinite(x)
                assert wrong[700]
                wrong[512:768] = False
                assert not wrong.any()


@pytest.mark.parametrize("factor", [4.0, 0.25])
def test_states_follow_gradients_that_change(pkg, factor):
    """4,000 steps of the optimiser; the gradients of every other element change by the factor after 1,000.  The stored
    roots of both halves of each block against float ones."""
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    n = 8192
    gen = torch.Generator(device="cuda").manual_seed(4)
    size = torch.exp(torch.randn(n, generator=gen, device="cuda")) * 1e-3
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.zeros(n, device="cuda")
    opt = nn_.AdamW([p], lr=1e-3, state_bits=8, weight_decay=0.0)
    v = torch.zeros(n, device="cuda")
    for step in range(4000):
        if step == 1000:
            size[::2] *= factor
        torch.randn(n, generator=gen, device="cuda", out=p.grad)
        p.grad.mul_(size)
        opt.step()
        v = v * 0.999 + 0.001 * p.grad.square()
    state = opt.state[p]
    ratio = decode(state["exp_avg_sq"], state["exp_avg_sq_scale"]) / v.double().sqrt()
    for half in (ratio[::2], ratio[1::2]):
        assert abs(float(half.median()) - 1) <= 0.045, float(half.median())


@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
@pytest.mark.parametrize("epsilon", [1e-30, 1e-39, 1e-42])
def test_small_epsilons(ops, gpu_handle, rounding, epsilon):
    """Elements without a gradient: 0 / epsilon = 0 for every epsilon that a float holds, denormal ones among them."""
    for misalign in (0, 1):
        state = make([2048 + 100], misalign=misalign)
        state[1][0].zero_()
        for t in state[2] + state[3] + state[4] + state[5]:
            t.zero_()
        before = state[0][0].clone()
        p, g, m, v, ms, vs = state
        ops.MultiTensorAdamW(p, m, v, ms, vs).step(gpu_handle, g, 1e-3, epsilon=epsilon, weight_decay=0.0, rounding=rounding)
        assert torch.equal(p[0], before)
