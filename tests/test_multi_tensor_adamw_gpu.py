"""mluOpMultiTensorAdamW on the GPU against the formula in 64 bits.

Tolerances.  u = 2^-24 is half a step of float.  With M = |b1 m| + |(1 - b1) g|: the new first
moment is two products of rounded constants and a sum, off by at most 4 u M; the second, of
positive terms, by 6 u v; its root by 4 u of itself.  The update step_size * m / (root * scale +
eps) has 4 u from the root, one rounding each for the product, the sum, the quotient, the
product with step_size and the two constants: 10 u of itself, and 4 u M / denominator *
step_size from m.  The parameter adds 3 u |p| (constant, product, difference) and its storage
type's half step.  8 bits: half a step of e4m3 is 2^-4 of the value, 2^-10 of the scale below
the normal range; a root raised to the smallest code is off by at most 2^-9 of the scale; the
scale itself by 2 u and by what the block's largest value is off.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# float16 values below 2^-14 lie 2^-24 apart whatever their size: half a step is 2^-25 there, more than 2^-11 of
# the value.
TINY = {torch.float32: 1e-40, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SIZES = [1, 255, 256, 257, 4095, 4096, 4097, 0, 12288, 100003]


def make(sizes, dtype, grad_dtype, bits, seed, misalign=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def place(values, dt):
        if misalign == 0:
            return values.to(dt)
        raw = torch.zeros(values.numel() + misalign, dtype=dt, device="cuda")
        raw[misalign:] = values.to(dt)
        return raw[misalign:]

    def normal(n, scale):
        return torch.randn(n, generator=gen, device="cuda") * scale

    p = [place(normal(n, 0.1), dtype) for n in sizes]
    g = [place(normal(n, 1e-2), grad_dtype) for n in sizes]
    m = [normal(n, 1e-3) for n in sizes]
    v = [normal(n, 5e-3).square() for n in sizes]
    if bits == 32:
        return p, g, [place(x, torch.float32) for x in m], [place(x, torch.float32) for x in v], [], []
    out = ([], [])
    scales = ([], [])
    for k, tensors in enumerate((m, [x.sqrt() for x in v])):
        for x in tensors:
            blocks = -(-x.numel() // 256)
            padded = torch.zeros(blocks * 256, device="cuda")
            padded[:x.numel()] = x
            s = padded.view(-1, 256).abs().amax(1) / 448.0
            codes = (padded.view(-1, 256) / s[:, None]).to(torch.float8_e4m3fn).view(-1)[:x.numel()]
            raw = torch.zeros(x.numel() + misalign, dtype=torch.uint8, device="cuda")
            raw[misalign:] = codes.view(torch.uint8)
            out[k].append(raw[misalign:])
            scales[k].append(s)
    return p, g, out[0], out[1], scales[0], scales[1]


def decode(codes, scales):
    n = codes.numel()
    return codes.view(torch.float8_e4m3fn).double() * scales.double().repeat_interleave(256)[:n]


def reference(p, g, m, v, lr, betas, eps, wd, step, gs):
    b1, b2 = betas
    g = g.double() * gs
    M = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = v.sqrt() / (1 - b2 ** step) ** 0.5 + eps
    size = lr / (1 - b1 ** step)
    update = size * m / denom
    new = p.double() * (1 - lr * wd) - update
    tol = 10 * U * update.abs() + size * 4 * U * M / denom + 3 * U * p.double().abs() + U * g.abs() * size / denom
    return new, m, v, tol, 5 * U * M, 8 * U * v


def assert_within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d elements off, worst %.3g of the tolerance" % (
        what, int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()))


def check_step(ops, handle, sizes, dtype, grad_dtype, bits, seed, misalign=0, gs=None, step=7, lr=2e-3, wd=0.1,
               betas=(0.9, 0.99), eps=1e-8, schedule=False):
    p, g, m, v, ms, vs = make(sizes, dtype, grad_dtype, bits, seed, misalign)
    before = [[t.clone() for t in x] for x in (p, g, m, v, ms, vs)]
    opt = ops.MultiTensorAdamW(p, m, v, *([ms, vs] if bits == 8 else []))
    scale = None if gs is None else torch.tensor([gs], device="cuda")
    gs64 = 1.0 if gs is None else float(scale.double())
    kw = {}
    if schedule:
        kw["schedule"] = torch.tensor([lr, 1 - betas[0] ** step, 1 - betas[1] ** step], device="cuda")
        opt.step(handle, g, 123.0, betas, eps, wd, 1, grad_scale=scale, **kw)
    else:
        opt.step(handle, g, lr, betas, eps, wd, step, grad_scale=scale)
    torch.cuda.synchronize()
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        p0, g0, m0, v0 = (before[k][i] for k in range(4))
        assert torch.equal(g[i], g0)
        if bits == 8:
            m0, v0 = decode(m0, before[4][i]), decode(v0, before[5][i]) ** 2
        new, m1, v1, tol, tm, tv = reference(p0, g0, m0.double(), v0.double(), lr, betas, eps, wd, step, gs64)
        if schedule:  # lr and the two corrections are floats there
            tol = tol + 3 * U * (new - p0.double()).abs() + U * p0.double().abs()
        assert_within(p[i], new, tol + HALF_STEP[dtype] * new.abs() + TINY[dtype], "param %d" % i)
        if bits == 32:
            assert_within(m[i], m1, tm + 1e-40, "exp_avg %d" % i)
            assert_within(v[i], v1, tv + 1e-40, "exp_avg_sq %d" % i)
            continue
        for codes, scales, want, slack, tiny in ((m[i], ms[i], m1, tm, 2.0 ** -10), (v[i], vs[i], v1.sqrt(), 8 * U * v1.sqrt(), 2.0 ** -9)):
            blocks = torch.zeros(-(-n // 256) * 256, dtype=torch.float64, device="cuda")
            blocks[:n] = want
            largest = blocks.view(-1, 256).abs().amax(1)
            off = torch.zeros_like(blocks)
            off[:n] = slack
            assert_within(scales, largest / 448.0, (4 * U * largest + off.view(-1, 256).amax(1)) / 448.0, "scale %d" % i)
            per = scales.double().repeat_interleave(256)[:n]
            got = decode(codes, scales)
            assert_within(got, want, torch.maximum(2.0 ** -4 * want.abs(), tiny * per) * 1.001 + slack, "state %d" % i)
            if tiny == 2.0 ** -9:
                assert (got[want > 0] > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                              (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                              (torch.float16, torch.float32)])
def test_one_step(ops, gpu_handle, dtype, grad_dtype, bits):
    check_step(ops, gpu_handle, SIZES, dtype, grad_dtype, bits, seed=1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("misalign", [1, 3])
def test_tensors_off_vector_alignment(ops, gpu_handle, bits, misalign):
    check_step(ops, gpu_handle, SIZES, torch.bfloat16, torch.bfloat16, bits, seed=2, misalign=misalign)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_take_several_launches(ops, gpu_handle, bits):
    check_step(ops, gpu_handle, [1 + (37 * i) % 700 for i in range(1100)], torch.float32, torch.float32, bits, seed=3)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_scale_and_schedule_on_the_device(ops, gpu_handle, bits):
    check_step(ops, gpu_handle, SIZES, torch.float32, torch.float32, bits, seed=4, gs=0.37)
    check_step(ops, gpu_handle, SIZES, torch.float32, torch.float32, bits, seed=4, gs=0.37, schedule=True)


@pytest.mark.parametrize("over", [dict(step=1), dict(step=1000000), dict(wd=0.0), dict(lr=0.0), dict(betas=(0.0, 0.0)),
                                  dict(eps=1e-3)])
def test_hyperparameters(ops, gpu_handle, over):
    check_step(ops, gpu_handle, [4096, 777], torch.float32, torch.float32, 32, seed=5, **over)
    check_step(ops, gpu_handle, [4096, 777], torch.float32, torch.float32, 8, seed=5, **over)


def test_vector_and_scalar_paths_agree_bit_for_bit(ops, gpu_handle):
    for bits in (32, 8):
        results = []
        for misalign in (0, 1):
            p, g, m, v, ms, vs = make([8192], torch.float32, torch.float32, bits, 6, misalign)
            ops.MultiTensorAdamW(p, m, v, *([ms, vs] if bits == 8 else [])).step(gpu_handle, g, 1e-3, step=3)
            results.append([t.clone() for t in p + m + v + ms + vs])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_zero_state_and_zero_gradient(ops, gpu_handle):
    n = 1000
    for bits in (32, 8):
        p = [torch.ones(n, device="cuda")]
        z = [[torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda")] for _ in range(2)]
        s = [[torch.zeros(4, device="cuda")] for _ in range(2)] if bits == 8 else []
        ops.MultiTensorAdamW(p, *z, *s).step(gpu_handle, [torch.zeros(n, device="cuda")], 0.5, weight_decay=0.5)
        assert torch.equal(p[0], torch.full((n,), 0.75, device="cuda"))
        assert not any(t[0].any() for t in z + s)


def test_nan_and_infinity_stay_where_they_belong(ops, gpu_handle):
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            p, g, m, v, ms, vs = make([2048], torch.float32, torch.float32, bits, 8)
            g[0][700] = bad
            ops.MultiTensorAdamW(p, m, v, *([ms, vs] if bits == 8 else [])).step(gpu_handle, g, 1e-3, step=2)
            wrong = ~torch.isfinite(p[0])
            assert wrong[700] and int(wrong.sum()) == 1
            values = (m[0], v[0]) if bits == 32 else (decode(m[0], ms[0]), decode(v[0], vs[0]))
            for x in values:
                wrong = ~torch.isfinite(x)
                assert wrong[700]
                wrong[512:768] = False  # 8 bits: the block of 256 it lies in
                assert not wrong.any()


def test_neighbouring_memory_is_left_alone(ops, gpu_handle):
    for bits in (32, 8):
        dt = torch.float32 if bits == 32 else torch.uint8
        raw = [torch.full((64 + 1003 + 64,), 3, dtype=d, device="cuda") for d in (torch.float32, dt, dt)]
        scales = [torch.full((64 + 4 + 64,), 3.0, device="cuda") for _ in range(2)] if bits == 8 else []
        inner = [[r[64:64 + 1003]] for r in raw] + [[s[64:68]] for s in scales]
        ops.MultiTensorAdamW(*inner).step(gpu_handle, [torch.ones(1003, device="cuda")], 1e-3)
        for r in raw + scales:
            assert (r[:64] == 3).all() and (r[-64:] == 3).all()


def test_captured_step_follows_gradient_and_schedule(ops, gpu_handle):
    for bits in (32, 8):
        p, g, m, v, ms, vs = make([5000, 300], torch.float32, torch.float32, bits, 9)
        q = [[t.clone() for t in x] for x in (p, m, v, ms, vs)]
        state = [ms, vs] if bits == 8 else []
        other = q[3:] if bits == 8 else []
        schedule = torch.zeros(3, device="cuda")
        captured, eager = ops.MultiTensorAdamW(p, m, v, *state), ops.MultiTensorAdamW(q[0], q[1], q[2], *other)
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
            captured.step(gpu_handle, g, 0.0, schedule=schedule)
        gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
        gen = torch.Generator(device="cuda").manual_seed(10)
        for step in range(1, 4):
            for t in g:
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
            schedule.copy_(torch.tensor([1e-3 * step, 1 - 0.9 ** step, 1 - 0.999 ** step]))
            graph.replay()
            eager.step(gpu_handle, g, 0.0, schedule=schedule)
        torch.cuda.synchronize()
        for a, b in zip([p, m, v, ms, vs], q):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_runs_on_the_handles_stream(ops):
    stream = torch.cuda.Stream()
    handle = ops.Handle(stream.cuda_stream)
    p, g, m, v, _, _ = make([100000], torch.float32, torch.float32, 32, 11)
    ref, _, ref_m, ref_v, _, _ = make([100000], torch.float32, torch.float32, 32, 11)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.MultiTensorAdamW(p, m, v).step(handle, g, 1e-3, step=2)
    torch.cuda.current_stream().wait_stream(stream)
    main = ops.Handle(torch.cuda.current_stream().cuda_stream)
    ops.MultiTensorAdamW(ref, ref_m, ref_v).step(main, g, 1e-3, step=2)
    assert torch.equal(p[0], ref[0]) and torch.equal(m[0], ref_m[0]) and torch.equal(v[0], ref_v[0])
    handle.destroy()
    main.destroy()


def test_trace_names_the_kernels(ops, gpu_handle, trace_kernels):
    for bits, name in ((32, "adamWKernel"), (8, "adamW8BitKernel")):
        p, g, m, v, ms, vs = make([5000], torch.float32, torch.float32, bits, 12)
        with trace_kernels() as names:
            ops.MultiTensorAdamW(p, m, v, *([ms, vs] if bits == 8 else [])).step(gpu_handle, g, 1e-3)
        assert names == [name]
