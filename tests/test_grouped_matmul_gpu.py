"""mluOpGroupedMatMul* on the GPU against the products in 64 bits.

Tolerance: a sum of K products of the stored values in float is off by at most K 2^-23 of the sum
of their magnitudes (a tensor core may cut a partial sum where a float addition would round it:
2^-23 instead of 2^-24 a step), and its storage by half a step of its type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}


def make(rows, ends, ci, co, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen, device="cuda").to(dtype)

    e = torch.tensor(ends, dtype=torch.int32, device="cuda")
    return normal(rows, ci), normal(len(ends), ci, co), normal(rows, co), e


def within(got, want, magnitude, k, what):
    tol = k * 2.0 ** -23 * magnitude + HALF_STEP[got.dtype] * want.abs() + TINY[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of the tolerance" % (
        what, int(bad.sum()), bad.numel(), float((off / tol.clamp(min=1e-300)).max()))


def clamped(ends, rows):
    out, top = [], 0
    for e in ends:
        top = max(top, min(max(e, 0), rows))
        out.append(top)
    return out


def check(ops, handle, rows, ends, ci, co, dtype, seed=0, weight_dtype=None):
    x, w, dy, e = make(rows, ends, ci, co, dtype, seed)
    y = ops.grouped_matmul_forward(handle, x, w, e)
    dx = ops.grouped_matmul_backward_input(handle, dy, w, e)
    dw = ops.grouped_matmul_backward_weight(handle, x, dy, e, dtype=weight_dtype)
    torch.cuda.synchronize()
    ends = clamped(ends, rows)
    for g, (a, b) in enumerate(zip([0] + ends[:-1], ends)):
        xg, wg, dg = x[a:b].double(), w[g].double(), dy[a:b].double()
        within(y[a:b], xg @ wg, xg.abs() @ wg.abs(), ci, "output of group %d" % g)
        within(dx[a:b], dg @ wg.T, dg.abs() @ wg.abs().T, co, "input gradient of group %d" % g)
        within(dw[g], xg.T @ dg, xg.abs().T @ dg.abs(), max(b - a, 1), "weight gradient of group %d" % g)
        if a == b:
            assert not dw[g].any()
    assert not y[ends[-1]:].any() and not dx[ends[-1]:].any()


@pytest.mark.parametrize("rows,ends", [(1, [1]), (5, [0, 5]), (128, [128]), (129, [128, 129]), (300, [7, 7, 200, 290]),
                                       (64, [0, 0, 0]), (1000, [1, 130, 131, 700, 1000])])
@pytest.mark.parametrize("ci,co", [(8, 8), (64, 64), (72, 136), (200, 328)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tensor_core_sizes(ops, gpu_handle, guard_bands, trace_kernels, rows, ends, ci, co, dtype):
    with trace_kernels() as names:
        check(ops, gpu_handle, rows, ends, ci, co, dtype, seed=1)
    assert {"groupedTcgen05Kernel:forward", "groupedTcgen05Kernel:input_grad", "groupedTcgen05Kernel:weight_grad"} <= set(names)


@pytest.mark.parametrize("rows,ends,ci,co", [(2600, [500, 501, 1100, 1800, 2590], 264, 1288),
                                             (2600, [513, 1025, 1500, 2100, 2600], 1288, 200),
                                             (20000, [19999], 64, 264), (9000, list(range(400, 8401, 400)), 264, 272),
                                             (3000, [i * 37 for i in range(80)], 136, 144), (4096, [4096], 512, 2048)])
def test_pairs_of_blocks(ops, gpu_handle, guard_bands, rows, ends, ci, co):
    """Sizes at which two blocks share a tile in at least one of the three products."""
    check(ops, gpu_handle, rows, ends, ci, co, torch.bfloat16, seed=2)


@pytest.mark.parametrize("rows,ends", [(1, [1]), (300, [7, 7, 200, 290]), (64, [0, 0]), (2000, [1999])])
@pytest.mark.parametrize("ci,co", [(1, 1), (3, 5), (16, 16), (64, 64), (37, 130), (132, 68)])
def test_general_kernel_float(ops, gpu_handle, guard_bands, rows, ends, ci, co):
    check(ops, gpu_handle, rows, ends, ci, co, torch.float32, seed=3)


@pytest.mark.parametrize("ci,co", [(1, 8), (12, 20), (37, 64), (130, 129)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_general_kernel_16_bits(ops, gpu_handle, guard_bands, trace_kernels, ci, co, dtype):
    with trace_kernels() as names:
        check(ops, gpu_handle, 700, [3, 300, 300, 690], ci, co, dtype, seed=4)
    assert set(names) <= {"groupedMatMulGeneralKernel", "groupedMatMulAddChunksKernel"}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,ends,ci,co", [(20000, [15000, 15001, 19990], 16, 24), (9000, [9000], 64, 64), (70000, [10, 69000], 32, 32)])
def test_long_groups_are_split(ops, gpu_handle, guard_bands, trace_kernels, dtype, rows, ends, ci, co):
    with trace_kernels() as names:
        check(ops, gpu_handle, rows, ends, ci, co, dtype, seed=5)
    assert "groupedMatMulAddChunksKernel" in names


def test_float_weight_gradient(ops, gpu_handle, guard_bands):
    for rows, ends, ci, co in ((500, [100, 480], 64, 72), (9000, [9000], 64, 64), (400, [400], 13, 7)):
        check(ops, gpu_handle, rows, ends, ci, co, torch.bfloat16, seed=6, weight_dtype=torch.float32)


def test_many_groups(ops, gpu_handle, guard_bands):
    for dtype, ci, co in ((torch.bfloat16, 32, 40), (torch.float32, 5, 6)):
        check(ops, gpu_handle, 5000, [int(4.7 * i) for i in range(1024)], ci, co, dtype, seed=7)


@pytest.mark.parametrize("ends", [[400, 100, 600], [-5, 2 ** 31 - 1, 7], [500, 0, 0], [-2 ** 31, -1, 0]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ends_are_clamped(ops, gpu_handle, guard_bands, ends, dtype):
    check(ops, gpu_handle, 500, ends, 64, 72, dtype, seed=8)


@pytest.mark.parametrize("dtype,ci,co", [(torch.float16, 64, 72), (torch.float16, 9, 10), (torch.float32, 64, 72)])
def test_other_rows_reach_nothing(ops, gpu_handle, dtype, ci, co):
    """NaN behind the last group and in another group change no other group's results."""
    x, w, dy, e = make(700, [100, 333, 600], ci, co, dtype, 9)
    clean = (ops.grouped_matmul_forward(gpu_handle, x, w, e), ops.grouped_matmul_backward_input(gpu_handle, dy, w, e),
             ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e))
    for t in (x, dy):
        t[600:] = float("nan")
        t[100:333] = float("nan")
    w[1] = float("inf")
    y, dx, dw = (ops.grouped_matmul_forward(gpu_handle, x, w, e), ops.grouped_matmul_backward_input(gpu_handle, dy, w, e),
                 ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e))
    for got, want in ((y, clean[0]), (dx, clean[1])):
        assert torch.equal(got[:100], want[:100]) and torch.equal(got[333:], want[333:]) and torch.isnan(got[100:333]).all()
    assert torch.equal(dw[0], clean[2][0]) and torch.equal(dw[2], clean[2][2]) and torch.isnan(dw[1]).all()


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_tensors_off_vector_alignment(ops, gpu_handle, which):
    for dtype in (torch.float16, torch.float32):
        x, w, dy, e = make(300, [100, 290], 64, 72, dtype, 10)

        def shifted(t):
            raw = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
            raw[1:] = t.reshape(-1)
            return raw[1:].view(t.shape)

        want = (ops.grouped_matmul_forward(gpu_handle, x, w, e), ops.grouped_matmul_backward_input(gpu_handle, dy, w, e),
                ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e))
        t = [shifted(v) if i == which else v for i, v in enumerate((x, w, dy))]
        outs = [shifted(v) if which == 3 else torch.empty_like(v) for v in want]
        ops.grouped_matmul_forward(gpu_handle, t[0], t[1], e, out=outs[0])
        ops.grouped_matmul_backward_input(gpu_handle, t[2], t[1], e, out=outs[1])
        ops.grouped_matmul_backward_weight(gpu_handle, t[0], t[2], e, out=outs[2])
        for got, ref in zip(outs, want):
            # two orders of at most 300 additions, and a half step each
            assert ((got.float() - ref.float()).abs() <= 300 * 2.0 ** -22 * 300 + 2 * HALF_STEP[dtype] * ref.float().abs()).all()


def test_products_are_each_others_adjoints(ops, gpu_handle):
    """<forward(x), dy> = <x, input gradient> = <w, weight gradient>, to the stored values' rounding."""
    x, w, dy, e = make(3000, [10, 1500, 2900], 128, 136, torch.bfloat16, 11)
    x[2900:], dy[2900:] = 0, 0
    y = ops.grouped_matmul_forward(gpu_handle, x, w, e).double()
    dx = ops.grouped_matmul_backward_input(gpu_handle, dy, w, e).double()
    dw = ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e).double()
    pairs = [(y, dy.double()), (dx, x.double()), (dw, w.double())]
    values = [(a * b).sum() for a, b in pairs]
    slack = [2.0 ** -8 * (a * b).abs().sum() for a, b in pairs]
    assert abs(values[0] - values[1]) <= slack[0] + slack[1] and abs(values[0] - values[2]) <= slack[0] + slack[2]


def test_captured_call_follows_the_group_ends(ops, gpu_handle):
    x, w, dy, e = make(3000, [10, 1500, 2900], 128, 136, torch.bfloat16, 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
        outs = (ops.grouped_matmul_forward(gpu_handle, x, w, e), ops.grouped_matmul_backward_input(gpu_handle, dy, w, e),
                ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e))
    gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
    for seed, ends in ((13, [3000, 3000, 3000]), (14, [0, 1, 2]), (15, [700, 1400, 2100])):
        x2, w2, dy2, e2 = make(3000, ends, 128, 136, torch.bfloat16, seed)
        for t, v in ((x, x2), (w, w2), (dy, dy2), (e, e2)):
            t.copy_(v)
        graph.replay()
        want = (ops.grouped_matmul_forward(gpu_handle, x2, w2, e2), ops.grouped_matmul_backward_input(gpu_handle, dy2, w2, e2),
                ops.grouped_matmul_backward_weight(gpu_handle, x2, dy2, e2))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_same_inputs_give_the_same_bits(ops, gpu_handle):
    x, w, dy, e = make(20000, [10, 15000, 19000], 64, 72, torch.float16, 16)
    runs = [(ops.grouped_matmul_forward(gpu_handle, x, w, e), ops.grouped_matmul_backward_input(gpu_handle, dy, w, e),
             ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e)) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_no_rows(ops, gpu_handle):
    e = torch.zeros(3, dtype=torch.int32, device="cuda")
    x, dy, w = (torch.zeros(s, dtype=torch.float16, device="cuda") for s in ((0, 16), (0, 24), (3, 16, 24)))
    assert ops.grouped_matmul_forward(gpu_handle, x, w, e).shape == (0, 24)
    assert ops.grouped_matmul_backward_input(gpu_handle, dy, w, e).shape == (0, 16)
    out = torch.full((3, 16, 24), 5.0, dtype=torch.float16, device="cuda")
    assert not ops.grouped_matmul_backward_weight(gpu_handle, x, dy, e, out=out).any()


@pytest.mark.parametrize("rows,ends,ci,co", [(300, [300], 1024, 64), (20000, [19999], 1024, 264)])
def test_bounded_wait_reports_an_error(ops, rows, ends, ci, co, monkeypatch):
    """A stage that is never released (more stages' worth of K than the ring holds) makes the loads' wait run out: the call
    reports it, nothing hangs, and the handle works afterwards."""
    handle = ops.Handle(torch.cuda.current_stream().cuda_stream)
    x, w, dy, e = make(rows, ends, ci, co, torch.float16, 17)
    monkeypatch.setenv("MLUOP_B200_TEST_GROUPED_WAIT", "2000000")
    with pytest.raises(ops.MluOpError):
        ops.grouped_matmul_forward(handle, x, w, e)
    monkeypatch.delenv("MLUOP_B200_TEST_GROUPED_WAIT")
    torch.cuda.synchronize()
    y = ops.grouped_matmul_forward(handle, x, w, e)
    within(y[:ends[0]], x[:ends[0]].double() @ w[0].double(), x[:ends[0]].double().abs() @ w[0].double().abs(), ci, "output")
    handle.destroy()
