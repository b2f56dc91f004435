"""mluOpGroupNormActForward / Backward on the GPU against the formulas in 64 bits.

Tolerances, u = 2^-24 (half a step of float), sums of n values in float off by at most d u times
the sum of magnitudes, d the number of additions that one value passes through: a thread adds at
most 64 rows here and a block joins its threads in 8 levels: d = 72; the blocks' sums are joined in
double.  (Short samples: a thread adds at most 64 rows of 4 pairs.  Deviations are from the group's mean as float sums give
it, each rounded once: with A1 and A2 the group's mean deviation and variance, the mean and the variance are off by no more
than the terms below, d = 4 * 64 + 1.)  Statistics: with k the block's first row, deviations from it average at most |x - k|, whose
mean over a group is bounded by the test from the data (A1, and A2 for squares): the mean is off by
d u A1 + 2 u |mean|, the variance by 2 d u A2 + 4 u A2.  xhat = (x - mean) rstd then by
(d_mean + u |x| ) rstd + |xhat| (d_var / (2 var') + 4 u); y adds the two roundings of the affine
map, 8 u |u| and 16 u |y| for the exponential of silu (2 steps each for it, its sum and its quotient),
and the storage type's half step.  Gradients: given mean and rstd, each du xhat is off by at most 16 u of its magnitude
(silu; cancelling 1 + u (1 - s): bounded with |u|), sums by (d + 16) u of the magnitudes, and the
input gradient by the sum of its three terms' errors and a half step.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
D = 72
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}  # half a step below the normal range
EPS = 1e-5


def spans(x, ends):
    if ends is None:
        rows = x[0].numel() // x.shape[-1] if x.shape[0] else 0
        return [(i * rows, (i + 1) * rows) for i in range(x.shape[0])]
    e = ends.tolist()
    return list(zip([0] + e[:-1], e))


def act64(u, act):
    return u.clamp(min=0) if act == "relu" else u * torch.sigmoid(u) if act == "silu" else u


def act_grad64(u, act):
    if act == "relu":
        return (u > 0).double()
    if act == "silu":
        s = torch.sigmoid(u)
        return s * (1 + u * (1 - s))
    return torch.ones_like(u)


def make(shape, dtype, seed, offset=1.0, affine="float"):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    c = shape[-1]
    x = (normal(*shape) * (0.5 + torch.rand(c, generator=gen, device="cuda")) + offset * normal(c)).to(dtype)
    if affine is None:
        return x, None, None, normal(*shape).to(dtype)
    w, b = 1 + 0.2 * normal(c), 0.2 * normal(c)
    if affine == "same":
        w, b = w.to(dtype), b.to(dtype)
    return x, w, b, normal(*shape).to(dtype)


def within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of the tolerance" % (
        what, int(bad.sum()), bad.numel(), float((off / tol.clamp(min=1e-300)).max()))


def check(ops, handle, shape, groups, dtype, act, ends=None, seed=0, affine="float", offset=1.0, grad_dtype=None):
    x, w, b, dy = make(shape, dtype, seed, offset, affine)
    c = shape[-1]
    ends_t = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(handle, x, w, b, groups, EPS, act, ends_t)
    dx, dw, db = ops.group_norm_act_backward(handle, dy, x, w, b, mean, rstd, groups, act, ends_t,
                                             affine_grad_dtype=grad_dtype)
    torch.cuda.synchronize()
    rows = x.reshape(-1, c).double()
    g = dy.reshape(-1, c).double()
    w64 = torch.ones(c, dtype=torch.float64, device="cuda") if w is None else w.double()
    b64 = torch.zeros(c, dtype=torch.float64, device="cuda") if b is None else b.double()
    y2, dx2 = y.reshape(-1, c), dx.reshape(-1, c)
    sums = [torch.zeros(c, dtype=torch.float64, device="cuda") for _ in range(4)]  # dbeta, dgamma, and their error bounds
    last = 0
    per = c // groups
    for i, (lo, hi) in enumerate(spans(x, ends_t)):
        last = max(last, hi)
        if hi <= lo:
            assert (mean[i] == 0).all() and torch.allclose(rstd[i], torch.full_like(rstd[i], EPS ** -0.5))
            continue
        r = rows[lo:hi].view(hi - lo, groups, per)
        m = r.mean((0, 2))
        var = ((r - m[None, :, None]) ** 2).mean((0, 2))
        # the largest deviation from any row of the sample bounds the one from the block's first row
        spread = (r.amax(0) - r.amin(0))
        a1, a2 = spread.mean(1), (spread ** 2).mean(1)
        depth = D
        if ends is None and hi - lo <= 64:
            depth = 4 * (hi - lo) + 1
            a1, a2 = (r - m[None, :, None]).abs().mean((0, 2)), var
        d_mean = depth * U * a1 + 4 * U * m.abs() + 1e-38
        d_var = 2 * (depth + 4) * U * a2
        within(mean[i], m, d_mean, "mean")
        want_r = (var + EPS) ** -0.5
        within(rstd[i], want_r, want_r * (d_var / (2 * (var + EPS)) + 4 * U) * 1.01, "rstd")

        def spread_out(v):
            return v[None, :, None]

        xhat = (r - spread_out(m)) * spread_out(want_r)
        d_xhat = (spread_out(d_mean) + 2 * U * r.abs()) * spread_out(want_r) + xhat.abs() * (
            spread_out(d_var / (2 * (var + EPS))) + 4 * U)
        wv, bv = w64.view(groups, per), b64.view(groups, per)
        u = xhat * wv + bv
        want = act64(u, act)
        tol = 1.1 * (d_xhat * wv.abs() + 2 * U * ((xhat * wv).abs() + bv.abs())) + 16 * U * (1 + u.abs()) * want.abs()
        tol = tol + HALF_STEP[dtype] * want.abs() + TINY[dtype]
        within(y2[lo:hi].view_as(want), want, tol, "output")
        # gradients from the call's own statistics
        m, s = mean[i].double(), rstd[i].double()
        xhat = (r - spread_out(m)) * spread_out(s)
        u = xhat * wv + bv
        near = act == "relu"
        du = g[lo:hi].view_as(xhat) * act_grad64(u, act)
        e = 4 * U * (r.abs() + spread_out(m).abs()) * spread_out(s) + 4 * U * xhat.abs()  # of xhat
        e_u = e * wv.abs() + 2 * U * ((xhat * wv).abs() + bv.abs())  # of u
        e_du = g[lo:hi].view_as(xhat).abs() * (e_u + 24 * U * (1 + u.abs())) if act == "silu" else 2 * U * du.abs()
        if near:  # where u is next to zero either side is right
            e_du = e_du + g[lo:hi].view_as(xhat).abs() * (u.abs() <= e_u)
        e_dux = e_du * xhat.abs() + du.abs() * e + U * (du * xhat).abs()
        sums[0] += du.sum(0).view(-1)
        sums[1] += (du * xhat).sum(0).view(-1)
        sums[2] += (e_du + (D + 2) * U * du.abs()).sum(0).view(-1)
        sums[3] += (e_dux + (D + 2) * U * (du * xhat).abs()).sum(0).view(-1)
        dxhat = du * wv
        n = (hi - lo) * per
        c1, c2 = dxhat.sum((0, 2)) / n, (dxhat * xhat).sum((0, 2)) / n
        e1 = ((e_du + (D + 4) * U * du.abs()) * wv.abs()).sum((0, 2)) / n
        e2 = ((e_dux + (D + 4) * U * (du * xhat).abs()) * wv.abs()).sum((0, 2)) / n
        want = (dxhat - spread_out(c1) - xhat * spread_out(c2)) * spread_out(s)
        terms = dxhat.abs() + spread_out(c1).abs() + (xhat * spread_out(c2)).abs()
        tol = (e_du * wv.abs() + spread_out(e1) + xhat.abs() * spread_out(e2) + e * spread_out(c2).abs() + 6 * U * terms)
        tol = tol * spread_out(s) * 1.01 + HALF_STEP[dtype] * want.abs() + TINY[dtype]
        within(dx2[lo:hi].view_as(want), want, tol, "input gradient")
    assert not y2[last:].any() and not dx2[last:].any()
    half = HALF_STEP[dw.dtype]
    within(db, sums[0], 1.01 * sums[2] + half * sums[0].abs() + 1e-37, "bias gradient")
    within(dw, sums[1], 1.01 * sums[3] + half * sums[1].abs() + 1e-37, "weight gradient")


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_maps(ops, gpu_handle, guard_bands, dtype, act):
    check(ops, gpu_handle, (2, 9, 7, 64), 8, dtype, act, seed=1)


@pytest.mark.parametrize("shape,groups", [((1, 1), 1), ((3, 1, 8), 8), ((1, 1, 200), 8), ((5, 33, 24), 3), ((2, 17, 30), 10),
                                          ((2, 50, 7), 7), ((1, 300, 2048), 32), ((1, 5, 5000), 5), ((64, 2, 16), 2),
                                          ((3, 1000, 320), 32), ((2, 40, 4104), 1), ((1, 7000, 8), 1)])
def test_shapes(ops, gpu_handle, guard_bands, shape, groups):
    check(ops, gpu_handle, shape, groups, torch.float32, "silu", seed=2)
    check(ops, gpu_handle, shape, groups, torch.float16, "relu", seed=3)


@pytest.mark.parametrize("shape,groups", [((2, 8), 2), ((300, 64), 8), ((600, 2048), 32), ((513, 4096), 4096), ((70, 1, 128), 128),
                                          ((33, 5, 48), 3), ((900, 3, 30), 10), ((5, 64, 256), 1), ((40, 2, 2048), 32),
                                          ((9, 64, 64), 4), ((9, 65, 64), 4), ((50, 2, 3, 24), 2), ((200, 45), 1), ((3, 33), 1),
                                          ((300, 512), 1), ((100, 3, 1024), 1), ((50, 2, 240), 2), ((30, 4, 1536), 1)])
@pytest.mark.parametrize("dtype,act", [(torch.float32, "none"), (torch.float16, "silu"), (torch.bfloat16, "relu")])
def test_short_samples(ops, gpu_handle, guard_bands, shape, groups, dtype, act):
    """Up to 64 rows a sample; [N, C] is a sample a row."""
    check(ops, gpu_handle, shape, groups, dtype, act, seed=21)


@pytest.mark.parametrize("shape,groups", [((40, 100, 64), 8), ((700, 80, 32), 4), ((5, 200, 24), 3), ((300, 65, 512), 1), ((600, 1, 45), 1)])
@pytest.mark.parametrize("dtype,act", [(torch.float32, "silu"), (torch.float16, "relu")])
def test_many_samples_of_few_rows(ops, gpu_handle, guard_bands, shape, groups, dtype, act):
    check(ops, gpu_handle, shape, groups, dtype, act, seed=23)


def test_many_ragged_samples(ops, gpu_handle, guard_bands):
    gen = torch.Generator().manual_seed(24)
    ends = torch.randint(0, 60, (150,), generator=gen).cumsum(0).tolist()
    check(ops, gpu_handle, (ends[-1] + 11, 32), 4, torch.float16, "silu", ends=ends, seed=25)
    ends = torch.randint(300, 600, (70,), generator=gen).cumsum(0).tolist()
    check(ops, gpu_handle, (ends[-1] + 11, 128), 8, torch.float32, "relu", ends=ends, seed=26)


@pytest.mark.parametrize("shape,thread_rows", [((1, 4096, 128), 64), ((3, 50, 32), 1), ((8, 200000, 16), 44)])
def test_an_outlier_in_the_first_row(ops, gpu_handle, shape, thread_rows):
    """One value of 1e4 among values of size 1.  The thread that has it in its n rows sums up to n squares about it, n times
    the sample's whole sum of squares, in n additions that round by half a step of what is there by then: n^2 / 2 half steps
    of the variance, half of that for rstd, and four half steps for the rest."""
    x, _, _, _ = make(shape, torch.float32, 27, affine=None)
    x[:, 0] = 1e4
    _, _, rstd = ops.group_norm_act_forward(gpu_handle, x, None, None, 4, EPS, "none")
    var = x.double().reshape(shape[0], shape[1], 4, -1).var((1, 3), unbiased=False)
    assert ((rstd.double() * (var + EPS).sqrt() - 1).abs() <= (thread_rows ** 2 / 4 + 4) * U).all()


def test_short_samples_in_place_and_unaligned(ops, gpu_handle):
    x, w, b, dy = make((700, 2, 64), torch.float16, 22)
    raw = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
    off = raw[1:].view(x.shape).copy_(x)
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 8, EPS, "silu")
    y1, mean1, rstd1 = ops.group_norm_act_forward(gpu_handle, off, w, b, 8, EPS, "silu", out=off)
    assert torch.allclose(y, y1, atol=2e-3) and torch.allclose(rstd, rstd1, rtol=1e-5)
    want = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "silu")
    got = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "silu", out=dy)
    assert got[0] is dy and all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("rows,ends", [(1000, [300, 301, 301, 900]), (700, [0, 0, 700]), (513, [513]), (90, [0]), (50, [50, 50, 50]),
                                       (5000, list(range(0, 4500, 9))), (20000, [1, 19998, 19999]), (64, [10, 20, 30]),
                                       (3000, [2999])])
@pytest.mark.parametrize("dtype,c,groups", [(torch.float16, 16, 4), (torch.bfloat16, 128, 8), (torch.float32, 20, 5)])
def test_ragged_samples(ops, gpu_handle, guard_bands, rows, ends, dtype, c, groups):
    check(ops, gpu_handle, (rows, c), groups, dtype, "relu", ends=ends, seed=4)


def test_affine_types(ops, gpu_handle, guard_bands):
    for dtype in (torch.float16, torch.bfloat16):
        check(ops, gpu_handle, (2, 100, 32), 4, dtype, "silu", affine="same", grad_dtype=dtype, seed=5)
    check(ops, gpu_handle, (2, 100, 32), 4, torch.float16, "none", affine=None, seed=6)


def test_values_far_from_zero(ops, gpu_handle):
    """A mean of a thousand deviations costs the statistics nothing beyond the inputs' own rounding."""
    check(ops, gpu_handle, (2, 2000, 64), 8, torch.float32, "none", offset=0.0, seed=7)
    x = torch.randn(1, 4000, 32, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") + 1000.0
    _, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, None, None, 4, EPS, "none")
    r = x.double().view(4000, 4, 8)
    var = r.var((0, 2), unbiased=False)
    assert ((rstd.double()[0] / (var + EPS) ** -0.5 - 1).abs() < 1e-4).all()
    assert ((mean.double()[0] - r.mean((0, 2))).abs() < 1e-3).all()


def test_constant_rows(ops, gpu_handle):
    x = torch.full((2, 50, 16), 3.0, dtype=torch.float16, device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, None, None, 4, EPS, "none")
    assert not y.any() and (mean == 3).all() and torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5))


@pytest.mark.parametrize("shape,ends", [((0, 5, 16), None), ((0, 16), None), ((3, 0, 16), None), ((0, 16), [0, 0]), ((0, 16), []),
                                        ((40, 16), []), ((40, 16), [0, 0, 0])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_nothing_to_normalise(ops, gpu_handle, guard_bands, shape, ends, dtype):
    x, w, b, dy = make(shape, dtype, 30)
    e = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "silu", e)
    dx, dw, db = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, "silu", e)
    assert mean.shape == ((shape[0] if ends is None else len(ends)), 4)
    assert not y.any() and not dx.any() and not dw.any() and not db.any() and not mean.any()
    assert torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5))


@pytest.mark.parametrize("shape,ends", [((50, 32), None), ((2, 32), [1, 2]), ((9, 32), [1, 2, 9]), ((600, 32), list(range(1, 601)))])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_a_group_of_one_value_has_no_input_gradient(ops, gpu_handle, shape, ends, act):
    """The value is its own mean: the terms cancel exactly, nothing is left for rstd = 1 / sqrt(EPS) to enlarge."""
    x, w, b, dy = make(shape, torch.float32, 31)
    e = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 32, EPS, act, e)
    dx, dw, db = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 32, act, e)
    ones = 2 if ends == [1, 2, 9] else shape[0]  # rows that are samples of their own
    assert torch.equal(mean[:ones], x[:ones]) and not dx[:ones].any()
    assert ones < shape[0] or not dw.any()


def test_rows_without_a_sample_reach_nothing(ops, gpu_handle):
    """NaN and infinities behind the last sample change no output, and their own outputs are zero."""
    ends = torch.tensor([100, 250], dtype=torch.int32, device="cuda")
    x, w, b, dy = make((400, 32), torch.float16, 9)
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        x[250:], dy[250:] = fill, fill
        y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "silu", ends)
        outs.append((y, mean, rstd) + ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, "silu", ends))
    for o in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], o))
    assert not outs[0][0][250:].any() and not outs[0][3][250:].any()


def test_a_nan_stays_in_its_group(ops, gpu_handle):
    x, w, b, dy = make((3, 40, 32), torch.float32, 10)
    x[1, 5, 9] = float("nan")
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "relu")
    bad = torch.zeros(3, 40, 32, dtype=torch.bool, device="cuda")
    bad[1, :, 8:16] = True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.isnan(mean[1, 1]) and int(torch.isnan(mean).sum()) == 1


@pytest.mark.parametrize("offset", [1, 3])
def test_tensors_off_vector_alignment(ops, gpu_handle, offset):
    x, w, b, dy = make((2, 60, 64), torch.float16, 11)

    def shifted(t):
        raw = torch.zeros(t.numel() + offset, dtype=t.dtype, device="cuda")
        raw[offset:] = t.reshape(-1)
        return raw[offset:].view(t.shape)

    want = ops.group_norm_act_forward(gpu_handle, x, w, b, 8, EPS, "silu")
    got = ops.group_norm_act_forward(gpu_handle, shifted(x), shifted(w), shifted(b), 8, EPS, "silu", out=shifted(x))
    assert torch.allclose(want[0], got[0], atol=2e-3) and torch.allclose(want[2], got[2], rtol=1e-5)
    want = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, want[1], want[2], 8, "silu")
    got = ops.group_norm_act_backward(gpu_handle, shifted(dy), shifted(x), w, b, got[1], got[2], 8, "silu")
    assert torch.allclose(want[0], got[0], atol=4e-3) and torch.allclose(want[1], got[1], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("shape", [(2, 300, 64), (1, 40000, 64)])
def test_in_place(ops, gpu_handle, shape):
    x, w, b, dy = make(shape, torch.bfloat16, 12)
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 8, EPS, "silu")
    dx, dw, db = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "silu")
    x2, dy2 = x.clone(), dy.clone()
    assert torch.equal(ops.group_norm_act_forward(gpu_handle, x2, w, b, 8, EPS, "silu", out=x2)[0], y)
    got = ops.group_norm_act_backward(gpu_handle, dy2, x, w, b, mean, rstd, 8, "silu", out=dy2)
    assert torch.equal(dy2, dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)


def test_without_affine_gradients(ops, gpu_handle):
    x, w, b, dy = make((2, 300, 64), torch.float32, 13)
    _, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 8, EPS, "silu")
    full = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "silu")
    part = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "silu", affine_grad=False)
    assert part[1] is None and part[2] is None and torch.equal(full[0], part[0])


def test_bad_sample_ends_touch_nothing_outside(ops, gpu_handle, guard_bands):
    """Ends that decrease or leave the rows give unspecified values inside the outputs only."""
    x, w, b, dy = make((500, 16), torch.float16, 14)
    for ends in ([400, 100, 600], [-5, 2 ** 31 - 1, 7], [500, 0, 0]):
        e = torch.tensor(ends, dtype=torch.int32, device="cuda")
        y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "relu", e)
        ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, "relu", e)
    torch.cuda.synchronize()


def test_gradient_against_differences(ops, gpu_handle):
    """The directional derivative of sum(y * dy) in float, against a central difference in 64 bits
    (h^2 of the third derivative: 1e-4^2, and the float gradients' own 1e-5)."""
    x, w, b, dy = make((2, 30, 16), torch.float32, 15)
    gen = torch.Generator(device="cuda").manual_seed(16)
    v = [torch.randn(t.shape, generator=gen, device="cuda") for t in (x, w, b)]

    def value(h):
        xx, ww, bb = (t.double() + h * d.double() for t, d in zip((x, w, b), v))
        r = xx.view(2, 30, 4, 4)
        m = r.mean((1, 3), keepdim=True)
        xhat = (r - m) * (((r - m) ** 2).mean((1, 3), keepdim=True) + EPS) ** -0.5
        return (act64(xhat.view(2, 30, 16) * ww + bb, "silu") * dy.double()).sum()

    _, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "silu")
    grads = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, "silu")
    got = sum((g.double() * d.double()).sum() for g, d in zip(grads, v))
    want = (value(1e-4) - value(-1e-4)) / 2e-4
    scale = sum((g.double() * d.double()).abs().sum() for g, d in zip(grads, v))
    assert abs(got - want) <= 1e-5 * scale


def test_captured_call_follows_its_inputs(ops, gpu_handle):
    x, w, b, dy = make((900, 32), torch.float16, 17)
    ends = torch.tensor([300, 900], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
        out = ops.group_norm_act_forward(gpu_handle, x, w, b, 4, EPS, "relu", ends)
        grads = ops.group_norm_act_backward(gpu_handle, dy, x, w, b, out[1], out[2], 4, "relu", ends)
    gpu_handle.set_queue(torch.cuda.current_stream().cuda_stream)
    for seed, e in ((18, [10, 800]), (19, [900, 900])):
        x2, _, _, dy2 = make((900, 32), torch.float16, seed)
        x.copy_(x2)
        dy.copy_(dy2)
        ends.copy_(torch.tensor(e, dtype=torch.int32))
        graph.replay()
        want = ops.group_norm_act_forward(gpu_handle, x2, w, b, 4, EPS, "relu", ends)
        want_grads = ops.group_norm_act_backward(gpu_handle, dy2, x2, w, b, want[1], want[2], 4, "relu", ends)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        assert all(torch.equal(p, q) for p, q in zip(grads, want_grads))


def test_same_inputs_give_the_same_bits(ops, gpu_handle):
    x, w, b, dy = make((50000, 64), torch.float16, 20)
    ends = torch.tensor([7, 20000, 50000], dtype=torch.int32, device="cuda")
    runs = []
    for _ in range(3):
        y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, w, b, 8, EPS, "relu", ends)
        runs.append((y, mean, rstd) + ops.group_norm_act_backward(gpu_handle, dy, x, w, b, mean, rstd, 8, "relu", ends))
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], r))
