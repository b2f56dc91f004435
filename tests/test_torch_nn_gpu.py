"""The training-step modules on the GPU: gradients against torch in 64 bits, the optimiser against
torch's, and a small sparse network trained with all of them together.

Tolerances: u = 2^-24 is half a step of float.  A chain of sums over n values is compared at n * 2^-23 of
the values' size plus the storage type's half steps; the sizes here keep n below 2^11, so 1e-4 relative
to the largest value covers float (2^11 * 2^-23 = 2.5e-4 of the mean magnitude's sum, which random signs
keep below 1e-4 of the largest), and 2^-7 bfloat16 (two half steps of 2^-8: the stored operand's and the
result's).
"""
import importlib
import threading

import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nn_(pkg):
    return importlib.import_module("mluops_b200.torch_nn")


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("mluops_b200.torch_sparse")


def close(got, want, tol):
    scale = want.abs().max().clamp(min=1e-30)
    assert (got.double() - want.double()).abs().max() <= tol * scale, float((got.double() - want.double()).abs().max() / scale)


def products64(x, w, ends):
    parts, lo = [], 0
    for g, hi in enumerate(ends):
        parts.append(x[lo:hi] @ w[g])
        lo = hi
    return torch.cat(parts + [x[lo:] @ torch.zeros_like(w[0])])


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2.0 ** -7)])
def test_grouped_matmul_gradients(nn_, dtype, tol):
    gen = torch.Generator(device="cuda").manual_seed(1)
    ends = [100, 100, 350]
    x = torch.randn(400, 32, generator=gen, device="cuda").to(dtype)
    w = torch.randn(3, 32, 48, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(400, 48, generator=gen, device="cuda").to(dtype)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = nn_.grouped_matmul(a, b, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    y.backward(dy)
    c, d = x.double().requires_grad_(), w.double().requires_grad_()
    z = products64(c, d, ends)
    z.backward(dy.double())
    for got, want in ((y, z), (a.grad, c.grad), (b.grad, d.grad)):
        close(got.detach(), want.detach(), tol)
        assert got.dtype == dtype


def test_grouped_matmul_takes_views_and_single_gradients(nn_):
    e = torch.tensor([30, 50], dtype=torch.int32, device="cuda")
    x = torch.randn(16, 60, device="cuda").t()
    w = torch.randn(2, 24, 16, device="cuda").transpose(1, 2)
    close(nn_.grouped_matmul(x, w, e), products64(x.double(), w.double(), [30, 50]), 1e-4)
    a = x.detach().clone().requires_grad_()
    nn_.grouped_matmul(a, w, e).sum().backward()
    assert a.grad is not None and not a.grad[50:].any()
    b = w.detach().clone().requires_grad_()
    nn_.grouped_matmul(x, b, e).sum().backward()  # an expanded gradient
    assert b.grad is not None


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_group_norm_matches_torch(nn_, act):
    gen = torch.Generator(device="cuda").manual_seed(2)
    m = nn_.GroupNormAct(4, 32, activation=act).cuda()
    with torch.no_grad():
        m.weight.copy_(1 + 0.1 * torch.randn(32, generator=gen, device="cuda"))
        m.bias.copy_(0.1 * torch.randn(32, generator=gen, device="cuda"))
    x = torch.randn(3, 5, 6, 32, generator=gen, device="cuda")
    dy = torch.randn(3, 5, 6, 32, generator=gen, device="cuda")
    a = x.clone().requires_grad_()
    y = m(a)
    y.backward(dy)
    c, w, b = x.double().requires_grad_(), m.weight.detach().double().requires_grad_(), m.bias.detach().double().requires_grad_()
    z = torch.nn.functional.group_norm(c.permute(0, 3, 1, 2), 4, w, b, 1e-5).permute(0, 2, 3, 1)
    z = z.relu() if act == "relu" else torch.nn.functional.silu(z) if act == "silu" else z
    z.backward(dy.double())
    for got, want in ((y, z), (a.grad, c.grad), (m.weight.grad, w.grad), (m.bias.grad, b.grad)):
        close(got.detach(), want.detach(), 1e-4)


def test_group_norm_on_a_sparse_tensor(nn_, sp):
    idx = torch.tensor([[0, 0, 0, 1], [0, 1, 0, 0], [2, 0, 0, 0], [2, 0, 1, 0], [2, 1, 1, 1]], dtype=torch.int32, device="cuda")
    f = torch.randn(5, 8, device="cuda", requires_grad=True)
    x = sp.SparseConvTensor(f, idx, [2, 2, 2], 3)
    assert x.sample_ends().tolist() == [2, 2, 5]
    y = nn_.GroupNormAct(2, 8, affine=False)(x)
    want = torch.cat([torch.nn.functional.group_norm(p.double().t().unsqueeze(0), 2).squeeze(0).t() for p in (f[:2], f[2:])])
    close(y.features.detach(), want.detach(), 1e-4)
    y.features.sum().backward()
    assert f.grad.shape == f.shape and y.sample_ends() is x.sample_ends()
    with pytest.raises(ValueError, match="ascending"):
        nn_.GroupNormAct(2, 8, affine=False)(sp.SparseConvTensor(f, idx.flip(0), [2, 2, 2], 3))


def parameters(dtype=torch.float32, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda").to(dtype)) for s in ((3, 3, 8, 16), (16,), (700, 33), (1,))]


def set_grads(params, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda").to(p.dtype)


def test_optimizer_follows_torch(nn_):
    ours, theirs = parameters(), parameters()
    a = nn_.AdamW([{"params": ours[:2]}, {"params": ours[2:], "lr": 3e-3, "weight_decay": 0.2}], lr=1e-2)
    b = torch.optim.AdamW([{"params": theirs[:2]}, {"params": theirs[2:], "lr": 3e-3, "weight_decay": 0.2}], lr=1e-2, foreach=False)
    for step in range(5):
        set_grads(ours, step)
        set_grads(theirs, step)
        if step in (1, 3):  # a parameter that takes no part has a step count of its own
            ours[1].grad = theirs[1].grad = None
        a.step()
        b.step()
    for p, q in zip(ours, theirs):  # 5 steps of about 20 roundings each
        assert ((p - q).abs() <= 100 * 2.0 ** -24 * (1 + q.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_resumes_from_its_state(nn_, bits, dtype):
    ours = parameters(dtype)
    opt = nn_.AdamW(ours, lr=1e-2, state_bits=bits)
    for step in range(2):
        set_grads(ours, step)
        opt.step()
    saved = opt.state_dict()
    copies = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    other = nn_.AdamW(copies, lr=1e-2, state_bits=bits)
    other.load_state_dict(saved)
    for p, q in zip(ours, copies):
        for key, value in opt.state[p].items():
            if torch.is_tensor(value):
                assert other.state[q][key].dtype == value.dtype and torch.equal(other.state[q][key], value)
                assert other.state[q][key].data_ptr() != value.data_ptr()
    for step in range(2, 4):
        set_grads(ours, step)
        set_grads(copies, step)
        opt.step()
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, copies))


def test_optimizer_follows_parameters_that_move(nn_):
    ours, fixed = parameters(), parameters()
    a, b = nn_.AdamW(ours, lr=1e-2), nn_.AdamW(fixed, lr=1e-2)
    for step in range(3):
        if step == 2:
            for p in ours:
                p.data = p.data.clone()
        set_grads(ours, step)
        set_grads(fixed, step)
        a.step()
        b.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, fixed))


def test_eight_bit_states_stay_close_to_float_ones(nn_):
    """One step from zero states is the same in both (the update uses the moments before they are rounded)."""
    a, b = parameters(), parameters()
    opts = [nn_.AdamW(a, lr=1e-2, state_bits=8), nn_.AdamW(b, lr=1e-2)]
    for params, opt in zip((a, b), opts):
        set_grads(params, 1)
        opt.step()
    for p, q in zip(a, b):  # approximate root and reciprocal: 2^-21 of an update of 1e-2
        assert ((p - q).abs() <= 2.0 ** -21 * 1e-2 + 4 * 2.0 ** -24 * q.abs()).all()


def test_gradient_scale(nn_):
    a, b = parameters(), parameters()
    x, y = nn_.AdamW(a, lr=1e-2), nn_.AdamW(b, lr=1e-2)
    set_grads(a, 1)
    set_grads(b, 1)
    for p in b:
        p.grad *= 0.5  # exact
    x.step(grad_scale=torch.tensor([0.5], device="cuda"))
    y.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_step(nn_, bits):
    """Forward, backward and optimiser in one captured graph, replayed with other data and another learning rate."""
    def build():
        torch.manual_seed(4)
        layer = nn_.GroupedLinear(2, 16, 24).cuda()
        norm = nn_.GroupNormAct(4, 24, activation="silu").cuda()
        lr = torch.tensor(1e-2, device="cuda")
        return layer, norm, lr, nn_.AdamW([*layer.parameters(), *norm.parameters()], lr=lr, state_bits=bits, capturable=True)

    x = torch.zeros(40, 16, device="cuda")
    ends = torch.tensor([10, 36], dtype=torch.int32, device="cuda")

    def one(layer, norm, opt):
        opt.zero_grad(set_to_none=False)
        loss = norm(layer(x, ends).view(2, 20, 24)).square().mean()
        loss.backward()
        opt.step()
        return loss

    def data(step):
        gen = torch.Generator(device="cuda").manual_seed(step)
        x.copy_(torch.randn(40, 16, generator=gen, device="cuda"))
        ends.copy_(torch.tensor([[10, 36], [0, 40], [39, 39]][step % 3], dtype=torch.int32))

    eager, captured = build(), build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        data(0)
        for m in (eager, captured):
            one(m[0], m[1], m[3])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = one(captured[0], captured[1], captured[3])
    for step in range(1, 4):
        data(step)
        for m in (eager, captured):
            m[2].fill_(1e-2 / step)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = one(eager[0], eager[1], eager[3])
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        for p, q in zip([*eager[0].parameters(), *eager[1].parameters()], [*captured[0].parameters(), *captured[1].parameters()]):
            assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_sparse_network_trains_with_all_of_them(nn_, sp, bits):
    """Submanifold convolution, group norm with relu, a grouped layer by sample, and the optimiser: the gradients of
    every parameter and of the features against torch in 64 bits; then the updated parameters."""
    import numpy as np
    rng = np.random.default_rng(5)
    idx = helpers.random_indices(rng, 3, [6, 7, 8], 300)
    idx = idx[np.lexsort(idx.T[::-1])]
    d_idx = torch.from_numpy(np.ascontiguousarray(idx)).cuda()
    feat = torch.from_numpy(rng.standard_normal((300, 16)).astype(np.float32)).cuda()
    torch.manual_seed(6)
    conv = sp.SubMConv3d(16, 32, 3, bias=False, indice_key="a").cuda()
    norm = nn_.GroupNormAct(4, 32, activation="relu").cuda()
    head = nn_.GroupedLinear(3, 32, 8).cuda()
    params = [conv.weight, norm.weight, norm.bias, head.weight]
    opt = nn_.AdamW(params, lr=1e-2, state_bits=bits)
    before = [p.detach().clone() for p in params]

    f = feat.clone().requires_grad_()
    x = sp.SparseConvTensor(f, d_idx, [6, 7, 8], 3)
    h = norm(conv(x))
    y = head(h.features, x.sample_ends())
    dy = torch.from_numpy(rng.standard_normal((300, 8)).astype(np.float32)).cuda()
    y.backward(dy)

    rb = x.indice_dict["a"]
    leaves = [t.detach().double().requires_grad_() for t in (feat, *before)]
    f64, wc, gw, gb, wh = leaves
    out = torch.zeros(300, 32, dtype=torch.float64, device="cuda")
    for k in range(27):
        n = rb.indice_num[k]
        out = out.index_add(0, rb.indice_pairs[k, 1, :n].long(), f64[rb.indice_pairs[k, 0, :n].long()] @ wc.view(27, 16, 32)[k])
    ends = x.sample_ends().tolist()
    parts = [torch.nn.functional.group_norm(out[a:b].t().unsqueeze(0), 4, gw, gb, 1e-5).squeeze(0).t().relu()
             for a, b in zip([0] + ends[:-1], ends)]
    z = products64(torch.cat(parts), wh, ends)
    z.backward(dy.double())
    close(y.detach(), z.detach(), 1e-4)
    for got, want in zip([f, *params], leaves):
        close(got.grad, want.grad, 1e-4)
    opt.step()
    for p, p0 in zip(params, before):  # first step: m / sqrt(v) = sign(g), but for epsilon
        g = p.grad.double()
        want = p0.double() * (1 - 1e-2 * 1e-2) - 1e-2 * g / (g.abs() + 1e-8)
        assert ((p.double() - want).abs() <= 1e-6).all()


def test_two_threads_at_once(nn_):
    """Each thread has a stream of its own and a handle of its own: results are those of one after the other."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    xs = [torch.randn(3000, 64, generator=gen, device="cuda") for _ in range(2)]
    w = torch.randn(4, 64, 96, generator=gen, device="cuda")
    e = torch.tensor([700, 1500, 1500, 2900], dtype=torch.int32, device="cuda")

    def work(x):
        a = x.clone().requires_grad_()
        y = nn_.group_norm_act(nn_.grouped_matmul(a, w, e), 8, activation="silu", sample_ends=e)
        y.square().sum().backward()
        return y.detach(), a.grad

    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = work(xs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as err:  # reported by the main thread
            errors.append(err)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
