"""The optimiser's states on the GPU: what is saved after replayed graphs, and what the class keeps between steps.

Tolerance against torch's optimiser: a step of 1e-2 has about 20 roundings of float (2^-24) of the value, as in
test_torch_nn_gpu.py; the capturable schedule rounds its three floats once more.
"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nn_(pkg):
    return importlib.import_module("mluops_b200.torch_nn")


def parameters(seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda")) for s in ((3, 3, 8, 16), (16,), (700, 33))]


def set_grads(params, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in params:
        g = torch.randn(p.shape, generator=gen, device="cuda")
        if p.grad is None:
            p.grad = g
        else:
            p.grad.copy_(g)


def copies(params):
    return [torch.nn.Parameter(p.detach().clone()) for p in params]


def capture(opt):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    return graph


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("second", [False, True])
def test_resumes_after_replays(nn_, bits, second):
    """Two eager steps, three replays, saved: three more steps elsewhere are those of an optimiser that ran eagerly."""
    ours, plain = parameters(), parameters()
    opt = nn_.AdamW(ours, lr=1e-2, state_bits=bits, capturable=True)
    ref = nn_.AdamW(plain, lr=1e-2, state_bits=bits, capturable=second)
    for step in range(2):
        set_grads(ours, step)
        set_grads(plain, step)
        opt.step()
        ref.step()
    graph = capture(opt)
    for step in range(2, 5):
        set_grads(ours, step)
        set_grads(plain, step)
        graph.replay()
        ref.step()
    saved = opt.state_dict()
    assert [s["step"] for s in saved["state"].values()] == [5, 5, 5]
    more = copies(ours)
    other = nn_.AdamW(more, lr=1e-2, state_bits=bits, capturable=second)
    other.load_state_dict(saved)
    for step in range(5, 8):
        set_grads(more, step)
        set_grads(plain, step)
        other.step()
        ref.step()
    assert [s["step"] for s in other.state_dict()["state"].values()] == [8, 8, 8]
    if bits == 32:
        for p, q in zip(more, plain):
            assert ((p - q).abs() <= 8 * 25 * 2.0 ** -24 * (1 + q.abs())).all()
    elif second:  # the same arithmetic throughout
        assert all(torch.equal(p, q) for p, q in zip(more, plain))


def test_state_of_torchs_optimizer(nn_):
    theirs = parameters()
    ref = torch.optim.AdamW(theirs, lr=1e-2, foreach=False)
    for step in range(4):
        set_grads(theirs, step)
        ref.step()
    for capturable in (False, True):
        ours, rest = copies(theirs), copies(theirs)
        opt, base = nn_.AdamW(ours, lr=1e-2, capturable=capturable), torch.optim.AdamW(rest, lr=1e-2, foreach=False)
        opt.load_state_dict(ref.state_dict())
        base.load_state_dict(ref.state_dict())
        for step in range(4, 7):
            set_grads(ours, step)
            set_grads(rest, step)
            opt.step()
            base.step()
        for p, q in zip(ours, rest):
            assert ((p - q).abs() <= 7 * 25 * 2.0 ** -24 * (1 + q.abs())).all()
        assert len(opt._plans) == 1


def test_betas_that_change_between_steps(nn_):
    """Eager and captured steps of a capturable optimiser use the betas of the moment, as the ordinary one does."""
    sets = [parameters() for _ in range(3)]
    opts = [nn_.AdamW(p, lr=1e-2, capturable=c) for p, c in zip(sets, (False, True, True))]
    for step, betas in enumerate([(0.9, 0.999), (0.5, 0.9), (0.5, 0.9), (0.8, 0.99)]):
        for i, (p, opt) in enumerate(zip(sets, opts)):
            set_grads(p, step)
            opt.param_groups[0]["betas"] = betas
            if i == 2 and step:  # captured anew whenever they change, and back
                if step != 2:
                    graph = capture(opt)
                graph.replay()
            else:
                opt.step()
    for p, q, r in zip(*sets):
        assert torch.equal(q, r)
        assert ((p - q).abs() <= 4 * 25 * 2.0 ** -24 * (1 + p.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_with_a_number_as_learning_rate(nn_, bits):
    ours, plain = parameters(), parameters()
    opt, ref = [nn_.AdamW(p, lr=1e-2, state_bits=bits, capturable=True) for p in (ours, plain)]
    for p, o in ((ours, opt), (plain, ref)):
        set_grads(p, 0)
        o.step()
    graph = capture(opt)
    for step in (1, 2):
        set_grads(ours, step)
        set_grads(plain, step)
        graph.replay()
        ref.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, plain))


def test_capture_of_an_ordinary_step_is_refused(nn_):
    """Its step count and learning rate would be those of the capture in every replay."""
    ours = parameters()
    opt = nn_.AdamW(ours, lr=1e-2)
    set_grads(ours, 0)
    opt.step()
    before = [p.detach().clone() for p in ours]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    one = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="capturable=True"):
            opt.step()
        one += 1
    graph.replay()
    assert one.item() == 1 and all(torch.equal(p, q) for p, q in zip(ours, before))
    assert [s["step"] for s in opt.state.values()] == [1, 1, 1]


@pytest.mark.parametrize("loaded", [False, True])
def test_capture_of_the_first_step_is_refused(nn_, loaded):
    """States and counts made inside a graph would be cleared by every replay.  (loaded: states without a step yet.)"""
    ours = parameters()
    opt = nn_.AdamW(ours, lr=1e-2, capturable=True)
    set_grads(ours, 0)
    if loaded:
        first = nn_.AdamW(copies(ours), lr=1e-2, capturable=True)
        for p in first.param_groups[0]["params"]:
            first.state[p] = first._new_state(p)
        opt.load_state_dict(first.state_dict())
    before = [p.detach().clone() for p in ours]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    one = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="before the capture"):
            opt.step()
        one += 1
    graph.replay()
    assert one.item() == 1 and all(torch.equal(p, q) for p, q in zip(ours, before))
    opt.step()
    graph = capture(opt)
    graph.replay()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2, 2]
