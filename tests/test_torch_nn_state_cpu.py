"""The optimiser's saved states without a GPU: step counts and moments between ordinary and capturable
optimisers and from PyTorch's.  The library's call is replaced by the formula in 64 bits, so that
what is tested is what the class hands to it.

Tolerance: the moments are floats (half a step of 2^-24 a product or sum, and a step makes five of
them); the parameters are held in 64 bits.  Ten steps of 2e-2 stay within 10 * 5 * 2^-24 * 2e-2 each.
"""
import importlib

import pytest
import torch

TOL = 10 * 5 * 2.0 ** -24 * 2e-2 * 10


class Formula:
    """ops.MultiTensorAdamW for float states on the CPU."""

    def __init__(self, params, exp_avgs, exp_avg_sqs):
        self.lists = params, exp_avgs, exp_avg_sqs

    def step(self, handle, grads, lr, betas, epsilon, weight_decay, step, grad_scale=None, schedule=None):
        assert type(step) is int
        b1, b2 = betas
        c1, c2 = 1 - b1 ** step, 1 - b2 ** step
        if schedule is not None:
            lr, c1, c2 = schedule.double().tolist()
        for p, m, v, g in zip(*self.lists, grads):
            g = g.double()
            assert m.dtype == v.dtype == torch.float32
            m.copy_(m.double() * b1 + (1 - b1) * g)
            v.copy_(v.double() * b2 + (1 - b2) * g * g)
            p.copy_(p * (1 - lr * weight_decay) - lr / c1 * m / (v.double().sqrt() / c2 ** 0.5 + epsilon))


@pytest.fixture
def nn_(pkg, monkeypatch):
    m = importlib.import_module("mluops_b200.torch_nn")
    monkeypatch.setattr(m.ops, "MultiTensorAdamW", Formula)
    monkeypatch.setattr(m, "_handle", lambda device: None)
    return m


def parameters():
    gen = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(n, generator=gen, dtype=torch.float64)) for n in (5, 300)]


def set_grads(params, step):
    gen = torch.Generator().manual_seed(100 + step)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, dtype=torch.float64)


def replayed(opt, step):
    """What a replayed graph does: the eager step's work on the device, nothing in Python."""
    counts = {p: opt.state[p]["step"] for g in opt.param_groups for p in g["params"]}
    opt.step()
    for p, n in counts.items():
        opt.state[p]["step"] = n


def close(a, b):
    assert all(((p - q).abs() <= TOL * (1 + q.abs())).all() for p, q in zip(a, b))


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("second", [False, True])
def test_resumed_step_counts(nn_, first, second):
    """Five steps (a capturable optimiser's last three as replays), saved, loaded, five more: as ten of torch's."""
    ours, theirs, more = parameters(), parameters(), parameters()
    opt = nn_.AdamW(ours, lr=1e-2, capturable=first)
    ref = torch.optim.AdamW(theirs, lr=1e-2)
    for step in range(5):
        set_grads(ours, step)
        set_grads(theirs, step)
        (lambda: replayed(opt, step) if first and step >= 2 else opt.step())()
        ref.step()
    close(ours, theirs)
    saved = opt.state_dict()
    assert [s["step"] for s in saved["state"].values()] == [5, 5]
    with torch.no_grad():
        for p, q in zip(more, ours):
            p.copy_(q)
    other = nn_.AdamW(more, lr=1e-2, capturable=second)
    other.load_state_dict(saved)
    for step in range(5, 10):
        set_grads(more, step)
        set_grads(theirs, step)
        other.step()
        ref.step()
    close(more, theirs)
    assert [s["step"] for s in other.state_dict()["state"].values()] == [10, 10]


@pytest.mark.parametrize("capturable", [False, True])
def test_state_of_torchs_optimizer(nn_, capturable):
    theirs, more = parameters(), parameters()
    ref = torch.optim.AdamW(theirs, lr=1e-2)
    for step in range(5):
        set_grads(theirs, step)
        ref.step()
    with torch.no_grad():
        for p, q in zip(more, theirs):
            p.copy_(q)
    opt = nn_.AdamW(more, lr=1e-2, capturable=capturable)
    opt.load_state_dict(ref.state_dict())
    for s in opt.state.values():
        assert type(s["step"]) is int and s["exp_avg"].dtype == s["exp_avg_sq"].dtype == torch.float32
    for step in range(5, 10):
        set_grads(more, step)
        set_grads(theirs, step)
        opt.step()
        ref.step()
    # the moments came over rounded to float: 2^-24 of each more
    close(more, theirs)
    assert len(opt._plans) == 1  # one call for all tensors


def test_states_that_do_not_fit_are_refused_and_change_nothing(nn_):
    p = parameters()
    opt = nn_.AdamW(p, lr=1e-2)
    set_grads(p, 0)
    opt.step()

    def saved(**over):
        out = opt.state_dict()
        out["state"] = {i: dict(s) for i, s in out["state"].items()}
        out["state"][1].update(over)
        return out

    one = nn_.AdamW(parameters(), lr=1e-2, capturable=True)
    with pytest.raises(ValueError, match="step"):  # one count for a capturable group
        one.load_state_dict(saved(step=7))
    for over in (dict(exp_avg=torch.zeros(299)), dict(exp_avg_sq=torch.zeros(300, dtype=torch.int32)),
                 dict(exp_avg=torch.zeros(300, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            nn_.AdamW(parameters(), lr=1e-2).load_state_dict(saved(**over))
    for key in ("amsgrad", "maximize"):
        bad = saved()
        bad["param_groups"] = [dict(bad["param_groups"][0], **{key: True})]
        with pytest.raises(ValueError, match=key):
            one.load_state_dict(bad)
    assert not one.state and not one._schedules
    eight = nn_.AdamW(parameters(), state_bits=8)
    for q in eight.param_groups[0]["params"]:
        eight.state[q] = eight._new_state(q)
    bad = eight.state_dict()
    bad["state"] = {i: dict(s, exp_avg=s["exp_avg"].float()) for i, s in bad["state"].items()}
    with pytest.raises(ValueError, match="8 bits"):
        nn_.AdamW(parameters(), state_bits=8).load_state_dict(bad)


def test_learning_rate_that_was_a_tensor(nn_):
    p = parameters()
    opt = nn_.AdamW(p, lr=torch.tensor(1e-2, dtype=torch.float64), capturable=True)
    set_grads(p, 0)
    opt.step()
    other = nn_.AdamW(parameters(), lr=1e-3)
    other.load_state_dict(opt.state_dict())
    assert type(other.param_groups[0]["lr"]) is float and other.param_groups[0]["lr"] == 1e-2


def test_state_saved_with_its_counters_apart(nn_):
    """The form that earlier versions wrote: the count beside the states, and the steps of the eager calls in them."""
    p = parameters()
    opt = nn_.AdamW(p, lr=1e-2, capturable=True)
    set_grads(p, 0)
    opt.step()
    saved = opt.state_dict()
    saved["state"] = {i: dict(s, step=1) for i, s in saved["state"].items()}
    saved["schedules"] = {0: (torch.tensor(40.0, dtype=torch.float64), torch.tensor([1.0, 0.9, 0.999], dtype=torch.float64))}
    for capturable in (False, True):
        other = nn_.AdamW(parameters(), lr=1e-2, capturable=capturable)
        other.load_state_dict(saved)
        assert [s["step"] for s in other.state_dict()["state"].values()] == [40, 40]


@pytest.mark.parametrize("capturable", [False, True])
def test_betas_that_change_between_steps(nn_, capturable):
    ours, theirs = parameters(), parameters()
    opt, ref = nn_.AdamW(ours, lr=1e-2, capturable=capturable), torch.optim.AdamW(theirs, lr=1e-2)
    for step, betas in enumerate([(0.9, 0.999), (0.5, 0.9), (0.5, 0.9), (0.8, 0.99)]):
        set_grads(ours, step)
        set_grads(theirs, step)
        opt.param_groups[0]["betas"] = ref.param_groups[0]["betas"] = betas
        opt.step()
        ref.step()
    close(ours, theirs)


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_changes_nothing(nn_, capturable):
    """A gradient that is refused, in the second group: no parameter of either group moves, and no step is counted."""
    ours, theirs = parameters(), parameters()
    odd = torch.nn.Parameter(torch.zeros(3, 2, dtype=torch.float64))
    opt = nn_.AdamW([{"params": ours}, {"params": [odd]}], lr=1e-2, capturable=capturable)
    ref = torch.optim.AdamW(theirs, lr=1e-2)
    for step in range(3):
        set_grads(ours, step)
        set_grads(theirs, step)
        if step == 1:
            before = [p.detach().clone() for p in ours]
            odd.grad = torch.sparse_coo_tensor([[0]], [[1.0, 1.0]], (3, 2), dtype=torch.float64)
            with pytest.raises(ValueError, match="sparse"):
                opt.step()
            assert all(torch.equal(p, q) for p, q in zip(ours, before))
            odd.grad = None
        opt.step()
        ref.step()
    close(ours, theirs)
    assert [s["step"] for s in opt.state_dict()["state"].values()][:2] == [3, 3]
