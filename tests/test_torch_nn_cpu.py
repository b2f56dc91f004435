"""What the training-step modules refuse before anything is launched (no GPU needed)."""
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def nn_(pkg):
    return importlib.import_module("mluops_b200.torch_nn")


def test_optimizer_refuses(nn_):
    p = [torch.nn.Parameter(torch.zeros(3))]
    for over in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                 dict(weight_decay=-0.1), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            nn_.AdamW(p, **over)


def test_optimizer_without_gradients_does_nothing(nn_):
    opt = nn_.AdamW([torch.nn.Parameter(torch.zeros(3))])
    assert opt.step() is None and not opt.state
    assert opt.step(lambda: 7) == 7


def test_sparse_gradient_is_refused(nn_):
    p = torch.nn.Parameter(torch.zeros(3, 2))
    p.grad = torch.sparse_coo_tensor([[0]], [[1.0, 1.0]], (3, 2))
    with pytest.raises(ValueError, match="sparse"):
        nn_.AdamW([p]).step()


def test_modules_hold_their_parameters(nn_):
    m = nn_.GroupedLinear(3, 8, 16, dtype=torch.bfloat16)
    assert m.weight.shape == (3, 8, 16) and m.weight.dtype == torch.bfloat16 and float(m.weight.detach().abs().max()) <= 8 ** -0.5 * (1 + 2.0 ** -8)
    g = nn_.GroupNormAct(4, 16)
    assert (g.weight == 1).all() and not g.bias.any()
    assert nn_.GroupNormAct(4, 16, affine=False).weight is None


def test_optimizer_copies_and_pickles(nn_):
    import copy
    import pickle
    p = torch.nn.Parameter(torch.zeros(4))
    opt = nn_.AdamW([p], lr=1e-2, state_bits=8, capturable=True)
    opt._plans[0] = lambda: None  # what is laid out for the calls stays behind
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.state_bits == 8 and other.capturable and other._plans == {} and other._schedules == {}
        assert other.param_groups[0]["lr"] == 1e-2 and other.param_groups[0]["params"][0] is not p


def test_optimizer_refuses_states_of_other_bits(nn_):
    p = torch.nn.Parameter(torch.zeros(4))
    saved = {bits: nn_.AdamW([p], state_bits=bits) for bits in (8, 32)}
    for opt in saved.values():
        opt.state[p] = opt._new_state(p)
    for bits in (8, 32):
        nn_.AdamW([p], state_bits=bits).load_state_dict(saved[bits].state_dict())
        with pytest.raises(ValueError):
            nn_.AdamW([p], state_bits=bits).load_state_dict(saved[40 - bits].state_dict())
