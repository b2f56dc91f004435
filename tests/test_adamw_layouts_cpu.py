"""Dense parameters in another order than the contiguous one, without a GPU: what the optimiser takes and refuses."""
import importlib
import types

import pytest
import torch


def handle():
    return types.SimpleNamespace(device=-1, ptr=None)


@pytest.fixture
def lib(ops, monkeypatch):
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(mluOpMultiTensorAdamW=lambda *a: 0, mluOpMultiTensorAdamW_v2=lambda *a: 0))


def like(p, dtype=torch.float32):
    return torch.zeros_like(p, dtype=dtype, requires_grad=False)


ORDERS = [lambda: torch.zeros(3, 4).t(), lambda: torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last),
          lambda: torch.zeros(4, 2, 1, 3).permute(3, 0, 2, 1), lambda: torch.zeros(5, 1).t(), lambda: torch.zeros(0, 3).t()]


@pytest.mark.parametrize("make", ORDERS)
def test_dense_orders_are_taken(ops, lib, make):
    p = make()
    for state in (torch.float32, torch.uint8):
        scales = [[torch.zeros(-(-p.numel() // 256))] for _ in range(2)] if state == torch.uint8 else []
        ops.MultiTensorAdamW([p], [like(p, state)], [like(p, state)], *scales).step(handle(), [like(p)], 1e-3)


def test_other_orders_are_refused(ops, lib):
    p = torch.zeros(4, 5).t()
    for bad in (torch.zeros(5, 4), torch.zeros(20), torch.zeros(4, 5)):
        with pytest.raises(ValueError, match="dense"):
            ops.MultiTensorAdamW([p], [bad], [like(p)])
        with pytest.raises(ValueError, match="dense"):
            ops.MultiTensorAdamW([p], [like(p)], [bad])
        with pytest.raises(ValueError, match="gradients are dense"):
            ops.MultiTensorAdamW([p], [like(p)], [like(p)]).step(handle(), [bad], 1e-3)
    q = torch.zeros(5, 4)
    with pytest.raises(ValueError, match="dense"):
        ops.MultiTensorAdamW([q], [like(p)], [like(q)])
    with pytest.raises(ValueError, match="gradients are dense"):
        ops.MultiTensorAdamW([q], [like(q)], [like(q)]).step(handle(), [like(p)], 1e-3)
    for sparse in (torch.zeros(8, 4)[::2], torch.zeros(4, 8)[:, ::2], torch.zeros(1, 4).expand(3, 4), torch.zeros(6, 6).t()[1:]):
        with pytest.raises(ValueError, match="dense"):
            ops.MultiTensorAdamW([sparse], [torch.zeros_like(sparse)], [torch.zeros_like(sparse)])


def test_states_and_gradients_follow_the_parameters_order(pkg, ops, lib, monkeypatch):
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    monkeypatch.setattr(nn_, "_handle", lambda device: handle())
    for bits in (32, 8):
        params = [torch.nn.Parameter(make()) for make in ORDERS]
        opt = nn_.AdamW(params, state_bits=bits)
        for p in params:
            p.grad = torch.zeros(p.shape)  # contiguous: the step lays it out anew
        opt.step()
        for p in params:
            assert opt.state[p]["exp_avg"].stride() == opt.state[p]["exp_avg_sq"].stride() == p.stride()
            assert opt.state[p]["exp_avg"].shape == p.shape
        other = nn_.AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=bits)
        other.load_state_dict(opt.state_dict())
        for p in other.param_groups[0]["params"]:
            p.grad = torch.zeros(p.shape)
        other.step()


def test_order_that_changes_under_the_same_address(pkg, ops, lib, monkeypatch):
    """A parameter that is transposed in place keeps its address; its states no longer fit it."""
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    monkeypatch.setattr(nn_, "_handle", lambda device: handle())
    p = torch.nn.Parameter(torch.zeros(4, 4))
    opt = nn_.AdamW([p])
    p.grad = torch.zeros(4, 4)
    opt.step()
    p.data = p.data.t()
    with pytest.raises(ValueError, match="dense"):
        opt.step()


def test_loaded_states_are_laid_out_like_the_parameter(pkg):
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    p = torch.nn.Parameter(torch.zeros(3, 4))
    values = torch.arange(12.0).view(3, 4)
    opt = nn_.AdamW([p])
    opt.state[p] = {"step": 2, "exp_avg": values, "exp_avg_sq": values.clone()}
    q = torch.nn.Parameter(torch.zeros(4, 3).t())
    other = nn_.AdamW([q])
    other.load_state_dict(opt.state_dict())
    assert torch.equal(other.state[q]["exp_avg"], values) and other.state[q]["exp_avg"].stride() == q.stride()
    eight = nn_.AdamW([p], state_bits=8)
    eight.state[p] = eight._new_state(p)
    with pytest.raises(ValueError, match="order"):  # the blocks of 256 lie in another order
        nn_.AdamW([q], state_bits=8).load_state_dict(eight.state_dict())
