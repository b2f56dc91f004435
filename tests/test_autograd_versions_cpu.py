"""Tensors that the library writes through their addresses count as changed for autograd: a backward pass that needs
their old values is refused instead of computed from the new ones.  Without a GPU: the library's call is left out."""
import types

import pytest
import torch


@pytest.fixture
def opt(ops, monkeypatch):
    p = torch.nn.Parameter(torch.ones(4))
    made = ops.MultiTensorAdamW([p], [torch.zeros(4)], [torch.zeros(4)])
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(mluOpMultiTensorAdamW=lambda *a: 0))
    made.handle = types.SimpleNamespace(device=-1, ptr=None)
    return made


def test_a_step_changes_parameters_and_states(opt):
    before = [t._version for t in opt.params + opt.exp_avgs + opt.exp_avg_sqs]
    opt.step(opt.handle, [torch.ones(4)], 1e-3)
    assert all(t._version > v for t, v in zip(opt.params + opt.exp_avgs + opt.exp_avg_sqs, before))


def test_backward_through_a_graph_from_before_the_step_is_refused(opt):
    p = opt.params[0]
    loss = (p * p).sum()
    opt.step(opt.handle, [torch.ones(4)], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_eight_bit_states_and_scales_too(ops, monkeypatch):
    state = [torch.zeros(4, dtype=torch.uint8) for _ in range(2)] + [torch.zeros(1) for _ in range(2)]
    made = ops.MultiTensorAdamW([torch.ones(4)], *[[t] for t in state])
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(mluOpMultiTensorAdamW=lambda *a: 0))
    made.step(types.SimpleNamespace(device=-1, ptr=None), [torch.ones(4)], 1e-3)
    assert all(t._version == 1 for t in state + made.params)


def test_tensors_of_inference_mode_have_no_count(ops, monkeypatch):
    with torch.inference_mode():
        tensors = [[torch.ones(4)] for _ in range(3)]
    made = ops.MultiTensorAdamW(*tensors)
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(mluOpMultiTensorAdamW=lambda *a: 0))
    made.step(types.SimpleNamespace(device=-1, ptr=None), [torch.ones(4)], 1e-3)


def test_views_count_for_their_base(ops, monkeypatch):
    flat = [torch.zeros(12) for _ in range(3)]
    made = ops.MultiTensorAdamW(*[[f[:4], f[4:].view(2, 4)] for f in flat])
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(mluOpMultiTensorAdamW=lambda *a: 0))
    made.step(types.SimpleNamespace(device=-1, ptr=None), [torch.ones(4), torch.ones(2, 4)], 1e-3)
    assert all(f._version == 1 for f in flat) and all(t._version == 1 for t in made.params)
