"""The same on the GPU, through the calls themselves: the optimiser's step and the operators' `out` arguments."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_backward_through_a_graph_from_before_the_step_is_refused(pkg):
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    for bits in (32, 8):
        layer = nn_.GroupedLinear(2, 16, 24).cuda()
        opt = nn_.AdamW(layer.parameters(), lr=1e-2, state_bits=bits)
        x = torch.randn(40, 16, device="cuda", requires_grad=True)
        ends = torch.tensor([10, 36], dtype=torch.int32, device="cuda")
        layer(x, ends).sum().backward()
        kept = layer(x, ends).sum()
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
        layer(x, ends).sum().backward()  # of the new weights


def test_out_counts_as_written(ops, gpu_handle):
    x = torch.randn(6, 5, 16, device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(gpu_handle, x, None, None, 4)
    rows, w = torch.randn(30, 16, device="cuda"), torch.randn(2, 16, 24, device="cuda")
    ends = torch.tensor([10, 30], dtype=torch.int32, device="cuda")
    for call, out in ((lambda t: ops.group_norm_act_forward(gpu_handle, x, None, None, 4, out=t), torch.empty_like(x)),
                      (lambda t: ops.group_norm_act_forward(gpu_handle, t, None, None, 4, out=t), x.clone()),
                      (lambda t: ops.group_norm_act_backward(gpu_handle, t, x, None, None, mean, rstd, 4, out=t), x.clone()),
                      (lambda t: ops.grouped_matmul_forward(gpu_handle, rows, w, ends, out=t), torch.empty(30, 24, device="cuda")),
                      (lambda t: ops.grouped_matmul_backward_input(gpu_handle, torch.ones(30, 24, device="cuda"), w, ends, out=t),
                       torch.empty_like(rows)),
                      (lambda t: ops.grouped_matmul_backward_weight(gpu_handle, rows, torch.ones(30, 24, device="cuda"), ends, out=t),
                       torch.empty_like(w))):
        a = torch.ones(out.numel(), device="cuda", requires_grad=True)
        loss = (a * out.view(-1)).sum()
        version = out._version
        call(out)
        assert out._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
