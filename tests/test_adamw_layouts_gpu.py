"""Parameters in channels-last and transposed order on the GPU: each step is that of the same values laid out contiguously."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orders_of_memory(pkg, bits, dtype):
    nn_ = importlib.import_module("mluops_b200.torch_nn")
    gen = torch.Generator(device="cuda").manual_seed(1)
    shapes = [((16, 8, 3, 5), (0, 2, 3, 1)), ((4, 8, 3, 3, 5), (0, 2, 3, 4, 1)), ((700, 33), (1, 0)), ((40, 7), (0, 1))]
    flat = [torch.randn([s[i] for i in order], generator=gen, device="cuda").to(dtype) for s, order in shapes]
    back = [[order.index(i) for i in range(len(order))] for _, order in shapes]
    ours = [torch.nn.Parameter(t.clone().permute(b)) for t, b in zip(flat, back)]
    plain = [torch.nn.Parameter(t.clone()) for t in flat]
    assert [tuple(p.shape) for p in ours] == [s for s, _ in shapes] and not ours[0].is_contiguous()
    opts = [nn_.AdamW(x, lr=1e-2, state_bits=bits) for x in (ours, plain)]
    for step in range(3):
        for p, q, b in zip(ours, plain, back):
            q.grad = torch.randn(q.shape, generator=gen, device="cuda").to(dtype)
            p.grad = q.grad.permute(b) if step == 1 else q.grad.permute(b).contiguous()
        for opt in opts:
            opt.step()
        for p, q, b in zip(ours, plain, back):
            assert torch.equal(p, q.permute(b))
            for key in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(opts[0].state[p][key], opts[1].state[q][key].permute(b))
