"""Calls of the training-step operators that other tests do not make: more shapes than a handle keeps plans for, and row
blocks that lie in one group.

Tolerance of a product: a sum of n products in float is off by at most n 2^-24 of the sum of their magnitudes, and the
stored type adds half a step (2^-11 for half) of the result.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_shapes_than_plans_are_kept(ops):
    handle = ops.Handle(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1300, 16, generator=gen, device="cuda")
    ends = torch.zeros(2, dtype=torch.int32, device="cuda")
    first = {}
    for turn in range(2):
        for rows in range(1, 1300):
            ends[0], ends[1] = rows // 3, rows
            out, mean, _ = ops.group_norm_act_forward(handle, x[:rows], None, None, 4, sample_ends=ends)
            if rows % 100 == 1:
                if turn == 0:
                    first[rows] = out, mean
                    want = torch.nn.functional.group_norm(x[rows // 3:rows].double().t().unsqueeze(0), 4).squeeze(0).t()
                    # one value a channel of groups of 4: 64 roundings of values up to rstd = 316 times x
                    assert (out[rows // 3:].double() - want).abs().max() <= 1e-4 * max(1.0, float(want.abs().max()))
                else:
                    assert all(torch.equal(a, b) for a, b in zip(first[rows], (out, mean)))
            assert len(handle.plans) <= 512
    handle.destroy()


@pytest.mark.parametrize("dtype,half_step", [(torch.float32, 2.0 ** -24), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("rows,groups,which,ci,co", [(8192, 4, 2, 64, 64), (8193, 4, 0, 64, 64), (8192, 32, 31, 40, 72),
                                                     (20000, 16, 5, 64, 24)])
def test_all_rows_in_one_group(ops, gpu_handle, dtype, half_step, rows, groups, which, ci, co):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, ci, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(rows, co, generator=gen, device="cuda").to(dtype)
    w = torch.randn(groups, ci, co, generator=gen, device="cuda").to(dtype)
    ends = torch.full((groups,), rows - 3, dtype=torch.int32, device="cuda")
    ends[:which] = 0

    def close(got, a, b):
        want, size = a.double() @ b.double(), a.double().abs() @ b.double().abs()
        bound = a.shape[1] * 2.0 ** -24 * size + half_step * want.abs() + 2.0 ** -25
        assert ((got.double() - want).abs() <= bound).all()

    y = ops.grouped_matmul_forward(gpu_handle, x, w, ends)
    dx = ops.grouped_matmul_backward_input(gpu_handle, dy, w, ends)
    dw = ops.grouped_matmul_backward_weight(gpu_handle, x, dy, ends)
    close(y[:-3], x[:-3], w[which])
    close(dx[:-3], dy[:-3], w[which].t())
    close(dw[which], x[:-3].t(), dy[:-3])
    assert not y[-3:].any() and not dx[-3:].any()
    assert not torch.cat([dw[:which], dw[which + 1:]]).any()
