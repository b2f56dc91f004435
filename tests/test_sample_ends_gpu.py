"""Sample ends of sparse tensors: handed on by convolutions and norms without a host read, and never stale."""
import importlib

import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu

SPACE, BATCH = [6, 9, 8], 3


@pytest.fixture(scope="module")
def nn_(pkg):
    return importlib.import_module("mluops_b200.torch_nn")


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("mluops_b200.torch_sparse")


def make(sp, n=300, channels=16, seed=1, batch=BATCH):
    rng = np.random.default_rng(seed)
    idx = helpers.random_indices(rng, batch, SPACE, n)
    idx = np.ascontiguousarray(idx[np.lexsort(idx.T[::-1])])
    f = torch.from_numpy(rng.standard_normal((n, channels)).astype(np.float32)).cuda()
    return sp.SparseConvTensor(f, torch.from_numpy(idx).cuda(), SPACE, batch)


def counted(x):
    return torch.bincount(x.indices[:, 0].long(), minlength=x.batch_size).cumsum(0).tolist()


class no_host_reads:
    def __enter__(self):
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")

    def __exit__(self, *_):
        torch.cuda.set_sync_debug_mode("default")


def test_strided_layers_need_no_host_read(sp):
    x = make(sp)
    for key in (None, "down"):
        y = sp.SparseConv3d(16, 8, 3, stride=2, padding=1, indice_key=key).cuda()(x)
        with no_host_reads():
            ends = y.sample_ends()
        assert ends.tolist() == counted(y) and ends.dtype == torch.int32


def test_submanifold_layers_hand_on_their_inputs_ends(sp, nn_):
    x = make(sp)
    conv = sp.SubMConv3d(16, 16, 3, indice_key="a").cuda()
    norm = nn_.GroupNormAct(4, 16).cuda()
    y = norm(conv(x))
    with no_host_reads():  # asked for once, by the first norm
        assert x.sample_ends() is y.sample_ends() is conv(y).sample_ends() is norm(conv(conv(x))).sample_ends()
    assert y.sample_ends().tolist() == counted(x)
    alone = sp.SubMConv3d(16, 16, 3).cuda()
    assert alone(x).sample_ends() is x.sample_ends()


def test_norm_behind_a_strided_layer(sp, nn_):
    """Values and gradients of a strided convolution and a norm against 64 bits.  Tolerance as in test_torch_nn_gpu.py."""
    x = make(sp)
    f = x.features.requires_grad_()
    conv = sp.SparseConv3d(16, 8, 3, stride=2, padding=1, bias=False, indice_key="b").cuda()
    y = nn_.GroupNormAct(2, 8, affine=False, activation="silu")(conv(x))
    dy = torch.randn(y.features.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    y.features.backward(dy)
    rb = x.indice_dict["b"]
    f64, w = f.detach().double().requires_grad_(), conv.weight.detach().double().requires_grad_()
    out = torch.zeros(rb.num_act_out, 8, dtype=torch.float64, device="cuda")
    for k in range(27):
        n = rb.indice_num[k]
        out = out.index_add(0, rb.indice_pairs[k, 1, :n].long(), f64[rb.indice_pairs[k, 0, :n].long()] @ w.view(27, 16, 8)[k])
    ends = counted(y)
    z = torch.cat([torch.nn.functional.silu(torch.nn.functional.group_norm(out[a:b].t().unsqueeze(0), 2).squeeze(0).t())
                   for a, b in zip([0] + ends[:-1], ends)])
    z.backward(dy.double())
    for got, want in ((y.features, z), (f.grad, f64.grad), (conv.weight.grad, w.grad)):
        assert (got.double() - want).abs().max() <= 1e-4 * want.abs().max()


def test_changed_indices_are_noticed(sp):
    x = make(sp)
    first = x.sample_ends()
    assert x.sample_ends() is first
    x.indices[:, 0] = 0  # in place
    assert x.sample_ends().tolist() == [300, 300, 300]
    x.indices[100:, 0] = 2
    x.indices = x.indices[50:].contiguous()  # replaced
    x.features = x.features[50:]
    assert x.sample_ends().tolist() == [50, 50, 250]
    x.batch_size = 4
    assert x.sample_ends().tolist() == [50, 50, 250, 250]
    x.indices[0, 0] = 3
    with pytest.raises(ValueError, match="ascending"):
        x.sample_ends()


def test_changed_outputs_of_a_strided_layer_are_checked(sp):
    y = sp.SparseConv3d(16, 8, 3, stride=2, padding=1).cuda()(make(sp))
    y.indices.copy_(y.indices.flip(0))
    with pytest.raises(ValueError, match="ascending"):
        y.sample_ends()


def test_stack_is_captured(sp, nn_, monkeypatch):
    """Convolutions that share rulebooks, norms between them: no host read once the rulebooks are there, and one graph."""
    monkeypatch.delenv("MLUOP_B200_CHECK_STATUS", raising=False)
    x = make(sp)
    layers = [sp.SubMConv3d(16, 16, 3, indice_key="a"), nn_.GroupNormAct(4, 16, activation="relu"),
              sp.SparseConv3d(16, 32, 3, stride=2, padding=1, indice_key="b"), nn_.GroupNormAct(4, 32, activation="silu"),
              sp.SubMConv3d(32, 32, 3, indice_key="c"), nn_.GroupNormAct(8, 32)]
    layers = [m.cuda() for m in layers]

    def run():
        y = sp.SparseConvTensor(x.features, x.indices, SPACE, BATCH, x.indice_dict)
        for m in layers:
            y = m(y)
        return y.features

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        run()
        with no_host_reads():
            run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side), torch.no_grad():
        out = run()
    for seed in (5, 6):
        x.features.copy_(torch.randn(x.features.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        with torch.no_grad():
            assert torch.equal(out, run())


def test_capture_without_known_ends_is_refused(sp, nn_):
    x = make(sp)
    norm = nn_.GroupNormAct(4, 16).cuda()
    norm(make(sp))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one = torch.ones(1, device="cuda")  # (the capture itself goes on)
        with pytest.raises(RuntimeError, match="before the capture"):
            norm(x)
        one += 1
    graph.replay()
    torch.cuda.synchronize()
    assert one.item() == 2 and x.sample_ends().tolist() == counted(x)


def test_ends_worked_out_in_a_graph_are_not_kept(sp):
    """A strided layer's ends can be worked out inside a capture; outside it they are worked out again."""
    y = sp.SparseConv3d(16, 8, 3, stride=2, padding=1).cuda()(make(sp))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        inside = y.sample_ends()
    outside = y.sample_ends()
    assert outside is not inside and outside.tolist() == counted(y)
    graph.replay()
    torch.cuda.synchronize()
    assert inside.tolist() == counted(y)


def test_inference_mode_and_empty_samples(sp, nn_):
    with torch.inference_mode():
        x = make(sp)
        y = nn_.GroupNormAct(4, 16).cuda()(sp.SubMConv3d(16, 16, 3, indice_key="a").cuda()(x))
        assert y.sample_ends() is x.sample_ends()
    none = sp.SparseConvTensor(torch.zeros(0, 16, device="cuda"), torch.zeros(0, 4, dtype=torch.int32, device="cuda"), SPACE, 2)
    assert none.sample_ends().tolist() == [0, 0]
    last = make(sp, batch=1)
    last = sp.SparseConvTensor(last.features, last.indices, SPACE, 3)
    assert last.sample_ends().tolist() == [300, 300, 300]
