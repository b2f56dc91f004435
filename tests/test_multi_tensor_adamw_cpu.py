"""mluOpMultiTensorAdamW without a GPU: status codes of the C ABI and the refusals of the
Python class (host-only handle; its tensors are CPU tensors, which no launch reaches)."""
import ctypes

import pytest
import torch

FLOAT, HALF, BF16, U8, I32 = 2, 1, 17, 7, 6


@pytest.fixture(scope="module")
def handle(ops):
    h = ops.Handle(0)
    yield h
    h.destroy()


GOOD = dict(param=FLOAT, grad=FLOAT, state=FLOAT, num=2, sizes=(5, 300), lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01,
            step=1)


def call(ops, handle, null=(), offset=None, **over):
    a = dict(GOOD, **over)
    buf = (ctypes.c_char * 65536)()
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    arrays = {}
    for i, name in enumerate(("param", "grad", "m", "v", "ms", "vs")):
        addrs = [base + 4096 * i + 1300 * k // 16 * 16 for k in range(len(a["sizes"]))]
        if offset and offset[0] == name:
            addrs[0] += offset[1]
        arrays[name] = (ctypes.c_void_p * len(addrs))(*addrs)
    if a["state"] != U8 and "keep_scales" not in over:
        arrays["ms"] = arrays["vs"] = None
    for name in null:
        arrays[name] = None
    sizes = None if "sizes" in null else (ctypes.c_int64 * len(a["sizes"]))(*a["sizes"])
    return ops.lib().mluOpMultiTensorAdamW(
        None if "handle" in null else handle.ptr, a["param"], a["grad"], a["state"], a["num"], sizes, arrays["param"],
        arrays["grad"], arrays["m"], arrays["v"], arrays["ms"], arrays["vs"], a["lr"], a["b1"], a["b2"], a["eps"],
        a["wd"], a["step"], a.get("grad_scale"), a.get("schedule"))


def test_valid_calls_reach_the_launch(ops, handle):
    for over in ({}, {"param": HALF, "grad": HALF}, {"param": BF16}, {"state": U8}, {"param": BF16, "grad": BF16, "state": U8},
                 {"lr": 0.0, "b1": 0.0, "b2": 0.0, "eps": 0.0, "wd": 0.0}):
        assert call(ops, handle, **over) == ops.STATUS_EXECUTION_FAILED, over  # host-only: nothing can be launched


def test_nothing_to_do(ops, handle):
    assert call(ops, handle, num=0, null=("param", "grad", "m", "v", "sizes")) == ops.STATUS_SUCCESS
    assert call(ops, handle, sizes=(0, 0)) == ops.STATUS_SUCCESS


@pytest.mark.parametrize("over", [
    {"param": I32, "grad": I32}, {"param": HALF, "grad": BF16}, {"param": FLOAT, "grad": HALF}, {"state": HALF},
    {"num": -1}, {"lr": -1.0}, {"lr": float("nan")}, {"lr": float("inf")}, {"b1": 1.0}, {"b1": -0.1}, {"b2": 1.0},
    {"b2": float("nan")}, {"eps": -1e-8}, {"eps": float("nan")}, {"wd": -0.1}, {"step": 0}, {"sizes": (5, -1)},
    {"grad_scale": 2}, {"schedule": 6}, {"keep_scales": True},
    {"null": ("handle",)}, {"null": ("param",)}, {"null": ("grad",)}, {"null": ("m",)}, {"null": ("v",)},
    {"null": ("sizes",)}, {"state": U8, "null": ("ms",)}, {"state": U8, "null": ("vs",)},
    {"offset": ("param", 2)}, {"offset": ("grad", 1)}, {"offset": ("m", 2)}, {"state": U8, "offset": ("vs", 2)},
])
def test_bad_parameters(ops, handle, over):
    assert call(ops, handle, **over) == ops.STATUS_BAD_PARAM


def lists(n=(5, 300), dtype=torch.float32, state=torch.float32):
    return ([torch.zeros(k, dtype=dtype) for k in n], [torch.zeros(k, dtype=state) for k in n],
            [torch.zeros(k, dtype=state) for k in n])


def test_class_refuses(ops, handle):
    p, m, v = lists()
    with pytest.raises(ValueError, match="lengths"):
        ops.MultiTensorAdamW(p, m[:1], v)
    with pytest.raises(ValueError, match="number of elements"):
        ops.MultiTensorAdamW(p, m[::-1], v)
    with pytest.raises(ValueError, match="overlap"):
        ops.MultiTensorAdamW([p[0], p[0]], [m[0], torch.zeros(5)], [v[0], torch.zeros(5)])
    with pytest.raises(ValueError, match="overlap"):
        ops.MultiTensorAdamW(p, m, m)
    with pytest.raises(ValueError, match="dense"):
        ops.MultiTensorAdamW([torch.zeros(3, 4).t()], [torch.zeros(12)], [torch.zeros(12)])
    with pytest.raises(ValueError, match="float32, or 8 bits"):
        ops.MultiTensorAdamW(*lists(state=torch.uint8))
    with pytest.raises(ValueError, match="come together"):
        ops.MultiTensorAdamW(*lists(state=torch.uint8), [torch.zeros(1), torch.zeros(2)])
    with pytest.raises(ValueError, match="one for each 256"):
        ops.MultiTensorAdamW(*lists(state=torch.uint8), [torch.zeros(1), torch.zeros(1)], [torch.zeros(1), torch.zeros(2)])
    opt = ops.MultiTensorAdamW(p, m, v)
    g = [torch.zeros(5), torch.zeros(300)]
    with pytest.raises(ValueError, match="1 gradients for 2"):
        opt.step(handle, g[:1], 1e-3)
    for bad in ([g[0], torch.zeros(301)], [g[0], torch.zeros(600)[::2]], [g[0], g[1].double()]):
        with pytest.raises(ValueError, match="gradients are dense"):
            opt.step(handle, bad, 1e-3)
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step(handle, g, 1e-3, grad_scale=torch.zeros(2))
    with pytest.raises(ValueError, match="schedule"):
        opt.step(handle, g, 1e-3, schedule=torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ops.MluOpError):  # passes every check; a host-only handle launches nothing
        opt.step(handle, g, 1e-3)
    ops.MultiTensorAdamW([], [], []).step(handle, [], 1e-3)
