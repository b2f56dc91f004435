"""mluOpGroupedMatMul* without a GPU: status codes of the C ABI and the refusals of the Python
wrappers (host-only handle, CPU tensors that no launch reaches)."""
import ctypes

import pytest
import torch

FLOAT, HALF, BF16, I32, I64, ARRAY = 2, 1, 17, 6, 9, 4


@pytest.fixture(scope="module")
def handle(ops):
    h = ops.Handle(0)
    yield h
    h.destroy()


class Call:
    APART = 1 << 22  # between the tensors' addresses, which nothing reads

    def __init__(self, ops, handle, dtype=HALF, rows=10, groups=3, ci=16, co=24, **over):
        self.ops, self.handle = ops, handle
        self.t = dict(x=(dtype, (rows, ci)), y=(dtype, (rows, co)), w=(dtype, (groups, ci, co)), e=(I32, (groups,)))
        self.t.update({k: v for k, v in over.items() if k in self.t})
        self.null, self.shift, self.short = over.get("null", ()), over.get("shift", {}), over.get("short", 0)
        self.d = {k: (None if v is None else ops.TensorDesc(ARRAY, *v)) for k, v in self.t.items()}
        self.buf = (ctypes.c_char * 65536)()
        self.base = (ctypes.addressof(self.buf) + 255) // 256 * 256

    def ptr(self, name):
        if name in self.null or self.d.get(name, 0) is None:
            return None
        return ctypes.c_void_p(self.base + self.APART * "xywes".index(name) + self.shift.get(name, 0))

    def pairs(self, *names):
        return [a for n in names for a in (self.d[n], self.ptr(n))]

    def forward(self):
        return self.ops.lib().mluOpGroupedMatMulForward(self.handle.ptr, *self.pairs("x", "w", "e", "y"))

    def backward_input(self):
        return self.ops.lib().mluOpGroupedMatMulBackwardInput(self.handle.ptr, *self.pairs("y", "w", "e", "x"))

    def query(self):
        size = ctypes.c_size_t(0)
        st = self.ops.lib().mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(self.handle.ptr, self.d["x"], self.d["y"],
                                                                             self.d["w"], ctypes.byref(size))
        return st, size.value

    def backward_weight(self):
        size = max(self.query()[1] - self.short, 0)
        return self.ops.lib().mluOpGroupedMatMulBackwardWeight(self.handle.ptr, *self.pairs("x", "y", "e"), self.ptr("s"),
                                                               size, *self.pairs("w"))

    def all(self):
        return [self.forward(), self.backward_input(), self.backward_weight()]


@pytest.mark.parametrize("over", [{}, {"dtype": BF16}, {"dtype": FLOAT}, {"ci": 7, "co": 9}, {"groups": 1}, {"groups": 1024},
                                  {"rows": 1}, {"ci": 1, "co": 1}])
def test_valid_calls_reach_the_launch(ops, handle, over):
    c = Call(ops, handle, **over)
    assert c.query()[0] == ops.STATUS_SUCCESS
    assert c.all() == [ops.STATUS_EXECUTION_FAILED] * 3  # host-only: nothing can be launched


def test_float_weight_gradient(ops, handle):
    c = Call(ops, handle, w=(FLOAT, (3, 16, 24)))
    assert c.all() == [ops.STATUS_BAD_PARAM, ops.STATUS_BAD_PARAM, ops.STATUS_EXECUTION_FAILED]


def test_outputs_lie_on_no_input(ops, handle):
    at = "xywes".index
    for out, call, inputs in (("y", "forward", "xwe"), ("x", "backward_input", "ywe"), ("w", "backward_weight", "xye")):
        for name in inputs:
            for off in (0, 4):
                c = Call(ops, handle)
                c.shift = {out: c.APART * (at(name) - at(out)) + off}
                assert getattr(c, call)() == ops.STATUS_BAD_PARAM


def test_no_rows(ops, handle):
    c = Call(ops, handle, rows=0, null=("x", "y", "e"))
    assert c.forward() == ops.STATUS_SUCCESS and c.backward_input() == ops.STATUS_SUCCESS
    assert c.backward_weight() == ops.STATUS_EXECUTION_FAILED  # zeros have to be written


@pytest.mark.parametrize("over", [
    {"dtype": I32}, {"y": (FLOAT, (10, 24))}, {"w": (BF16, (3, 16, 24))}, {"x": (HALF, (10,))}, {"y": (HALF, (9, 24))},
    {"w": (HALF, (3, 24, 16))}, {"w": (HALF, (48, 24))}, {"e": (I64, (3,))}, {"e": (I32, (4,))}, {"e": (I32, (3, 1))},
    {"w": (HALF, (0, 16, 24)), "e": (I32, (0,))}, {"null": ("x",)}, {"null": ("y",)}, {"null": ("w",)}, {"null": ("e",)},
    {"shift": {"x": 1}}, {"shift": {"w": 1}}, {"shift": {"e": 2}}, {"shift": {"y": 1}}])
def test_bad_parameters(ops, handle, over):
    assert Call(ops, handle, **over).all() == [ops.STATUS_BAD_PARAM] * 3


def test_null_handle_and_descriptors(ops, handle):
    for name in "xywe":
        assert Call(ops, handle, **{name: None}).forward() == ops.STATUS_BAD_PARAM
        assert Call(ops, handle, **{name: None}).backward_input() == ops.STATUS_BAD_PARAM
    c = Call(ops, handle)
    lib, size = ops.lib(), ctypes.c_size_t(0)
    assert lib.mluOpGroupedMatMulForward(None, *c.pairs("x", "w", "e", "y")) == ops.STATUS_BAD_PARAM
    assert lib.mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(handle.ptr, c.d["x"], c.d["y"], None, ctypes.byref(size)) == ops.STATUS_BAD_PARAM
    assert lib.mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(handle.ptr, c.d["x"], c.d["y"], c.d["w"], None) == ops.STATUS_BAD_PARAM
    assert Call(ops, handle, null=("s",)).backward_weight() == ops.STATUS_BAD_PARAM
    assert Call(ops, handle, short=1).backward_weight() == ops.STATUS_BAD_PARAM


def test_limits(ops, handle):
    for over in ({"groups": 1025}, {"ci": 65544}, {"co": 65544}, {"rows": 1 << 31}, {"rows": (1 << 31) - 1, "co": 65536}):
        c = Call(ops, handle, **over)
        assert c.forward() == ops.STATUS_NOT_SUPPORTED
        assert c.query()[0] == ops.STATUS_NOT_SUPPORTED
    d = ops.TensorDesc(ARRAY, HALF, (10, 16))
    assert ops.lib().mluOpSetTensorDescriptorEx_v2(d.ptr, ARRAY, HALF, 2, ops.i64_array((10, 16)), ops.i64_array((32, 1))) == 0
    c = Call(ops, handle)
    c.d["x"] = d
    assert c.all() == [ops.STATUS_NOT_SUPPORTED] * 3


@pytest.mark.parametrize("rows,groups,ci,co", [(1, 1, 8, 8), (100000, 1, 64, 64), (65536, 32, 2048, 4096), (2000000, 27, 16, 16),
                                               (1 << 24, 1, 128, 128), (5000, 1024, 256, 256)])
def test_workspace_stays_within_its_bound(ops, handle, rows, groups, ci, co):
    for dtype in (HALF, FLOAT):
        st, size = Call(ops, handle, dtype=dtype, rows=rows, groups=groups, ci=ci, co=co).query()
        assert st == ops.STATUS_SUCCESS and size <= 160e6 + 256 * groups + 512


def test_wrappers_refuse(ops, handle):
    x, w, e = torch.zeros(10, 16), torch.zeros(3, 16, 24), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.grouped_matmul_forward(handle, torch.zeros(16, 10).t(), w, e)
    for bad in ((x, w, e.long()), (x, w.half(), e), (x, w[:, :8].contiguous(), e), (x, w, e[:2])):
        with pytest.raises(ops.MluOpError):
            ops.grouped_matmul_forward(handle, *bad)
    with pytest.raises(ops.MluOpError):
        ops.grouped_matmul_backward_input(handle, torch.zeros(10, 23), w, e)
    with pytest.raises(ops.MluOpError):
        ops.grouped_matmul_backward_weight(handle, x, torch.zeros(9, 24), e)
