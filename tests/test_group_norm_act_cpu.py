"""mluOpGroupNormActForward / Backward without a GPU: status codes of the C ABI and the
refusals of the Python wrappers (host-only handle, CPU tensors that no launch reaches)."""
import ctypes

import pytest
import torch

FLOAT, HALF, BF16, I32, ARRAY = 2, 1, 17, 6, 4


@pytest.fixture(scope="module")
def handle(ops):
    h = ops.Handle(0)
    yield h
    h.destroy()


class Call:
    """Arguments of a good call; `over` replaces descriptors (dtype, dims), None leaves one out."""

    def __init__(self, ops, handle, dtype=HALF, dims=(2, 5, 16), samples=2, groups=4, ends=False, **over):
        self.ops, self.handle, self.groups = ops, handle, groups
        self.buf = (ctypes.c_char * 262144)()
        self.base = (ctypes.addressof(self.buf) + 255) // 256 * 256
        c = dims[-1]
        self.t = dict(x=(dtype, dims), y=(dtype, dims), dy=(dtype, dims), dx=(dtype, dims), w=(FLOAT, (c,)), b=(FLOAT, (c,)),
                      dw=(FLOAT, (c,)), db=(FLOAT, (c,)), mean=(FLOAT, (samples, groups)), rstd=(FLOAT, (samples, groups)),
                      ends=(I32, (samples,)) if ends else None)
        self.eps, self.act = 1e-5, 1
        self.t.update({k: v for k, v in over.items() if k in self.t})
        self.eps, self.act = over.get("eps", self.eps), over.get("act", self.act)
        self.null, self.shift = over.get("null", ()), over.get("shift", {})
        self.short = over.get("short", 0)
        self.d = {k: (None if v is None else ops.TensorDesc(ARRAY, *v)) for k, v in self.t.items()}

    def ptr(self, name):
        if name in self.null or self.d[name] is None:
            return None
        return ctypes.c_void_p(self.base + 4096 * sorted(self.t).index(name) + self.shift.get(name, 0))

    def workspace(self, backward):
        size = ctypes.c_size_t(0)
        fn = "mluOpGetGroupNormAct%sWorkspaceSize" % ("Backward" if backward else "Forward")
        st = getattr(self.ops.lib(), fn)(self.handle.ptr, self.d["x"], self.d["ends"], self.groups, ctypes.byref(size))
        return st, size.value

    def pairs(self, *names):
        return [a for n in names for a in (self.d[n], self.ptr(n))]

    def forward(self):
        st, size = self.workspace(False)
        size -= self.short
        ws = None if "ws" in self.null else ctypes.c_void_p(self.base + 131072)
        return self.ops.lib().mluOpGroupNormActForward(self.handle.ptr, *self.pairs("x", "w", "b", "ends"), self.groups,
                                                       self.eps, self.act, ws, max(size, 0), *self.pairs("y", "mean", "rstd"))

    def backward(self):
        st, size = self.workspace(True)
        size -= self.short
        ws = None if "ws" in self.null else ctypes.c_void_p(self.base + 131072)
        return self.ops.lib().mluOpGroupNormActBackward(self.handle.ptr, *self.pairs("dy", "x", "w", "b", "ends", "mean", "rstd"),
                                                        self.groups, self.act, ws, max(size, 0),
                                                        *self.pairs("dx", "dw", "db"))


GOOD = [{}, {"dtype": FLOAT}, {"dtype": BF16, "act": 2}, {"act": 0, "w": None, "b": None}, {"dw": None, "db": None},
        {"dims": (7, 16), "ends": True}, {"dims": (7, 16), "samples": 7}, {"w": (HALF, (16,)), "b": (HALF, (16,))},
        {"dw": (HALF, (16,)), "db": (HALF, (16,))}, {"dims": (2, 3, 4, 5, 16)}, {"groups": 1}, {"groups": 16},
        {"dims": (0, 16), "ends": True}, {"dims": (2, 0, 16)}]


@pytest.mark.parametrize("over", GOOD)
def test_valid_calls_reach_the_launch(ops, handle, over):
    c = Call(ops, handle, **over)
    assert c.workspace(False)[0] == ops.STATUS_SUCCESS and c.workspace(True)[0] == ops.STATUS_SUCCESS
    assert c.forward() == ops.STATUS_EXECUTION_FAILED
    assert c.backward() == ops.STATUS_EXECUTION_FAILED


def test_nothing_to_do(ops, handle):
    c = Call(ops, handle, dims=(0, 16), samples=0, dw=None, db=None)
    assert c.forward() == ops.STATUS_SUCCESS and c.backward() == ops.STATUS_SUCCESS


BOTH = [{"dtype": I32}, {"dims": (16,)}, {"groups": 3}, {"groups": 0}, {"groups": 32}, {"act": 3}, {"act": -1},
        {"w": None}, {"b": None}, {"w": (FLOAT, (15,))}, {"w": (BF16, (16,)), "b": (BF16, (16,))},
        {"w": (HALF, (16,))}, {"mean": (HALF, (2, 4))}, {"rstd": (FLOAT, (4, 2))}, {"mean": (FLOAT, (8,))},
        {"dims": (2, 5, 16), "ends": True}, {"dims": (7, 16), "ends": True, "null": ("ends",)},
        {"null": ("x",)}, {"null": ("w",)}, {"null": ("b",)}, {"null": ("mean",)}, {"null": ("rstd",)},
        {"null": ("ws",), "dims": (2, 70000, 16)}, {"short": 1, "dims": (2, 70000, 16)}, {"shift": {"x": 1}}, {"shift": {"w": 2}}, {"shift": {"mean": 2}}]
FORWARD = [{"eps": 0.0}, {"eps": -1.0}, {"eps": float("nan")}, {"y": (FLOAT, (2, 5, 16))}, {"y": (HALF, (2, 16, 5))},
           {"null": ("y",)}, {"shift": {"y": 1}}]
BACKWARD = [{"dy": (FLOAT, (2, 5, 16))}, {"dy": (HALF, (10, 16))}, {"dx": (HALF, (2, 5, 8))}, {"null": ("dy",)}, {"null": ("dx",)},
            {"null": ("dw",)}, {"null": ("db",)}, {"dw": None}, {"db": (HALF, (16,))}, {"dw": (FLOAT, (2,)), "db": (FLOAT, (2,))},
            {"shift": {"db": 2}}]


@pytest.mark.parametrize("over", BOTH + FORWARD)
def test_forward_refuses(ops, handle, over):
    assert Call(ops, handle, **over).forward() == ops.STATUS_BAD_PARAM


@pytest.mark.parametrize("over", BOTH + BACKWARD)
def test_backward_refuses(ops, handle, over):
    assert Call(ops, handle, **over).backward() == ops.STATUS_BAD_PARAM


def test_few_rows_need_no_workspace(ops, handle):
    c = Call(ops, handle, dims=(2, 20, 16), null=("ws",))
    assert c.workspace(False) == (ops.STATUS_SUCCESS, 0) and c.workspace(True) == (ops.STATUS_SUCCESS, 0)
    assert c.forward() == ops.STATUS_EXECUTION_FAILED and c.backward() == ops.STATUS_EXECUTION_FAILED


def test_in_place_or_apart(ops, handle):
    size = 2 * 20 * 16 * 2
    for shift, want in ((0, ops.STATUS_EXECUTION_FAILED), (16, ops.STATUS_BAD_PARAM), (-16, ops.STATUS_BAD_PARAM),
                        (size, ops.STATUS_EXECUTION_FAILED), (size - 2, ops.STATUS_BAD_PARAM)):
        for name in ("x", "dy"):
            c = Call(ops, handle, dims=(2, 20, 16))
            out = ("y", "dx") if name == "x" else ("dx",)
            for o in out:
                c.shift = {o: 4096 * (sorted(c.t).index(name) - sorted(c.t).index(o)) + shift}
                assert (c.forward() if o == "y" else c.backward()) == want


def test_epsilon_is_positive_in_float(ops, handle):
    assert Call(ops, handle, eps=1e-50).forward() == ops.STATUS_BAD_PARAM
    assert Call(ops, handle, eps=1e39).forward() == ops.STATUS_BAD_PARAM


def test_null_handle_and_descriptors(ops, handle):
    lib, size = ops.lib(), ctypes.c_size_t(0)
    assert lib.mluOpGetGroupNormActForwardWorkspaceSize(None, None, None, 1, ctypes.byref(size)) == ops.STATUS_BAD_PARAM
    assert lib.mluOpGetGroupNormActBackwardWorkspaceSize(handle.ptr, None, None, 1, ctypes.byref(size)) == ops.STATUS_BAD_PARAM
    assert Call(ops, handle, x=None).forward() == ops.STATUS_BAD_PARAM
    for name in ("y", "mean", "rstd"):
        assert Call(ops, handle, **{name: None}).forward() == ops.STATUS_BAD_PARAM
    for name in ("dy", "x", "mean", "rstd", "dx"):
        assert Call(ops, handle, **{name: None}).backward() == ops.STATUS_BAD_PARAM


def test_large_and_strided_tensors_are_not_supported(ops, handle):
    c = Call(ops, handle, dims=(1 << 16, 1 << 15, 16), samples=1 << 16)
    assert c.workspace(False)[0] == ops.STATUS_NOT_SUPPORTED
    assert Call(ops, handle, dims=(2, 65544), groups=8).workspace(True)[0] == ops.STATUS_NOT_SUPPORTED
    d = ops.TensorDesc(ARRAY, HALF, (4, 16))
    assert ops.lib().mluOpSetTensorDescriptorEx_v2(d.ptr, ARRAY, HALF, 2, ops.i64_array((4, 16)), ops.i64_array((32, 1))) == 0
    size = ctypes.c_size_t(0)
    assert ops.lib().mluOpGetGroupNormActForwardWorkspaceSize(handle.ptr, d.ptr, None, 4, ctypes.byref(size)) == ops.STATUS_NOT_SUPPORTED


def test_wrappers_refuse(ops, handle):
    x, w, b = torch.zeros(2, 5, 16), torch.ones(16), torch.zeros(16)
    with pytest.raises(ValueError, match="activation"):
        ops.group_norm_act_forward(handle, x, w, b, 4, activation="gelu")
    with pytest.raises(ValueError, match="contiguous"):
        ops.group_norm_act_forward(handle, x.transpose(0, 1), w, b, 4)
    with pytest.raises(ops.MluOpError):
        ops.group_norm_act_forward(handle, x, w, None, 4)
    with pytest.raises(ops.MluOpError):
        ops.group_norm_act_forward(handle, x.double(), w, b, 4)
    m = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="contiguous"):
        ops.group_norm_act_backward(handle, x.transpose(0, 1), x, w, b, m, m, 4)
    with pytest.raises(ops.MluOpError):
        ops.group_norm_act_backward(handle, x[:1], x, w, b, m, m, 4)
