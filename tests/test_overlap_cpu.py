"""Outputs of the group norm and of the grouped products that lie on another tensor of the call, or on the workspace,
are refused before anything is launched (host-only handle, host memory that no launch reaches)."""
import ctypes

import pytest

FLOAT, HALF, I32, ARRAY = 2, 1, 6, 4


@pytest.fixture(scope="module")
def handle(ops):
    h = ops.Handle(0)
    yield h
    h.destroy()


class Call:
    """on={a: b}: tensor a lies on the last value of tensor b."""

    def __init__(self, ops, handle, specs, on):
        self.ops, self.handle = ops, handle
        self.buf = (ctypes.c_char * (1 << 21))()
        base = (ctypes.addressof(self.buf) + 255) // 256 * 256
        self.at, sizes = {}, {}
        for i, (name, spec) in enumerate(specs.items()):
            self.at[name] = base + (1 << 16) * i
            if spec is not None:
                n = {FLOAT: 4, HALF: 2, I32: 4}[spec[0]]
                for d in spec[1]:
                    n *= d
                sizes[name] = n
        self.d = {k: None if v is None else ops.TensorDesc(ARRAY, *v) for k, v in specs.items()}
        for a, b in on.items():
            self.at[a] = self.at[b] + (sizes[b] - 4 if b in sizes else 512)

    def pairs(self, *names):
        return [x for n in names for x in (self.d[n], ctypes.c_void_p(self.at[n]))]


def norm(ops, handle, backward, **on):
    dims, stats = (40, 16), (FLOAT, (2, 4))
    c = Call(ops, handle, dict(x=(HALF, dims), y=(HALF, dims), dy=(HALF, dims), w=(FLOAT, (16,)), b=(FLOAT, (16,)),
                               ends=(I32, (2,)), mean=stats, rstd=stats, dw=(FLOAT, (16,)), db=(FLOAT, (16,)), ws=None), on)
    size = ctypes.c_size_t(1 << 14)
    ws = [ctypes.c_void_p(c.at["ws"]), size]
    if backward:
        return ops.lib().mluOpGroupNormActBackward(handle.ptr, *c.pairs("dy", "x", "w", "b", "ends", "mean", "rstd"), 4, 1, *ws,
                                                   *c.pairs("y", "dw", "db"))
    return ops.lib().mluOpGroupNormActForward(handle.ptr, *c.pairs("x", "w", "b", "ends"), 4, 1e-5, 1, *ws,
                                              *c.pairs("y", "mean", "rstd"))


FORWARD = [(a, b) for a in ("y", "mean", "rstd") for b in ("x", "w", "b", "ends", "y", "mean", "rstd", "ws") if a != b]
BACKWARD = [(a, b) for a in ("y", "dw", "db") for b in ("dy", "x", "w", "b", "ends", "mean", "rstd", "y", "dw", "db", "ws") if a != b]


def test_apart_reaches_the_launch(ops, handle):
    for backward in (False, True):
        assert norm(ops, handle, backward) == ops.STATUS_EXECUTION_FAILED


@pytest.mark.parametrize("a,b", FORWARD)
def test_norm_forward(ops, handle, a, b):
    assert norm(ops, handle, False, **{a: b}) == ops.STATUS_BAD_PARAM


@pytest.mark.parametrize("a,b", BACKWARD)
def test_norm_backward(ops, handle, a, b):
    assert norm(ops, handle, True, **{a: b}) == ops.STATUS_BAD_PARAM


def weight_gradient(ops, handle, **on):
    c = Call(ops, handle, dict(x=(HALF, (40, 16)), dy=(HALF, (40, 24)), ends=(I32, (3,)), dw=(FLOAT, (3, 16, 24)), ws=None), on)
    return ops.lib().mluOpGroupedMatMulBackwardWeight(handle.ptr, *c.pairs("x", "dy", "ends"), ctypes.c_void_p(c.at["ws"]),
                                                      ctypes.c_size_t(1 << 14), *c.pairs("dw"))


def test_workspace_of_the_weight_gradient(ops, handle):
    assert weight_gradient(ops, handle) == ops.STATUS_EXECUTION_FAILED
    for a, b in (("dw", "ws"), ("x", "ws"), ("dy", "ws"), ("ends", "ws"), ("dw", "x"), ("dw", "dy"), ("dw", "ends")):
        assert weight_gradient(ops, handle, **{a: b}) == ops.STATUS_BAD_PARAM, (a, b)
