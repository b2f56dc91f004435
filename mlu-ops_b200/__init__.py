"""Python harness over the C ABI of libmluops_b200.so.

The product is the shared library (include/mlu_op.h); this package only loads
it with ctypes and wraps the calls so that tests, the benchmark and the
backbone driver can pass torch CUDA tensors.  Function and argument names
follow the reference's C API.  There is no CPU fallback: if the library has not
been built, loading raises.
"""
import array
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libmluops_b200.so")

# mluOpStatus_t
STATUS_SUCCESS = 0
STATUS_NOT_INITIALIZED = 1
STATUS_ALLOC_FAILED = 2
STATUS_BAD_PARAM = 3
STATUS_INTERNAL_ERROR = 4
STATUS_ARCH_MISMATCH = 5
STATUS_EXECUTION_FAILED = 6
STATUS_NOT_SUPPORTED = 7
STATUS_NUMERICAL_OVERFLOW = 8

# mluOpTensorLayout_t
LAYOUT_NCHW, LAYOUT_NHWC, LAYOUT_HWCN, LAYOUT_NDHWC, LAYOUT_ARRAY, LAYOUT_NCDHW = 0, 1, 2, 3, 4, 5
# mluOpDataType_t
DTYPE_INVALID, DTYPE_HALF, DTYPE_FLOAT, DTYPE_INT16, DTYPE_INT32, DTYPE_INT64 = 0, 1, 2, 4, 6, 9
DTYPE_UINT8, DTYPE_BFLOAT16 = 7, 17
# mluOpAdamWRounding_t
ADAMW_ROUNDINGS = {"nearest": 0, "stochastic": 1}
# mluOpGroupNormAct_t
GROUP_NORM_ACTS = {"none": 0, "relu": 1, "silu": 2}

_vp = ctypes.c_void_p
_int = ctypes.c_int
_i64 = ctypes.c_int64
_szt = ctypes.c_size_t
_intp = ctypes.POINTER(ctypes.c_int)
_i64p = ctypes.POINTER(ctypes.c_int64)

# name -> (restype, argtypes); exactly the entry points include/mlu_op.h and include/mlu_op_trace.h declare
SIGNATURES = {
    "mluOpCreate": (_int, [ctypes.POINTER(_vp)]),
    "mluOpDestroy": (_int, [_vp]),
    "mluOpSetQueue": (_int, [_vp, _vp]),
    "mluOpGetQueue": (_int, [_vp, ctypes.POINTER(_vp)]),
    "mluOpGetDevice": (_int, [_vp, _intp]),
    "mluOpGetErrorString": (ctypes.c_char_p, [_int]),
    "mluOpGetSizeOfDataType": (_int, [_int, ctypes.POINTER(_szt)]),
    "mluOpGetLibVersion": (None, [_intp, _intp, _intp]),
    "mluOpSetAtomicsMode": (_int, [_vp, _int]),
    "mluOpGetAtomicsMode": (_int, [_vp, _intp]),
    "mluOpCreateTensorDescriptor": (_int, [ctypes.POINTER(_vp)]),
    "mluOpSetTensorDescriptor": (_int, [_vp, _int, _int, _int, _intp]),
    "mluOpSetTensorDescriptor_v2": (_int, [_vp, _int, _int, _int, _i64p]),
    "mluOpSetTensorDescriptorEx": (_int, [_vp, _int, _int, _int, _intp, _intp]),
    "mluOpSetTensorDescriptorEx_v2": (_int, [_vp, _int, _int, _int, _i64p, _i64p]),
    "mluOpResetTensorDescriptor": (_int, [_vp]),
    "mluOpGetTensorDescriptor": (_int, [_vp, _intp, _intp, _intp, _intp]),
    "mluOpGetTensorDescriptor_v2": (_int, [_vp, _intp, _intp, _intp, _i64p]),
    "mluOpGetTensorDescriptorEx": (_int, [_vp, _intp, _intp, _intp, _intp, _intp]),
    "mluOpGetTensorElementNum": (ctypes.c_uint64, [_vp]),
    "mluOpDestroyTensorDescriptor": (_int, [_vp]),
    "mluOpCreateSparseConvolutionDescriptor": (_int, [ctypes.POINTER(_vp)]),
    "mluOpDestroySparseConvolutionDescriptor": (_int, [_vp]),
    "mluOpSetSparseConvolutionDescriptor": (_int, [_vp, _int, _int, _intp, _intp, _intp, _intp, _intp, _intp,
                                                  _int, _int, _int]),
    "mluOpGetSparseConvolutionNumActOut": (_int, [_vp, _intp]),
    "mluOpGetIndicePairsWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, ctypes.POINTER(_szt)]),
    "mluOpGetIndicePairs": (_int, [_vp, _vp, _vp, _vp, _vp, _szt, _vp, _vp, _vp, _vp, _vp, _vp]),
    "mluOpGetIndicePairsWithNeighbourTable": (_int, [_vp, _vp, _vp, _vp, _vp, _szt, _vp, _vp, _vp, _vp, _vp, _vp,
                                                    _vp, _szt]),
    "mluOpGetIndiceConvolutionForwardWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64, _i64,
                                                            ctypes.POINTER(_szt)]),
    "mluOpIndiceConvolutionForward": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64, _i64, _vp,
                                            _szt, _vp, _vp]),
    "mluOpIndiceConvolutionForwardBuiltinWorkspace": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64,
                                                            _i64, _vp, _vp]),
    "mluOpGetIndiceConvolutionBackwardDataWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _i64p, _i64,
                                                                 ctypes.POINTER(_szt)]),
    "mluOpIndiceConvolutionBackwardData": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64, _vp, _szt,
                                                 _vp, _vp]),
    "mluOpGetIndiceConvolutionBackwardFilterWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64,
                                                                   ctypes.POINTER(_szt)]),
    "mluOpIndiceConvolutionBackwardFilter": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64, _vp,
                                                   _szt, _vp, _vp]),
    "mluOpGetIndiceNeighbourTableSize": (_int, [_vp, _vp, _i64, ctypes.POINTER(_szt)]),
    "mluOpBuildIndiceNeighbourTable": (_int, [_vp, _vp, _vp, _i64p, _i64, _vp, _szt]),
    "mluOpGetIndiceConvolutionForwardFromTableWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _i64p, _i64, _i64,
                                                                     _i64, ctypes.POINTER(_szt)]),
    "mluOpIndiceConvolutionForwardFromTable": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _szt, _i64p, _i64, _i64,
                                                     _i64, _vp, _szt, _vp, _vp]),
    "mluOpGetIndiceInputNeighbourTableSize": (_int, [_vp, _vp, ctypes.POINTER(_szt)]),
    "mluOpBuildIndiceInputNeighbourTable": (_int, [_vp, _vp, _vp, _i64p, _i64, _vp, _szt]),
    "mluOpGetIndiceConvolutionBackwardDataFromTableWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, _vp, _i64p, _i64,
                                                                          ctypes.POINTER(_szt)]),
    "mluOpIndiceConvolutionBackwardDataFromTable": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _szt, _i64p, _i64,
                                                          _i64, _vp, _szt, _vp, _vp]),
    "mluOpIndiceConvolutionBackwardDataFromForwardTable": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _szt, _i64p,
                                                                 _i64, _i64, _vp, _szt, _vp, _vp]),
    "mluOpIndiceConvolutionBackwardFilterFromTable": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _szt, _i64p, _i64,
                                                            _i64, _vp, _szt, _vp, _vp]),
    "mluOpGetVoxelizationWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, ctypes.c_int32, ctypes.c_int32,
                                                ctypes.c_int32, ctypes.c_bool, _vp, _vp, _vp, _vp,
                                                ctypes.POINTER(_szt)]),
    "mluOpVoxelization": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                ctypes.c_bool, _vp, _szt, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "mluOpGetDynamicPointToVoxelForwardWorkspaceSize": (_int, [_vp, _vp, _vp, ctypes.POINTER(_szt)]),
    "mluOpDynamicPointToVoxelForward": (_int, [_vp, _int, _vp, _vp, _vp, _vp, _vp, _szt, _vp, _vp, _vp, _vp, _vp, _vp,
                                              _vp, _vp, _vp, _vp]),
    "mluOpGetDynamicPointToVoxelBackwardWorkspaceSize": (_int, [_vp, _int, _vp, _vp, _vp, _vp, _vp, _vp,
                                                               ctypes.POINTER(_szt)]),
    "mluOpDynamicPointToVoxelBackward": (_int, [_vp, _int, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                               _vp, _szt, _vp, _vp]),
    "mluOpMultiTensorAdamW": (_int, [_vp, _int, _int, _int, _i64] + [_vp] * 7 + [ctypes.c_double] * 5 + [_i64, _vp, _vp]),
    "mluOpMultiTensorAdamW_v2": (_int, [_vp, _int, _int, _int, _i64] + [_vp] * 7 + [ctypes.c_double] * 5 + [_i64, _vp, _vp, _int, _vp]),
    "mluOpGetGroupNormActForwardWorkspaceSize": (_int, [_vp, _vp, _vp, _i64, ctypes.POINTER(_szt)]),
    "mluOpGroupNormActForward": (_int, [_vp] * 9 + [_i64, ctypes.c_double, _int, _vp, _szt] + [_vp] * 6),
    "mluOpGetGroupNormActBackwardWorkspaceSize": (_int, [_vp, _vp, _vp, _i64, ctypes.POINTER(_szt)]),
    "mluOpGroupNormActBackward": (_int, [_vp] * 15 + [_i64, _int, _vp, _szt] + [_vp] * 6),
    "mluOpGroupedMatMulForward": (_int, [_vp] * 9),
    "mluOpGroupedMatMulBackwardInput": (_int, [_vp] * 9),
    "mluOpGetGroupedMatMulBackwardWeightWorkspaceSize": (_int, [_vp, _vp, _vp, _vp, ctypes.POINTER(_szt)]),
    "mluOpGroupedMatMulBackwardWeight": (_int, [_vp] * 8 + [_szt, _vp, _vp]),
    # include/mlu_op_trace.h
    "mluOpTraceKernelEnable": (_int, [_int]),
    "mluOpTraceKernelReset": (_int, []),
    "mluOpTraceKernelReport": (_int, [ctypes.c_char_p, _szt, ctypes.POINTER(_szt)]),
}

_lib = None


def lib():
    """The loaded C-ABI library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.isfile(LIB_PATH):
            raise RuntimeError(
                "libmluops_b200.so is missing (%s); build it with `python mlu-ops_b200/build.py`. "
                "There is no fallback path." % LIB_PATH)
        _lib = ctypes.CDLL(LIB_PATH)
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(_lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
    return _lib


class MluOpError(RuntimeError):
    def __init__(self, call, status):
        self.status = status
        name = lib().mluOpGetErrorString(status).decode()
        super().__init__("%s returned %s (%d)" % (call, name, status))


def check(call, status):
    if status != STATUS_SUCCESS:
        raise MluOpError(call, status)


def int_array(values):
    return (ctypes.c_int * len(values))(*[int(v) for v in values])


def i64_array(values):
    return (ctypes.c_int64 * len(values))(*[int(v) for v in values])


class Handle:
    """mluOpHandle_t bound to a CUDA stream (raw cudaStream_t integer, 0 = default)."""

    def __init__(self, stream=0):
        self.ptr = _vp()
        check("mluOpCreate", lib().mluOpCreate(ctypes.byref(self.ptr)))
        device = ctypes.c_int(-1)
        check("mluOpGetDevice", lib().mluOpGetDevice(self.ptr, ctypes.byref(device)))
        self.device = device.value  # CUDA device ordinal, -1 for a host-only handle
        self.plans = {}  # descriptors and workspace sizes of the calls seen, by types and shapes
        self.set_queue(stream)

    def set_queue(self, stream):
        check("mluOpSetQueue", lib().mluOpSetQueue(self.ptr, _vp(stream)))
        self.stream = stream

    def destroy(self):
        if self.ptr:
            check("mluOpDestroy", lib().mluOpDestroy(self.ptr))
            self.ptr = _vp()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class TensorDesc:
    """mluOpTensorDescriptor_t with contiguous strides."""

    def __init__(self, layout, dtype, dims):
        self.ptr = _vp()
        check("mluOpCreateTensorDescriptor", lib().mluOpCreateTensorDescriptor(ctypes.byref(self.ptr)))
        check("mluOpSetTensorDescriptor_v2",
              lib().mluOpSetTensorDescriptor_v2(self.ptr, layout, dtype, len(dims), i64_array(dims)))
        self.dims = tuple(int(d) for d in dims)
        self._as_parameter_ = self.ptr  # the object itself can be handed to a call

    def destroy(self):
        if self.ptr:
            lib().mluOpDestroyTensorDescriptor(self.ptr)
            self.ptr = _vp()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class SparseConvDesc:
    """mluOpSparseConvolutionDescriptor_t; the three-element lists are (D, H, W)."""

    def __init__(self, batch, pad, stride, dilation, input_space, filter_space, output_space, sub_m):
        self.ptr = _vp()
        check("mluOpCreateSparseConvolutionDescriptor",
              lib().mluOpCreateSparseConvolutionDescriptor(ctypes.byref(self.ptr)))
        check("mluOpSetSparseConvolutionDescriptor",
              lib().mluOpSetSparseConvolutionDescriptor(
                  self.ptr, 5, int(batch), int_array(pad), int_array(stride), int_array(dilation),
                  int_array(input_space), int_array(filter_space), int_array(output_space), int(bool(sub_m)),
                  0, 0))
        self.batch = int(batch)
        self.pad, self.stride, self.dilation = list(pad), list(stride), list(dilation)
        self.input_space, self.filter_space = list(input_space), list(filter_space)
        self.output_space, self.sub_m = list(output_space), int(bool(sub_m))

    @property
    def kernel_volume(self):
        return self.filter_space[0] * self.filter_space[1] * self.filter_space[2]

    def num_act_out(self):
        n = ctypes.c_int(0)
        check("mluOpGetSparseConvolutionNumActOut",
              lib().mluOpGetSparseConvolutionNumActOut(self.ptr, ctypes.byref(n)))
        return n.value

    def destroy(self):
        if self.ptr:
            lib().mluOpDestroySparseConvolutionDescriptor(self.ptr)
            self.ptr = _vp()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def output_space(input_space, pad, stride, dilation, filter_space):
    """o = (i + 2p - d(k-1) - 1)/s + 1 per dim: the size callers pass as output_space."""
    return [(i + 2 * p - d * (k - 1) - 1) // s + 1
            for i, p, s, d, k in zip(input_space, pad, stride, dilation, filter_space)]


def _ptr(t):
    return _vp(t.data_ptr() if t is not None else 0)


class Guards:
    """Poisoned bands around every buffer the harness allocates for a call (outputs and
    workspace), checked after the call: a kernel that writes outside the buffer it was given
    is caught even when the stray write lands in memory nobody reads.  The reference's own
    harness brackets each device buffer with a mask the same way
    (test/mlu_op_gtest/pb_gtest/src/runtime.cpp:86-145); it stands in for a memory checker.

        with ops.guarded() as guards:
            ... calls through this module ...
        # leaving the block synchronises and asserts that every band is intact
    """
    BAND = 1024  # bytes before and after; a multiple of the 256-byte alignment the library assumes

    def __init__(self):
        self.items = []

    def empty(self, shape, dtype, device):
        import torch
        shape = tuple(int(v) for v in shape)
        count = 1
        for v in shape:
            count *= v
        nbytes = count * torch.empty((), dtype=dtype).element_size()
        raw = torch.empty((2 * self.BAND + nbytes,), dtype=torch.uint8, device=device)
        gen = torch.Generator(device="cpu").manual_seed(len(self.items) + 1)
        band = torch.randint(0, 256, (2 * self.BAND,), dtype=torch.uint8, generator=gen).to(device)
        raw[:self.BAND] = band[:self.BAND]
        raw[self.BAND + nbytes:] = band[self.BAND:]
        self.items.append((raw, nbytes, band))
        return raw[self.BAND:self.BAND + nbytes].view(dtype).view(shape)

    def check(self):
        import torch
        torch.cuda.synchronize()
        for i, (raw, nbytes, band) in enumerate(self.items):
            assert torch.equal(raw[:self.BAND], band[:self.BAND]), "buffer %d: bytes before it were overwritten" % i
            assert torch.equal(raw[self.BAND + nbytes:], band[self.BAND:]), \
                "buffer %d (%d bytes): bytes after it were overwritten" % (i, nbytes)
        return len(self.items)


_guards = None


class guarded:
    """Context manager: allocations of this module get guard bands inside the block."""

    def __enter__(self):
        global _guards
        self.previous, _guards = _guards, Guards()
        return _guards

    def __exit__(self, exc_type, exc, tb):
        global _guards
        mine, _guards = _guards, self.previous
        if exc_type is None:
            mine.check()
        return False


def _alloc(shape, dtype, device):
    import torch
    if _guards is not None:
        return _guards.empty(shape, dtype, device)
    return torch.empty(tuple(shape), dtype=dtype, device=device)


def get_indice_pairs_workspace_size(handle, conv, indices_desc, pairs_desc, out_indices_desc, num_desc):
    size = _szt(0)
    check("mluOpGetIndicePairsWorkspaceSize",
          lib().mluOpGetIndicePairsWorkspaceSize(handle.ptr, conv.ptr, indices_desc.ptr, pairs_desc.ptr,
                                                 out_indices_desc.ptr, num_desc.ptr, ctypes.byref(size)))
    return size.value


def max_active_outputs(L, batch, output_space, filter_space, stride, dilation):
    """Upper bound on the active outputs of a default-mode rulebook with L inputs: an input
    reaches an output through offset k only when (i + pad - k*dilation) is a multiple of the
    stride, so per dimension at most ceil(kernel / (stride / gcd(stride, dilation))) offsets
    can be valid for one input (2 of 3 for a 3-wide kernel at stride 2).  Callers size
    out_indices by it instead of by the whole output grid."""
    import math
    per_input = 1
    for k, s, d in zip(filter_space, stride, dilation):
        period = s // math.gcd(s, d)
        per_input *= -(-k // period)
    cells = batch * output_space[0] * output_space[1] * output_space[2]
    return max(1, min(L * per_input, cells))


def get_indice_pairs(handle, conv, indices, out_rows=None, workspace=None, with_table=False):
    """Rulebook of one layer through mluOpGetIndicePairs.

    indices: int32 CUDA tensor [L,4].  Returns (indice_pairs [K,2,L], out_indices
    [out_rows,4], indice_num [K] (device), num_act_out (host int)); with_table the call
    goes through mluOpGetIndicePairsWithNeighbourTable and the table (int32 [K, rows padded
    to 512]) is appended to the result.
    """
    import torch
    L = indices.shape[0]
    K = conv.kernel_volume
    if out_rows is None:
        out_rows = L if conv.sub_m else max_active_outputs(L, conv.batch, conv.output_space, conv.filter_space,
                                                           conv.stride, conv.dilation)
    dev = indices.device
    pairs = _alloc((K, 2, L), torch.int32, dev)
    out_indices = _alloc((out_rows, 4), torch.int32, dev)
    num = _alloc((K,), torch.int32, dev)
    d_in = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (L, 4))
    d_pairs = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    d_out = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (out_rows, 4))
    d_num = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K,))
    ws_size = get_indice_pairs_workspace_size(handle, conv, d_in, d_pairs, d_out, d_num)
    if workspace is None or workspace.numel() < ws_size:
        workspace = _alloc((max(ws_size, 1),), torch.uint8, dev)
    args = [handle.ptr, conv.ptr, d_in.ptr, _ptr(indices), _ptr(workspace), ws_size, d_pairs.ptr, _ptr(pairs),
            d_out.ptr, _ptr(out_indices), d_num.ptr, _ptr(num)]
    table = None
    try:
        if with_table:
            size = _szt(0)
            check("mluOpGetIndiceNeighbourTableSize",
                  lib().mluOpGetIndiceNeighbourTableSize(handle.ptr, d_pairs.ptr, L, ctypes.byref(size)))
            table = _alloc((K, size.value // (4 * K)), torch.int32, dev)
            check("mluOpGetIndicePairsWithNeighbourTable",
                  lib().mluOpGetIndicePairsWithNeighbourTable(*args, _ptr(table), size.value))
        else:
            check("mluOpGetIndicePairs", lib().mluOpGetIndicePairs(*args))
    finally:
        for d in (d_in, d_pairs, d_out, d_num):
            d.destroy()
    n_out = conv.num_act_out()
    if with_table:
        return pairs, out_indices, num, n_out, table
    return pairs, out_indices, num, n_out


def build_neighbour_table(handle, indice_pairs, indice_num, num_act_out):
    """The neighbour table of a rulebook from its pair lists (mluOpBuildIndiceNeighbourTable):
    int32 [K, rows padded to 512]."""
    import torch
    K, _, L = indice_pairs.shape
    d_pairs = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    size = _szt(0)
    try:
        check("mluOpGetIndiceNeighbourTableSize",
              lib().mluOpGetIndiceNeighbourTableSize(handle.ptr, d_pairs.ptr, num_act_out, ctypes.byref(size)))
        table = _alloc((K, size.value // (4 * K)), torch.int32, indice_pairs.device)
        check("mluOpBuildIndiceNeighbourTable",
              lib().mluOpBuildIndiceNeighbourTable(handle.ptr, d_pairs.ptr, _ptr(indice_pairs),
                                                   i64_array([int(v) for v in indice_num]), num_act_out,
                                                   _ptr(table), size.value))
    finally:
        d_pairs.destroy()
    return table


def build_input_neighbour_table(handle, indice_pairs, indice_num, num_act_out):
    """The table the input gradient works from (mluOpBuildIndiceInputNeighbourTable): for every
    kernel offset and input row the output row it feeds, int32 [K, L padded to 512]."""
    import torch
    K, _, L = indice_pairs.shape
    d_pairs = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    size = _szt(0)
    try:
        check("mluOpGetIndiceInputNeighbourTableSize",
              lib().mluOpGetIndiceInputNeighbourTableSize(handle.ptr, d_pairs.ptr, ctypes.byref(size)))
        table = _alloc((K, size.value // (4 * K)), torch.int32, indice_pairs.device)
        check("mluOpBuildIndiceInputNeighbourTable",
              lib().mluOpBuildIndiceInputNeighbourTable(handle.ptr, d_pairs.ptr, _ptr(indice_pairs),
                                                        i64_array([int(v) for v in indice_num]), num_act_out,
                                                        _ptr(table), size.value))
    finally:
        d_pairs.destroy()
    return table


FILTER_LAYOUTS = {"ARRAY": LAYOUT_ARRAY, "NDHWC": LAYOUT_NDHWC, "NCDHW": LAYOUT_NCDHW,
                  "HWCN": LAYOUT_HWCN, "NHWC": LAYOUT_NHWC, "NCHW": LAYOUT_NCHW}


def filter_dims(layout, filter_space, ci, co):
    kd, kh, kw = filter_space
    if layout == "ARRAY":
        return (kd, kh, kw, ci, co)
    if layout == "NDHWC":
        return (co, kd, kh, kw, ci)
    if layout == "NCDHW":
        return (co, ci, kd, kh, kw)
    raise ValueError(layout)


def indice_convolution_forward(handle, features, filters, filter_layout, filter_space, indice_pairs,
                               indice_num_host, num_act_out, sub_m, workspace=None, out=None, table=None):
    """features_out [num_act_out, Co] through mluOpIndiceConvolutionForward.

    features [L,Ci] and filters (5-D, in `filter_layout`) are CUDA tensors of the
    same dtype (float16 or float32); indice_num_host is a sequence of K ints.  table: the
    rulebook's neighbour table (build_neighbour_table); with it the call is
    mluOpIndiceConvolutionForwardFromTable and indice_pairs only gives the shapes.
    """
    import torch
    L, ci = features.shape
    dims = tuple(filters.shape)
    co = dims[4] if filter_layout == "ARRAY" else dims[0]
    K = indice_pairs.shape[0]
    dt = DTYPE_HALF if features.dtype == torch.float16 else DTYPE_FLOAT
    dev = features.device
    if out is None:
        out = _alloc((num_act_out, co), features.dtype, dev)
    d_f = TensorDesc(LAYOUT_ARRAY, dt, (L, ci))
    d_w = TensorDesc(FILTER_LAYOUTS[filter_layout], dt, dims)
    d_p = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    d_o = TensorDesc(LAYOUT_ARRAY, dt, (num_act_out, co))
    num = i64_array(indice_num_host)
    size = _szt(0)
    if table is not None:
        check("mluOpGetIndiceConvolutionForwardFromTableWorkspaceSize",
              lib().mluOpGetIndiceConvolutionForwardFromTableWorkspaceSize(handle.ptr, d_f.ptr, d_w.ptr, d_p.ptr,
                                                                           d_o.ptr, num, num_act_out, 0,
                                                                           int(bool(sub_m)), ctypes.byref(size)))
        if workspace is None or workspace.numel() < size.value:
            workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
        check("mluOpIndiceConvolutionForwardFromTable",
              lib().mluOpIndiceConvolutionForwardFromTable(handle.ptr, d_f.ptr, _ptr(features), d_w.ptr,
                                                           _ptr(filters), d_p.ptr, _ptr(table), table.numel() * 4,
                                                           num, num_act_out, 0, int(bool(sub_m)), _ptr(workspace),
                                                           size.value, d_o.ptr, _ptr(out)))
        for d in (d_f, d_w, d_p, d_o):
            d.destroy()
        return out
    check("mluOpGetIndiceConvolutionForwardWorkspaceSize",
          lib().mluOpGetIndiceConvolutionForwardWorkspaceSize(handle.ptr, d_f.ptr, d_w.ptr, d_p.ptr, d_o.ptr,
                                                              num, num_act_out, 0, int(bool(sub_m)),
                                                              ctypes.byref(size)))
    if workspace is None or workspace.numel() < size.value:
        workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    check("mluOpIndiceConvolutionForward",
          lib().mluOpIndiceConvolutionForward(handle.ptr, d_f.ptr, _ptr(features), d_w.ptr, _ptr(filters),
                                              d_p.ptr, _ptr(indice_pairs), num, num_act_out, 0,
                                              int(bool(sub_m)), _ptr(workspace), size.value, d_o.ptr,
                                              _ptr(out)))
    for d in (d_f, d_w, d_p, d_o):
        d.destroy()
    return out


def indice_convolution_backward_data(handle, output_grad, filters, filter_layout, indice_pairs,
                                     indice_num_host, sub_m, workspace=None, out=None, table=None,
                                     forward_table=None):
    """input_grad [L, Ci] through mluOpIndiceConvolutionBackwardData.

    output_grad [N_out,Co] and filters (4-D or 5-D, in `filter_layout`: ARRAY, HWCN,
    NDHWC, NCDHW, NHWC, NCHW) are CUDA tensors of the same dtype; L is indice_pairs'
    last dimension; indice_num_host is a sequence of K ints.  table: the rulebook's input
    neighbour table (build_input_neighbour_table); with it the call is
    mluOpIndiceConvolutionBackwardDataFromTable and indice_pairs only gives the shapes.
    forward_table: the FORWARD table of a submanifold rulebook with centred padding; tried first
    (mluOpIndiceConvolutionBackwardDataFromForwardTable), NOT_SUPPORTED falls through to the rest;
    a callable is called for `table` only then.
    """
    import torch
    n_out, co = output_grad.shape
    dims = tuple(filters.shape)
    if filter_layout in ("ARRAY", "HWCN"):
        ci = dims[-2]
    elif filter_layout in ("NDHWC", "NHWC"):
        ci = dims[-1]
    else:
        ci = dims[1]
    K, _, L = indice_pairs.shape
    dt = DTYPE_HALF if output_grad.dtype == torch.float16 else DTYPE_FLOAT
    dev = output_grad.device
    if out is None:
        out = _alloc((L, ci), output_grad.dtype, dev)
    d_g = TensorDesc(LAYOUT_ARRAY, dt, (n_out, co))
    d_w = TensorDesc(FILTER_LAYOUTS[filter_layout], dt, dims)
    d_p = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    d_o = TensorDesc(LAYOUT_ARRAY, dt, (L, ci))
    num = i64_array(indice_num_host)
    size = _szt(0)
    if forward_table is not None and sub_m:
        check("mluOpGetIndiceConvolutionBackwardDataFromTableWorkspaceSize",
              lib().mluOpGetIndiceConvolutionBackwardDataFromTableWorkspaceSize(handle.ptr, d_g.ptr, d_w.ptr, d_p.ptr,
                                                                                d_o.ptr, num, 0, ctypes.byref(size)))
        if workspace is None or workspace.numel() < size.value:
            workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
        st = lib().mluOpIndiceConvolutionBackwardDataFromForwardTable(
            handle.ptr, d_g.ptr, _ptr(output_grad), d_w.ptr, _ptr(filters), d_p.ptr, _ptr(forward_table),
            forward_table.numel() * 4, num, 0, 1, _ptr(workspace), size.value, d_o.ptr, _ptr(out))
        if st != STATUS_NOT_SUPPORTED:
            check("mluOpIndiceConvolutionBackwardDataFromForwardTable", st)
            for d in (d_g, d_w, d_p, d_o):
                d.destroy()
            return out
    if callable(table):
        table = table()
    if table is not None:
        check("mluOpGetIndiceConvolutionBackwardDataFromTableWorkspaceSize",
              lib().mluOpGetIndiceConvolutionBackwardDataFromTableWorkspaceSize(handle.ptr, d_g.ptr, d_w.ptr, d_p.ptr,
                                                                                d_o.ptr, num, 0, ctypes.byref(size)))
        if workspace is None or workspace.numel() < size.value:
            workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
        check("mluOpIndiceConvolutionBackwardDataFromTable",
              lib().mluOpIndiceConvolutionBackwardDataFromTable(handle.ptr, d_g.ptr, _ptr(output_grad), d_w.ptr,
                                                                _ptr(filters), d_p.ptr, _ptr(table),
                                                                table.numel() * 4, num, 0, int(bool(sub_m)),
                                                                _ptr(workspace), size.value, d_o.ptr, _ptr(out)))
        for d in (d_g, d_w, d_p, d_o):
            d.destroy()
        return out
    check("mluOpGetIndiceConvolutionBackwardDataWorkspaceSize",
          lib().mluOpGetIndiceConvolutionBackwardDataWorkspaceSize(handle.ptr, d_g.ptr, d_w.ptr, d_p.ptr, d_o.ptr,
                                                                   num, 0, ctypes.byref(size)))
    if workspace is None or workspace.numel() < size.value:
        workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    check("mluOpIndiceConvolutionBackwardData",
          lib().mluOpIndiceConvolutionBackwardData(handle.ptr, d_g.ptr, _ptr(output_grad), d_w.ptr, _ptr(filters),
                                                   d_p.ptr, _ptr(indice_pairs), num, 0, int(bool(sub_m)),
                                                   _ptr(workspace), size.value, d_o.ptr, _ptr(out)))
    for d in (d_g, d_w, d_p, d_o):
        d.destroy()
    return out


def indice_convolution_backward_filter(handle, features, output_grad, filter_space, indice_pairs,
                                       indice_num_host, sub_m, workspace=None, out=None, table=None,
                                     forward_table=None):
    """filters_grad [kd,kh,kw,Ci,Co] through mluOpIndiceConvolutionBackwardFilter.

    features [L,Ci] and output_grad [N_out,Co] are CUDA tensors of the same dtype;
    indice_num_host is a sequence of K = kd*kh*kw ints.  table: the rulebook's FORWARD
    neighbour table; with it the call is mluOpIndiceConvolutionBackwardFilterFromTable where the
    shapes allow it (STATUS_NOT_SUPPORTED falls back to the reference-shaped call).
    """
    import torch
    L, ci = features.shape
    n_out, co = output_grad.shape
    K = indice_pairs.shape[0]
    dt = DTYPE_HALF if features.dtype == torch.float16 else DTYPE_FLOAT
    dev = features.device
    dims = tuple(filter_space) + (ci, co)
    if out is None:
        out = _alloc(dims, features.dtype, dev)
    d_f = TensorDesc(LAYOUT_ARRAY, dt, (L, ci))
    d_g = TensorDesc(LAYOUT_ARRAY, dt, (n_out, co))
    d_p = TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (K, 2, L))
    d_w = TensorDesc(LAYOUT_ARRAY, dt, dims)
    num = i64_array(indice_num_host)
    size = _szt(0)
    check("mluOpGetIndiceConvolutionBackwardFilterWorkspaceSize",
          lib().mluOpGetIndiceConvolutionBackwardFilterWorkspaceSize(handle.ptr, d_f.ptr, d_g.ptr, d_p.ptr,
                                                                     d_w.ptr, num, 0, int(bool(sub_m)),
                                                                     ctypes.byref(size)))
    if workspace is None or workspace.numel() < size.value:
        workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    st = STATUS_NOT_SUPPORTED
    if table is not None:
        st = lib().mluOpIndiceConvolutionBackwardFilterFromTable(handle.ptr, d_f.ptr, _ptr(features), d_g.ptr,
                                                                 _ptr(output_grad), d_p.ptr, _ptr(table),
                                                                 table.numel() * 4, num, 0, int(bool(sub_m)),
                                                                 _ptr(workspace), size.value, d_w.ptr, _ptr(out))
        if st != STATUS_NOT_SUPPORTED:
            check("mluOpIndiceConvolutionBackwardFilterFromTable", st)
    if st == STATUS_NOT_SUPPORTED:
        check("mluOpIndiceConvolutionBackwardFilter",
              lib().mluOpIndiceConvolutionBackwardFilter(handle.ptr, d_f.ptr, _ptr(features), d_g.ptr,
                                                         _ptr(output_grad), d_p.ptr, _ptr(indice_pairs), num, 0,
                                                         int(bool(sub_m)), _ptr(workspace), size.value, d_w.ptr,
                                                         _ptr(out)))
    for d in (d_f, d_g, d_p, d_w):
        d.destroy()
    return out


def voxelization(handle, points, voxel_size, coors_range, max_points, max_voxels, workspace=None):
    """Deterministic hard voxelization through mluOpVoxelization.

    points [N,F] float32 (x, y, z first), voxel_size [3] and coors_range [6] float32,
    all CUDA tensors.  Returns (voxels [max_voxels,max_points,F], coors [max_voxels,3]
    int32 (z,y,x), num_points_per_voxel [max_voxels] int32, voxel_num [1] int32), all on
    the device.
    """
    import torch
    n, f = points.shape
    dev = points.device
    voxels = _alloc((max_voxels, max_points, f), torch.float32, dev)
    coors = _alloc((max_voxels, 3), torch.int32, dev)
    npv = _alloc((max_voxels,), torch.int32, dev)
    num = torch.zeros((1,), dtype=torch.int32, device=dev)
    descs = [TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (n, f)), TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (3,)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (6,)), TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, tuple(voxels.shape)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (max_voxels, 3)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (max_voxels,)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (1,))]
    d_p, d_vs, d_cr, d_v, d_c, d_n, d_num = (d.ptr for d in descs)
    size = _szt(0)
    check("mluOpGetVoxelizationWorkspaceSize",
          lib().mluOpGetVoxelizationWorkspaceSize(handle.ptr, d_p, d_vs, d_cr, max_points, max_voxels, 3, True, d_v,
                                                  d_c, d_n, d_num, ctypes.byref(size)))
    if workspace is None or workspace.numel() < size.value:
        workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    check("mluOpVoxelization",
          lib().mluOpVoxelization(handle.ptr, d_p, _ptr(points), d_vs, _ptr(voxel_size), d_cr, _ptr(coors_range),
                                  max_points, max_voxels, 3, True, _ptr(workspace), size.value, d_v, _ptr(voxels),
                                  d_c, _ptr(coors), d_n, _ptr(npv), d_num, _ptr(num)))
    for d in descs:
        d.destroy()
    return voxels, coors, npv, num


REDUCE_MODES = {"sum": 0, "mean": 1, "max": 2}


def dynamic_point_to_voxel_forward(handle, feats, coors, reduce_type="max", workspace=None):
    """Groups points by voxel through mluOpDynamicPointToVoxelForward.

    feats [N,C] float32 and coors [N,3] int32 are CUDA tensors; coors rows with a
    negative entry are overwritten with -1 (as the reference does).  Returns
    (voxel_feats [N,C], voxel_coors [N,3], point2voxel_map [N], voxel_points_count [N],
    voxel_num [1]), all on the device; the first voxel_num rows are the voxels.
    """
    import torch
    n, c = feats.shape
    dev = feats.device
    voxel_feats = _alloc((n, c), torch.float32, dev)
    voxel_coors = _alloc((n, 3), torch.int32, dev)
    p2v = _alloc((n,), torch.int32, dev)
    counts = _alloc((n,), torch.int32, dev)
    num = torch.zeros((1,), dtype=torch.int32, device=dev)
    descs = [TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (n, c)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (n, 3)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (n, c)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (n, 3)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (n,)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (n,)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (1,))]
    d_f, d_c, d_vf, d_vc, d_map, d_cnt, d_num = (d.ptr for d in descs)
    size = _szt(0)
    check("mluOpGetDynamicPointToVoxelForwardWorkspaceSize",
          lib().mluOpGetDynamicPointToVoxelForwardWorkspaceSize(handle.ptr, d_f, d_c, ctypes.byref(size)))
    if workspace is None or workspace.numel() < size.value:
        workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    check("mluOpDynamicPointToVoxelForward",
          lib().mluOpDynamicPointToVoxelForward(handle.ptr, REDUCE_MODES[reduce_type], d_f, _ptr(feats), d_c,
                                                _ptr(coors), _ptr(workspace), size.value, d_vf, _ptr(voxel_feats),
                                                d_vc, _ptr(voxel_coors), d_map, _ptr(p2v), d_cnt, _ptr(counts),
                                                d_num, _ptr(num)))
    for d in descs:
        d.destroy()
    return voxel_feats, voxel_coors, p2v, counts, num


def dynamic_point_to_voxel_backward(handle, grad_voxel_feats, feats, voxel_feats, point2voxel_map,
                                    voxel_points_count, voxel_num):
    """grad_feats [N,C] of the maximum reduction through mluOpDynamicPointToVoxelBackward."""
    import torch
    n, c = feats.shape
    m = grad_voxel_feats.shape[0]
    dev = feats.device
    grad_feats = _alloc((n, c), torch.float32, dev)
    descs = [TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (m, c)), TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (n, c)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (m, c)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (n,)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (m,)), TensorDesc(LAYOUT_ARRAY, DTYPE_INT32, (1,)),
             TensorDesc(LAYOUT_ARRAY, DTYPE_FLOAT, (n, c))]
    d_g, d_f, d_vf, d_map, d_cnt, d_num, d_out = (d.ptr for d in descs)
    size = _szt(0)
    check("mluOpGetDynamicPointToVoxelBackwardWorkspaceSize",
          lib().mluOpGetDynamicPointToVoxelBackwardWorkspaceSize(handle.ptr, REDUCE_MODES["max"], d_g, d_f, d_vf,
                                                                 d_map, d_cnt, d_num, ctypes.byref(size)))
    workspace = _alloc((max(size.value, 1),), torch.uint8, dev)
    check("mluOpDynamicPointToVoxelBackward",
          lib().mluOpDynamicPointToVoxelBackward(handle.ptr, REDUCE_MODES["max"], d_g, _ptr(grad_voxel_feats), d_f,
                                                 _ptr(feats), d_vf, _ptr(voxel_feats), d_map, _ptr(point2voxel_map),
                                                 d_cnt, _ptr(voxel_points_count), d_num, _ptr(voxel_num),
                                                 _ptr(workspace), size.value, d_out, _ptr(grad_feats)))
    for d in descs:
        d.destroy()
    return grad_feats


# ---------------------------------------------------------------- operators of a training step
#
# A call of these operators checks its tensors, then finds the descriptors and the workspace size
# for their types and shapes in a table that its handle keeps: building them anew would take longer
# than a small operator runs.

_dtype_codes = {}


def _dtype_code(torch_dtype):
    if not _dtype_codes:
        import torch
        _dtype_codes.update({torch.float16: DTYPE_HALF, torch.bfloat16: DTYPE_BFLOAT16, torch.float32: DTYPE_FLOAT,
                             torch.int32: DTYPE_INT32, torch.int64: DTYPE_INT64, torch.uint8: DTYPE_UINT8,
                             torch.float8_e4m3fn: DTYPE_UINT8})
    return _dtype_codes.get(torch_dtype, DTYPE_INVALID)


def _address(handle, name, t):
    """The address of tensor `t`, which must lie densely on the handle's device."""
    if t.get_device() != handle.device:
        raise ValueError("%s lies on %s, the handle on CUDA device %d" % (name, t.device, handle.device))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


class _CallPlan:
    """Descriptors of the tensors of a call (d: their addresses; None stays None) and its workspace bytes."""
    __slots__ = ("descs", "d", "workspace")

    def __init__(self, handle, key, specs, query=None):
        self.descs = [None if s is None else TensorDesc(LAYOUT_ARRAY, _dtype_code(s[0]), tuple(s[1])) for s in specs]
        self.d = [None if t is None else t.ptr.value for t in self.descs]
        self.workspace = 0
        if query is not None:
            size = _szt(0)
            query(self.d, ctypes.byref(size))
            self.workspace = size.value
        if len(handle.plans) >= 512:  # shapes that change from step to step do not pile up
            handle.plans.clear()
        handle.plans[key] = self


def _on_own_queue(handle):
    """Whether tensors of the current stream's memory pool are the handle's queue's to use at once."""
    import torch
    return _guards is None and (handle.device < 0
                                or torch._C._cuda_getCurrentRawStream(handle.device) == (handle.stream or 0))


def _new(handle, like, shape, dtype):
    """A tensor that the handle's queue may use at once: where that is not the current stream, from the queue's own memory
    pool, and kept until the current stream is done with it too."""
    if _guards is not None:
        return _guards.empty(shape, dtype, like.device)
    if _on_own_queue(handle):
        return like.new_empty(shape) if dtype == like.dtype else like.new_empty(shape, dtype=dtype)
    import torch
    current = torch.cuda.current_stream(handle.device)
    with torch.cuda.stream(torch.cuda.ExternalStream(handle.stream or 0, device=handle.device)):
        t = like.new_empty(shape, dtype=dtype)
    t.record_stream(current)
    return t


def _written(t):
    """Tells autograd that the library has written the caller's tensor: a backward pass that saved its old values then
    refuses.  (Tensors of inference mode are not counted.)"""
    import torch
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _spec(t):
    return None if t is None else (t.dtype, t.shape)


def _activation(name):
    code = GROUP_NORM_ACTS.get(name)
    if code is None:
        raise ValueError("activation is one of %s" % ", ".join(GROUP_NORM_ACTS))
    return code


def group_norm_act_forward(handle, input, weight, bias, num_groups, epsilon=1e-5, activation="none", sample_ends=None,
                           out=None):
    """Group norm of channels-last rows with an activation ("none", "relu", "silu") through
    mluOpGroupNormActForward.

    input [N, ..., C] with a sample for each index of the first dimension, or [rows, C] with
    sample_ends, int32 [N]: where each sample's rows end (rows behind the last end: zeros out).
    weight and bias [C] (float32 or input's type) or both None.  Returns (output, mean, rstd),
    mean and rstd float32 [N, num_groups].  out: the output tensor, may be input.
    """
    import torch
    act = _activation(activation)
    p_x = _address(handle, "input", input)
    p_w = None if weight is None else _address(handle, "weight", weight)
    p_b = None if bias is None else _address(handle, "bias", bias)
    p_e = None if sample_ends is None else _address(handle, "sample_ends", sample_ends)
    stats = ((input if sample_ends is None else sample_ends).shape[0], int(num_groups))
    if _on_own_queue(handle):
        y = torch.empty_like(input) if out is None else out
        mean = input.new_empty(stats, dtype=torch.float32)
        rstd = torch.empty_like(mean)
    else:
        y = _new(handle, input, input.shape, input.dtype) if out is None else out
        mean, rstd = _new(handle, input, stats, torch.float32), _new(handle, input, stats, torch.float32)
    p_y = y.data_ptr() if out is None else _address(handle, "out", out)
    key = ("norm", num_groups, input.shape, input.dtype, None if weight is None else (weight.shape, weight.dtype),
           None if bias is None else (bias.shape, bias.dtype), None if sample_ends is None else (sample_ends.shape, sample_ends.dtype),
           None if out is None else (out.shape, out.dtype))
    plan = handle.plans.get(key)
    if plan is None:
        plan = _CallPlan(handle, key, [_spec(t) for t in (input, weight, bias, sample_ends, y)] + [(torch.float32, stats)],
                         lambda d, size: check("mluOpGetGroupNormActForwardWorkspaceSize",
                                               lib().mluOpGetGroupNormActForwardWorkspaceSize(
                                                   handle.ptr, d[0], d[3], stats[1], size)))
    d_x, d_w, d_b, d_e, d_y, d_m = plan.d
    workspace = _new(handle, input, (plan.workspace,), torch.uint8) if plan.workspace else None
    st = lib().mluOpGroupNormActForward(handle.ptr, d_x, p_x, d_w, p_w, d_b, p_b, d_e, p_e, stats[1], epsilon, act,
                                        workspace.data_ptr() if plan.workspace else None, plan.workspace, d_y, p_y, d_m,
                                        mean.data_ptr(), d_m, rstd.data_ptr())
    if st:
        check("mluOpGroupNormActForward", st)
    if out is not None:
        _written(out)
    return y, mean, rstd


def group_norm_act_backward(handle, output_grad, input, weight, bias, mean, rstd, num_groups, activation="none",
                            sample_ends=None, affine_grad=True, affine_grad_dtype=None, out=None):
    """(input_grad, weight_grad, bias_grad) of group_norm_act_forward through mluOpGroupNormActBackward.

    mean and rstd are the forward call's; affine_grad=False leaves the two affine gradients out
    (None); affine_grad_dtype: float32 (default) or input's type.  out: the input gradient's
    tensor, may be output_grad.
    """
    import torch
    act = _activation(activation)
    p_g = _address(handle, "output_grad", output_grad)
    p_x = _address(handle, "input", input)
    p_w = None if weight is None else _address(handle, "weight", weight)
    p_b = None if bias is None else _address(handle, "bias", bias)
    p_e = None if sample_ends is None else _address(handle, "sample_ends", sample_ends)
    p_m, p_r = _address(handle, "mean", mean), _address(handle, "rstd", rstd)
    num_groups = int(num_groups)
    given = out is not None
    if out is None:
        out = torch.empty_like(input) if _on_own_queue(handle) else _new(handle, input, input.shape, input.dtype)
    p_o = _address(handle, "out", out)
    weight_grad = bias_grad = p_wg = p_bg = None
    if affine_grad:
        weight_grad = _new(handle, input, input.shape[-1:], affine_grad_dtype or torch.float32)
        bias_grad = torch.empty_like(weight_grad) if _on_own_queue(handle) else _new(handle, input, input.shape[-1:], weight_grad.dtype)
        p_wg, p_bg = weight_grad.data_ptr(), bias_grad.data_ptr()
    key = ("norm_grad", num_groups, input.shape, input.dtype, output_grad.shape, output_grad.dtype, out.shape, out.dtype,
           mean.shape, mean.dtype, rstd.shape, rstd.dtype, None if weight is None else (weight.shape, weight.dtype),
           None if bias is None else (bias.shape, bias.dtype), None if sample_ends is None else (sample_ends.shape, sample_ends.dtype),
           weight_grad.dtype if affine_grad else None)
    plan = handle.plans.get(key)
    if plan is None:
        plan = _CallPlan(handle, key, [_spec(t) for t in (output_grad, input, weight, bias, sample_ends, mean, rstd, out,
                                                          weight_grad, bias_grad)],
                         lambda d, size: check("mluOpGetGroupNormActBackwardWorkspaceSize",
                                               lib().mluOpGetGroupNormActBackwardWorkspaceSize(
                                                   handle.ptr, d[1], d[4], num_groups, size)))
    d_g, d_x, d_w, d_b, d_e, d_m, d_r, d_o, d_wg, d_bg = plan.d
    workspace = _new(handle, input, (plan.workspace,), torch.uint8) if plan.workspace else None
    st = lib().mluOpGroupNormActBackward(handle.ptr, d_g, p_g, d_x, p_x, d_w, p_w, d_b, p_b, d_e, p_e, d_m, p_m, d_r, p_r,
                                         num_groups, act, workspace.data_ptr() if plan.workspace else None, plan.workspace,
                                         d_o, p_o, d_wg, p_wg, d_bg, p_bg)
    if st:
        check("mluOpGroupNormActBackward", st)
    if given:
        _written(out)
    return out, weight_grad, bias_grad


SCALE_BLOCK = 256  # consecutive elements of an 8-bit optimiser state that share a scale


def _addresses(tensors):
    """A C array of the tensors' addresses."""
    import torch
    return array.array("Q", map(torch.Tensor.data_ptr, tensors))


def same_order(a, b):
    """Whether tensors a and b are dense and have their elements in the same order in memory."""
    if a.is_contiguous() and b.is_contiguous():
        return a.numel() == b.numel()
    if a.shape != b.shape:
        return False
    expected = 1
    for stride, other, size in sorted(zip(a.stride(), b.stride(), a.shape)):
        if size != 1:
            if stride != expected or other != expected:
                return False
            expected *= size
    return True


class MultiTensorAdamW:
    """AdamW steps over the same tensors through mluOpMultiTensorAdamW.

    params: dense CUDA tensors of one type (float32, float16 or bfloat16), updated in place;
    exp_avgs and exp_avg_sqs: their states, of the same element counts; a parameter that is not
    contiguous (channels last, say) has states and gradients of its shape and strides.  float32 states hold the
    moments themselves.  8-bit states (uint8 or float8_e4m3fn) hold the first moment and the
    square root of the second as e4m3 codes; exp_avg_scales and exp_avg_sq_scales then hold one
    float32 for each 256 elements of their tensor (code * scale is the value).  The object keeps
    references to the tensors, whose storage has to stay where it is between the steps.
    """

    def __init__(self, params, exp_avgs, exp_avg_sqs, exp_avg_scales=None, exp_avg_sq_scales=None):
        import torch
        self.params, self.exp_avgs, self.exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)
        if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
            raise ValueError("the scales of both states come together")
        self.eight_bit = exp_avg_scales is not None
        self.scales = [list(exp_avg_scales), list(exp_avg_sq_scales)] if self.eight_bit else []
        if any(len(v) != len(self.params) for v in [self.exp_avgs, self.exp_avg_sqs] + self.scales):
            raise ValueError("the lists have different lengths")
        self.numels = [p.numel() for p in self.params]
        self.dtype = self.params[0].dtype if self.params else torch.float32
        self.device = self.params[0].get_device() if self.params else None
        states = (torch.uint8, torch.float8_e4m3fn) if self.eight_bit else (torch.float32,)
        spans = []
        for p, m, v, n in zip(self.params, self.exp_avgs, self.exp_avg_sqs, self.numels):
            if p.dtype != self.dtype or m.dtype not in states or v.dtype not in states:
                raise ValueError("parameters have one type, states are float32, or 8 bits with scales")
            if m.numel() != n or v.numel() != n:
                raise ValueError("a state has another number of elements than its parameter")
            if not (p.is_contiguous() and m.is_contiguous() and v.is_contiguous()
                    or same_order(p, p) and same_order(p, m) and same_order(p, v)):
                raise ValueError("every tensor is dense, and a state laid out like its parameter")
            spans += [p, m, v]
        for scales in self.scales:
            for q, n in zip(scales, self.numels):
                if q.dtype != torch.float32 or q.numel() != -(-n // SCALE_BLOCK):
                    raise ValueError("scales are float32, one for each %d elements" % SCALE_BLOCK)
                if not q.is_contiguous():
                    raise ValueError("every tensor is dense")
                spans.append(q)
        end = 0
        for begin, size, t in sorted(((t.data_ptr(), t.numel() * t.element_size(), t) for t in spans),
                                     key=lambda x: x[:2]):
            if t.get_device() != self.device:
                raise ValueError("every tensor is dense and on the same device")
            if size and begin < end:
                raise ValueError("two of the tensors overlap")
            end = max(end, begin + size)
        self._param_p, self._m_p, self._v_p = _addresses(self.params), _addresses(self.exp_avgs), _addresses(self.exp_avg_sqs)
        self._scale_p = [_addresses(v) for v in self.scales] or [None, None]
        self._numel_p = i64_array(self.numels)
        self._contiguous = all(p.is_contiguous() for p in self.params)
        # whose change autograd has to hear of: views share the count of their base (tensors of inference mode have none)
        updated = [t for t in self.params + self.exp_avgs + self.exp_avg_sqs + sum(self.scales, []) if not t.is_inference()]
        self._updated = list({id(t): t for t in (t._base if t._is_view() else t for t in updated)}.values())

    def step(self, handle, grads, lr, betas=(0.9, 0.999), epsilon=1e-8, weight_decay=0.01, step=1, grad_scale=None,
             schedule=None, rounding="nearest", step_count=None):
        """One step with the gradients `grads` (dense, in the parameters' order; their type or float32).

        step counts from 1.  grad_scale: a float32 CUDA tensor of one element that every gradient is
        multiplied by (a clipping or loss-scale factor).  schedule: a float32 CUDA tensor {lr,
        1 - beta1^step, 1 - beta2^step} that takes the place of lr and step when the kernels run.

        rounding of 8-bit states: "nearest", or "stochastic" for a training run, whose states stop following the
        gradients when they are rounded to the nearest code at every step (mluOpMultiTensorAdamW_v2).  step_count: an
        int64 CUDA tensor of one element that takes the place of step in the stochastic choice; a schedule needs it there.
        """
        import torch
        if rounding not in ADAMW_ROUNDINGS:
            raise ValueError("rounding is one of %s" % ", ".join(ADAMW_ROUNDINGS))
        if rounding == "stochastic" and self.eight_bit and schedule is not None and step_count is None:
            raise ValueError("stochastic rounding with a schedule needs a step_count")
        if len(grads) != len(self.params):
            raise ValueError("%d gradients for %d parameters" % (len(grads), len(self.params)))
        if not grads:
            return
        if self.device != handle.device:
            raise ValueError("the tensors lie on device %s, the handle on CUDA device %d" % (self.device, handle.device))
        dtype, of = grads[0].dtype, torch.Tensor  # (mapped methods: a step of many small tensors is mostly this)
        if (list(map(of.numel, grads)) != self.numels or {g.dtype for g in grads} != {dtype}
                or set(map(of.get_device, grads)) != {self.device}
                or not (all(map(of.is_contiguous, grads)) if self._contiguous else all(map(same_order, self.params, grads)))):
            raise ValueError("gradients are dense, of one type, on the parameters' device and of their sizes and order")
        for name, t, n in (("grad_scale", grad_scale, 1), ("schedule", schedule, 3)):
            if t is not None and (t.dtype != torch.float32 or t.numel() != n or t.get_device() != self.device
                                  or not t.is_contiguous()):
                raise ValueError("%s is a dense float32 tensor of %d element(s) on the parameters' device" % (name, n))
        if step_count is not None and (step_count.dtype != torch.int64 or step_count.numel() != 1
                                       or step_count.get_device() != self.device):
            raise ValueError("step_count is an int64 tensor of one element on the parameters' device")
        grad_p = _addresses(grads)
        args = (handle.ptr, _dtype_code(self.dtype), _dtype_code(dtype), DTYPE_UINT8 if self.eight_bit else DTYPE_FLOAT,
                len(self.params), self._numel_p, self._param_p.buffer_info()[0], grad_p.buffer_info()[0],
                self._m_p.buffer_info()[0], self._v_p.buffer_info()[0], *[p and p.buffer_info()[0] for p in self._scale_p],
                lr, betas[0], betas[1], epsilon, weight_decay, int(step), _ptr(grad_scale), _ptr(schedule))
        if rounding == "nearest":
            check("mluOpMultiTensorAdamW", lib().mluOpMultiTensorAdamW(*args))
        else:
            check("mluOpMultiTensorAdamW_v2",
                  lib().mluOpMultiTensorAdamW_v2(*args, ADAMW_ROUNDINGS[rounding], _ptr(step_count)))
        torch.autograd.graph.increment_version(self._updated)


def _grouped_rows_call(name, handle, rows, weight, group_ends, columns, out):
    """The forward product and the input gradient: rows [R,K] times each group's matrix into [R, columns]."""
    p_x, p_w, p_e = (_address(handle, "the row matrix", rows), _address(handle, "weight", weight),
                     _address(handle, "group_ends", group_ends))
    given = out is not None
    if out is None:
        out = _new(handle, rows, (rows.shape[0], columns), rows.dtype)
    p_y = _address(handle, "out", out)
    key = ("product", rows.shape, rows.dtype, weight.shape, weight.dtype, group_ends.shape, group_ends.dtype, out.shape,
           out.dtype)
    plan = handle.plans.get(key)
    if plan is None:
        plan = _CallPlan(handle, key, [_spec(t) for t in (rows, weight, group_ends, out)])
    d_x, d_w, d_e, d_y = plan.d
    st = getattr(lib(), name)(handle.ptr, d_x, p_x, d_w, p_w, d_e, p_e, d_y, p_y)
    if st:
        check(name, st)
    if given:
        _written(out)
    return out


def grouped_matmul_forward(handle, input, weight, group_ends, out=None):
    """output [rows,Co] with output[r] = input[r] @ weight[g] for the rows r of group g, through
    mluOpGroupedMatMulForward.

    input [rows,Ci], weight [G,Ci,Co] of one type (float16, bfloat16, float32); group_ends int32
    [G] on the device: group g's rows end there, the next group's begin.  Rows behind the last
    group's end: zeros.
    """
    return _grouped_rows_call("mluOpGroupedMatMulForward", handle, input, weight, group_ends, weight.shape[-1], out)


def grouped_matmul_backward_input(handle, output_grad, weight, group_ends, out=None):
    """input_grad [rows,Ci] with input_grad[r] = output_grad[r] @ weight[g].T through
    mluOpGroupedMatMulBackwardInput (the forward call's arguments)."""
    return _grouped_rows_call("mluOpGroupedMatMulBackwardInput", handle, output_grad, weight, group_ends, weight.shape[-2], out)


def grouped_matmul_backward_weight(handle, input, output_grad, group_ends, dtype=None, out=None):
    """weight_grad [G,Ci,Co] with weight_grad[g] = input[rows of g].T @ output_grad[rows of g] through
    mluOpGroupedMatMulBackwardWeight; dtype: input's (default) or float32."""
    import torch
    p_x, p_g, p_e = (_address(handle, "input", input), _address(handle, "output_grad", output_grad),
                     _address(handle, "group_ends", group_ends))
    given = out is not None
    if out is None:
        out = _new(handle, input, (group_ends.shape[0], input.shape[-1], output_grad.shape[-1]), dtype or input.dtype)
    p_w = _address(handle, "out", out)
    key = ("product_weight", input.shape, input.dtype, output_grad.shape, output_grad.dtype, group_ends.shape,
           group_ends.dtype, out.shape, out.dtype)
    plan = handle.plans.get(key)
    if plan is None:
        plan = _CallPlan(handle, key, [_spec(t) for t in (input, output_grad, group_ends, out)],
                         lambda d, size: check("mluOpGetGroupedMatMulBackwardWeightWorkspaceSize",
                                               lib().mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(
                                                   handle.ptr, d[0], d[1], d[3], size)))
    d_x, d_g, d_e, d_w = plan.d
    workspace = _new(handle, input, (plan.workspace,), torch.uint8)
    st = lib().mluOpGroupedMatMulBackwardWeight(handle.ptr, d_x, p_x, d_g, p_g, d_e, p_e, workspace.data_ptr(),
                                                plan.workspace, d_w, p_w)
    if st:
        check("mluOpGroupedMatMulBackwardWeight", st)
    if given:
        _written(out)
    return out
