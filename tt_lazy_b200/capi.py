"""ctypes binding of the tt_cuda_lib C-ABI (``include/tt_cuda.h``).

This is the same boundary a C or C++ caller uses: device pointers, sizes and
strides, an int status. Every non-zero status raises :class:`TTCError` with
the library's ``ttc_last_error()`` text. The library is loaded from the
in-tree build (``tt_lazy_b200/lib/libtt_cuda.so``); a missing library is an
ImportError, never a silent fallback.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libtt_cuda.so")

MAX_INPUTS, MAX_OUTPUTS, MAX_INSTR, SLOTS = 6, 4, 32, 4

# ttc_status
OK, ERR_INVALID, ERR_CUDA, ERR_OOM, ERR_UNSUPPORTED, ERR_NOT_INIT, ERR_NCCL, ERR_TIMEOUT = range(8)
# ttc_opcode
OP_LOAD, OP_RELU, OP_SIGMOID, OP_ADD, OP_MUL, OP_SAVE, OP_STORE = range(1, 8)
# ttc_src_kind
SRC_ACC, SRC_INPUT, SRC_SLOT = range(3)
# ttc_reduce_mode
REDUCE_NONE, REDUCE_ALL, REDUCE_ROWS, REDUCE_COLS = range(4)
# ttc_gemm_path
GEMM_AUTO, GEMM_FFMA, GEMM_TF32, GEMM_TF32X3 = range(4)
# ttc_dtype
F32, F16, BF16, E4M3 = range(4)
DTYPES = {"f32": F32, "f16": F16, "bf16": BF16, "e4m3": E4M3}
# ttc_activation
ACT_NONE, ACT_RELU, ACT_SILU, ACT_GELU, ACT_GELU_TANH = range(5)
ACTIVATIONS = {"none": ACT_NONE, "relu": ACT_RELU, "silu": ACT_SILU, "gelu": ACT_GELU, "gelu_tanh": ACT_GELU_TANH}


class Instr(C.Structure):
    _fields_ = [("op", C.c_uint8), ("src", C.c_uint8), ("idx", C.c_uint8), ("pad", C.c_uint8)]


class InView(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("row_stride", C.c_int64), ("col_stride", C.c_int64),
                ("seg_stride", C.c_int64)]


class OutView(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("row_stride", C.c_int64), ("seg_stride", C.c_int64)]


class ChainDesc(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("nseg", C.c_int32),
                ("n_inputs", C.c_int32), ("n_outputs", C.c_int32), ("n_instr", C.c_int32),
                ("inputs", InView * MAX_INPUTS), ("outputs", OutView * MAX_OUTPUTS),
                ("program", Instr * MAX_INSTR),
                ("reduce", C.c_int32), ("reduce_mean", C.c_int32),
                ("reduce_out", C.c_void_p), ("reduce_seg_stride", C.c_int64)]


class GemmDesc(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
                ("a", C.c_void_p), ("lda", C.c_int64), ("trans_a", C.c_int32),
                ("b", C.c_void_p), ("ldb", C.c_int64), ("trans_b", C.c_int32),
                ("c", C.c_void_p), ("ldc", C.c_int64),
                ("path", C.c_int32),
                ("epilogue", ChainDesc)]


class RmsNormDesc(C.Structure):
    _fields_ = [("rows", C.c_int64), ("cols", C.c_int32),
                ("dtype", C.c_int32), ("weight_dtype", C.c_int32), ("y_dtype", C.c_int32), ("eps", C.c_float),
                ("x", C.c_void_p), ("ldx", C.c_int64), ("residual", C.c_void_p), ("ldr", C.c_int64),
                ("weight", C.c_void_p), ("y", C.c_void_p), ("ldy", C.c_int64),
                ("hidden", C.c_void_p), ("ldh", C.c_int64), ("scales", C.c_void_p)]


class RmsNormBackwardDesc(C.Structure):
    _fields_ = [("rows", C.c_int64), ("cols", C.c_int32),
                ("dtype", C.c_int32), ("weight_dtype", C.c_int32), ("eps", C.c_float),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("hidden", C.c_void_p), ("ldh", C.c_int64),
                ("weight", C.c_void_p), ("dhidden", C.c_void_p), ("lddh", C.c_int64),
                ("dx", C.c_void_p), ("lddx", C.c_int64), ("dweight", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class LinearDesc(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
                ("dtype", C.c_int32), ("y_dtype", C.c_int32), ("trans_w", C.c_int32), ("act", C.c_int32),
                ("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p), ("ldw", C.c_int64),
                ("y", C.c_void_p), ("ldy", C.c_int64), ("bias", C.c_void_p),
                ("residual", C.c_void_p), ("ldr", C.c_int64), ("pre", C.c_void_p), ("ldp", C.c_int64),
                ("x_scales", C.c_void_p), ("w_scales", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class LinearBackwardDesc(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
                ("dtype", C.c_int32), ("trans_w", C.c_int32), ("act", C.c_int32),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("w", C.c_void_p), ("ldw", C.c_int64), ("pre", C.c_void_p), ("ldp", C.c_int64),
                ("dx", C.c_void_p), ("lddx", C.c_int64), ("dw", C.c_void_p), ("lddw", C.c_int64),
                ("dbias", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class GatedLinearDesc(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
                ("dtype", C.c_int32), ("y_dtype", C.c_int32), ("trans_w", C.c_int32), ("act", C.c_int32),
                ("x", C.c_void_p), ("ldx", C.c_int64), ("wg", C.c_void_p), ("wu", C.c_void_p), ("ldw", C.c_int64),
                ("y", C.c_void_p), ("ldy", C.c_int64), ("gate", C.c_void_p), ("up", C.c_void_p), ("ldp", C.c_int64),
                ("x_scales", C.c_void_p), ("wg_scales", C.c_void_p), ("wu_scales", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class GatedLinearBackwardDesc(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
                ("dtype", C.c_int32), ("trans_w", C.c_int32), ("act", C.c_int32),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("wg", C.c_void_p), ("wu", C.c_void_p), ("ldw", C.c_int64),
                ("gate", C.c_void_p), ("up", C.c_void_p), ("ldp", C.c_int64),
                ("dx", C.c_void_p), ("lddx", C.c_int64), ("dwg", C.c_void_p), ("dwu", C.c_void_p),
                ("lddw", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class MemoryStats(C.Structure):
    _fields_ = [("bytes_in_use", C.c_size_t), ("peak_bytes", C.c_size_t), ("workspace_bytes", C.c_size_t),
                ("kernels_launched", C.c_uint64)]


# Every symbol include/tt_cuda.h declares (checked by tests/test_capi.py).
EXPORTS = ["ttc_last_error", "ttc_init", "ttc_shutdown", "ttc_device_count", "ttc_version", "ttc_get_stream",
           "ttc_set_stream", "ttc_synchronize", "ttc_malloc", "ttc_free", "ttc_memcpy_h2d", "ttc_memcpy_d2h", "ttc_h2d_prefetch", "ttc_wait_ticket", "ttc_capture_begin", "ttc_capture_end", "ttc_graph_launch", "ttc_graph_destroy", "ttc_range_push", "ttc_range_pop", "ttc_timer_mark", "ttc_timer_elapsed",
           "ttc_memcpy_d2d", "ttc_memset_zero", "ttc_host_alloc", "ttc_host_free", "ttc_get_memory_stats",
           "ttc_eltwise_chain", "ttc_eltwise_chain_noalloc", "ttc_chain_jit_source", "ttc_reduce", "ttc_transpose", "ttc_copy2d", "ttc_gemm", "ttc_gemm_select_path",
           "ttc_rms_norm", "ttc_rms_norm_backward", "ttc_rms_norm_backward_workspace",
           "ttc_linear", "ttc_linear_workspace", "ttc_linear_backward", "ttc_linear_backward_workspace",
           "ttc_gated_linear", "ttc_gated_linear_workspace",
           "ttc_gated_linear_backward", "ttc_gated_linear_backward_workspace",
           "ttc_comm_unique_id", "ttc_comm_init", "ttc_allreduce_sum", "ttc_comm_destroy"]


# Descriptors whose calls take a workspace, and those calls.
_WITH_WORKSPACE = {RmsNormBackwardDesc: "ttc_rms_norm_backward", LinearDesc: "ttc_linear",
                   LinearBackwardDesc: "ttc_linear_backward", GatedLinearDesc: "ttc_gated_linear",
                   GatedLinearBackwardDesc: "ttc_gated_linear_backward"}
_calls = {}  # descriptor type -> (the call, its _workspace function), filled when the library is loaded


class TTCError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(msg)
        self.code = code


_lib = None


def lib():
    """Load libtt_cuda.so (raises ImportError when it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"tt_cuda library not built: {LIB_PATH} (run python tt_lazy_b200/build.py)")
        L = C.CDLL(LIB_PATH, mode=C.RTLD_GLOBAL)
        L.ttc_last_error.restype = C.c_char_p
        L.ttc_get_stream.restype = C.c_void_p
        L.ttc_malloc.argtypes = [C.c_size_t, C.POINTER(C.c_void_p)]
        L.ttc_free.argtypes = [C.c_void_p]
        for fn in (L.ttc_memcpy_h2d, L.ttc_memcpy_d2h, L.ttc_memcpy_d2d):
            fn.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t]
        L.ttc_memset_zero.argtypes = [C.c_void_p, C.c_size_t]
        L.ttc_h2d_prefetch.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.POINTER(C.c_int)]
        L.ttc_wait_ticket.argtypes = [C.c_int]
        L.ttc_capture_end.argtypes = [C.POINTER(C.c_void_p)]
        L.ttc_graph_launch.argtypes = [C.c_void_p]
        L.ttc_graph_destroy.argtypes = [C.c_void_p]
        L.ttc_range_push.argtypes = [C.c_char_p]
        L.ttc_timer_mark.argtypes = [C.POINTER(C.c_int)]
        L.ttc_timer_elapsed.argtypes = [C.c_int, C.c_int, C.POINTER(C.c_float)]
        L.ttc_host_alloc.argtypes = [C.c_size_t, C.POINTER(C.c_void_p)]
        L.ttc_host_free.argtypes = [C.c_void_p]
        L.ttc_set_stream.argtypes = [C.c_void_p]
        L.ttc_eltwise_chain.argtypes = [C.POINTER(ChainDesc)]
        L.ttc_eltwise_chain_noalloc.argtypes = [C.POINTER(ChainDesc)]
        L.ttc_chain_jit_source.argtypes = [C.POINTER(ChainDesc), C.c_char_p, C.c_size_t, C.POINTER(C.c_size_t)]
        L.ttc_gemm.argtypes = [C.POINTER(GemmDesc)]
        L.ttc_gemm_select_path.argtypes = [C.POINTER(GemmDesc)]
        L.ttc_rms_norm.argtypes = [C.POINTER(RmsNormDesc)]
        for desc, fn in _WITH_WORKSPACE.items():
            call, size = getattr(L, fn), getattr(L, fn + "_workspace")
            call.argtypes = [C.POINTER(desc)]
            size.argtypes = [C.POINTER(desc), C.POINTER(C.c_size_t)]
            _calls[desc] = call, size
        L.ttc_reduce.argtypes = [C.c_void_p, C.POINTER(C.c_uint32), C.c_int, C.POINTER(C.c_int32), C.c_int,
                                 C.c_int, C.c_void_p]
        L.ttc_transpose.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64]
        L.ttc_copy2d.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int64, C.c_int64]
        L.ttc_get_memory_stats.argtypes = [C.POINTER(MemoryStats)]
        L.ttc_allreduce_sum.argtypes = [C.c_void_p, C.c_size_t, C.c_int]
        L.ttc_comm_init.argtypes = [C.c_int, C.c_int, C.c_char_p, C.c_int]
        L.ttc_comm_unique_id.argtypes = [C.c_char_p]
        _lib = L
    return _lib


def check(rc):
    if rc != OK:
        raise TTCError(rc, lib().ttc_last_error().decode())
    return rc


def init(device=0):
    check(lib().ttc_init(device))


def set_stream(stream=None):
    """Run the library's calls on `stream`, a CUDA stream handle (an int, as in
    torch.cuda.Stream.cuda_stream); None restores the library's own stream.
    Handle 0, CUDA's legacy default stream, is passed on by its other name,
    since 0 means the library's own stream to ttc_set_stream."""
    check(lib().ttc_set_stream(None if stream is None else (stream or 1)))


def synchronize():
    check(lib().ttc_synchronize())


def stats() -> MemoryStats:
    s = MemoryStats()
    check(lib().ttc_get_memory_stats(C.byref(s)))
    return s


def kernels_launched() -> int:
    return int(stats().kernels_launched)


class DeviceArray:
    """A buffer in device memory, owned through ttc_malloc/ttc_free: float32,
    or another numpy type of the same bits as its elements (float16; uint16
    for bf16 and uint8 for e4m3, which numpy does not have)."""

    def __init__(self, shape, ptr=None, owner=True, dtype=np.float32):
        self.shape = tuple(int(s) for s in shape)
        self.size = int(np.prod(self.shape)) if self.shape else 1
        self.dtype = np.dtype(dtype)
        self.nbytes = self.size * self.dtype.itemsize
        if ptr is None:
            p = C.c_void_p()
            check(lib().ttc_malloc(self.nbytes, C.byref(p)))
            ptr = p.value
        self.ptr = ptr
        self._owner = owner

    @classmethod
    def from_numpy(cls, a, dtype=np.float32):
        a = np.ascontiguousarray(a, dtype=dtype)
        d = cls(a.shape, dtype=dtype)
        check(lib().ttc_memcpy_h2d(d.ptr, a.ctypes.data, d.nbytes))
        return d

    @classmethod
    def empty(cls, shape, dtype=np.float32):
        return cls(shape, dtype=dtype)

    @classmethod
    def zeros(cls, shape, dtype=np.float32):
        d = cls(shape, dtype=dtype)
        check(lib().ttc_memset_zero(d.ptr, d.nbytes))
        return d

    def numpy(self):
        out = np.empty(self.shape, dtype=self.dtype)
        check(lib().ttc_memcpy_d2h(out.ctypes.data, self.ptr, self.nbytes))
        return out

    def at(self, elem_offset):
        """Pointer to element `elem_offset` (a view; no ownership)."""
        return (self.ptr or 0) + self.dtype.itemsize * int(elem_offset)

    def free(self):
        if self._owner and self.ptr:
            lib().ttc_free(self.ptr)
        self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ------------------------------------------------------------ descriptor helpers
def in_view(ptr, row_stride, col_stride=1, seg_stride=0):
    return InView(ptr, row_stride, col_stride, seg_stride)


def out_view(ptr, row_stride, seg_stride=0):
    return OutView(ptr, row_stride, seg_stride)


def instr(op, src=SRC_ACC, idx=0):
    return Instr(op, src, idx, 0)


def chain_desc(rows, cols, inputs, outputs, program, reduce=REDUCE_NONE, reduce_out=None, mean=False, nseg=1,
               reduce_seg_stride=0):
    d = ChainDesc()
    d.rows, d.cols, d.nseg = rows, cols, nseg
    d.n_inputs, d.n_outputs, d.n_instr = len(inputs), len(outputs), len(program)
    for i, v in enumerate(inputs):
        d.inputs[i] = v
    for i, v in enumerate(outputs):
        d.outputs[i] = v
    for i, v in enumerate(program):
        d.program[i] = v
    d.reduce = reduce
    d.reduce_mean = int(mean)
    d.reduce_out = reduce_out
    d.reduce_seg_stride = reduce_seg_stride
    return d


def eltwise_chain(desc):
    check(lib().ttc_eltwise_chain(C.byref(desc)))


def chain_jit_source(desc):
    """CUDA source of the specialised kernel for `desc` (no device needed)."""
    n = C.c_size_t(0)
    check(lib().ttc_chain_jit_source(C.byref(desc), None, 0, C.byref(n)))
    buf = C.create_string_buffer(n.value + 1)
    check(lib().ttc_chain_jit_source(C.byref(desc), buf, n.value + 1, C.byref(n)))
    return buf.value.decode()


def gemm(M, N, K, a, lda, b, ldb, c=None, ldc=0, trans_a=False, trans_b=False, path=GEMM_AUTO, epilogue=None):
    g = GemmDesc()
    g.M, g.N, g.K = M, N, K
    g.a, g.lda, g.trans_a = a, lda, int(trans_a)
    g.b, g.ldb, g.trans_b = b, ldb, int(trans_b)
    g.c, g.ldc = c, ldc
    g.path = path
    if epilogue is not None:
        g.epilogue = epilogue
    check(lib().ttc_gemm(C.byref(g)))
    return g


def gemm_select_path(g) -> int:
    return lib().ttc_gemm_select_path(C.byref(g))


def reduce(in_ptr, shape, dims, mean, out_ptr):
    sh = (C.c_uint32 * len(shape))(*shape)
    dd = (C.c_int32 * max(1, len(dims)))(*dims)
    check(lib().ttc_reduce(in_ptr, sh, len(shape), dd, len(dims), int(mean), out_ptr))


def transpose(in_ptr, out_ptr, batch, rows, cols):
    check(lib().ttc_transpose(in_ptr, out_ptr, batch, rows, cols))


def copy2d(in_ptr, in_ld, out_ptr, out_ld, rows, cols):
    check(lib().ttc_copy2d(in_ptr, in_ld, out_ptr, out_ld, rows, cols))


# ------------------------------------------------- feed-forward block operators
# Each operator has a descriptor builder, like chain_desc, and a call that takes
# the descriptor. Pointers are device addresses (ints); dtype and y_dtype are
# F32 / F16 / BF16 / E4M3. See include/tt_cuda.h for the formulas and rules.
def rms_norm_desc(rows, cols, x, ldx, weight, y, ldy, dtype, y_dtype=None, weight_dtype=None, eps=1e-6,
                  residual=None, ldr=0, hidden=None, ldh=0, scales=None):
    return RmsNormDesc(rows, cols, dtype, dtype if weight_dtype is None else weight_dtype,
                       dtype if y_dtype is None else y_dtype, eps, x, ldx, residual, ldr, weight, y, ldy, hidden, ldh,
                       scales)


def rms_norm_backward_desc(rows, cols, dy, lddy, hidden, ldh, weight, dx, lddx, dweight, dtype, weight_dtype=None,
                           eps=1e-6, dhidden=None, lddh=0):
    return RmsNormBackwardDesc(rows, cols, dtype, dtype if weight_dtype is None else weight_dtype, eps, dy, lddy,
                               hidden, ldh, weight, dhidden, lddh, dx, lddx, dweight)


def linear_desc(M, N, K, x, ldx, w, ldw, y, ldy, dtype, y_dtype=None, trans_w=False, act=ACT_NONE, bias=None,
                residual=None, ldr=0, pre=None, ldp=0, x_scales=None, w_scales=None):
    return LinearDesc(M, N, K, dtype, dtype if y_dtype is None else y_dtype, trans_w, act, x, ldx, w, ldw, y, ldy,
                      bias, residual, ldr, pre, ldp, x_scales, w_scales)


def linear_backward_desc(M, N, K, dy, lddy, x, ldx, w, ldw, dtype, trans_w=False, act=ACT_NONE, pre=None, ldp=0,
                         dx=None, lddx=0, dw=None, lddw=0, dbias=None):
    return LinearBackwardDesc(M, N, K, dtype, trans_w, act, dy, lddy, x, ldx, w, ldw, pre, ldp, dx, lddx, dw, lddw,
                              dbias)


def gated_linear_desc(M, N, K, x, ldx, wg, wu, ldw, y, ldy, dtype, y_dtype=None, trans_w=False, act=ACT_SILU,
                      gate=None, up=None, ldp=0, x_scales=None, wg_scales=None, wu_scales=None):
    return GatedLinearDesc(M, N, K, dtype, dtype if y_dtype is None else y_dtype, trans_w, act, x, ldx, wg, wu, ldw,
                           y, ldy, gate, up, ldp, x_scales, wg_scales, wu_scales)


def gated_linear_backward_desc(M, N, K, dy, lddy, x, ldx, wg, wu, ldw, gate, up, ldp, dtype, trans_w=False,
                               act=ACT_SILU, dx=None, lddx=0, dwg=None, dwu=None, lddw=0):
    return GatedLinearBackwardDesc(M, N, K, dtype, trans_w, act, dy, lddy, x, ldx, wg, wu, ldw, gate, up, ldp, dx,
                                   lddx, dwg, dwu, lddw)


def workspace_size(desc) -> int:
    """Bytes of workspace that the call with this descriptor needs (0: none)."""
    lib()
    n = C.c_size_t()
    check(_calls[type(desc)][1](desc, n))
    return n.value


def _call(desc, workspace):
    """`workspace`: None, a DeviceArray or a torch CUDA tensor."""
    if workspace is not None:
        desc.workspace = workspace.ptr if isinstance(workspace, DeviceArray) else workspace.data_ptr()
        desc.workspace_bytes = workspace.nbytes
    lib()
    check(_calls[type(desc)][0](desc))


def rms_norm(desc):
    check(lib().ttc_rms_norm(desc))


def rms_norm_backward(desc, workspace=None):
    _call(desc, workspace)


def linear(desc, workspace=None):
    _call(desc, workspace)


def linear_backward(desc, workspace=None):
    _call(desc, workspace)


def gated_linear(desc, workspace=None):
    _call(desc, workspace)


def gated_linear_backward(desc, workspace=None):
    _call(desc, workspace)
