"""tinygnn_amd -- TinyGNN's sparse-inference path on MI355X (gfx950).

The product is the C-ABI library ``_build/libtinygnn_amd.so`` (hand-written
HIP kernels, declared in ``include/tinygnn_amd.h``) and the C++ API over it
(``include/tinygnn/*.hpp``).  This Python module is a thin ctypes front end
used by the tests and the benchmark: it takes torch tensors for device
memory and the current torch stream for ordering, and passes raw pointers
through the C-ABI.  There is no CPU fallback: without the library or a GPU
every call raises.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass

from ._lib import InvalidArgument, NativeLibraryMissing, OutOfRange, TgError, lib  # noqa: F401

ACT_NONE, ACT_RELU = 0, 1
POST_NONE, POST_RELU, POST_ELU = 0, 1, 2
AGG_MEAN, AGG_MAX = 0, 1
GEMM_AUTO, GEMM_INORDER, GEMM_MFMA = 0, 1, 2
EPI_NONE, EPI_RELU, EPI_ELU = 0, 1, 2
EPI_GELU, EPI_SILU = 3, 4   # linear's alone
SAGE_AUTO, SAGE_CONCAT, SAGE_TRANSFORM_FIRST = 0, 1, 2
FORWARD_REFERENCE, FORWARD_CACHED = 0, 1
PRECISION_FAST, PRECISION_EXACT = 0, 1
TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2


def _torch():
    import torch
    return torch


def stream_handle(stream=None) -> int:
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream)


def _on(stream) -> int:
    """The handle of the stream that a call runs on.  One that is not the
    current one waits for what is queued there: a call's inputs may come from
    it, and its outputs and workspaces are torch's memory of the current stream,
    on which work of whoever held a block before may still be pending.  (Not
    where either is being captured, and could not: there the order is the
    caller's.)"""
    handle = stream_handle(stream)
    if stream is None:
        return handle
    cuda = _torch().cuda
    current = cuda.current_stream()
    if int(current.cuda_stream) == handle:
        return handle
    wait = getattr(stream, "wait_stream", None)
    if wait is None:   # no torch stream: a handle alone
        if not _capturing(None):
            current.synchronize()
    elif not _capturing(None) and not _capturing(stream):
        wait(current)
    return handle


def _capturing(stream) -> bool:
    """Whether `stream` (None: the current one) is being captured."""
    cuda = _torch().cuda
    if not cuda.is_initialized():
        return False
    with cuda.stream(stream):
        return cuda.is_current_stream_capturing()


def _finish(stream) -> None:
    """Waits for `stream` where it is not the current one.  The outputs of a
    call are torch's memory of the current stream: reading a result's size, the
    caller's next operation and the allocator's reuse of what the caller drops
    are all ordered there, not after another stream's kernels."""
    if stream is None or int(stream.cuda_stream) == stream_handle():
        return
    wait = getattr(stream, "synchronize", None)
    (wait or _torch().cuda.ExternalStream(int(stream.cuda_stream)).synchronize)()


def trim() -> None:
    """Gives the memory kept for the temporaries of later calls (at most 512
    MiB per device) back to the driver, for other allocators."""
    lib.check(lib.tg_trim())


def dptr(t, dtype=None) -> int:
    """Device pointer of a CUDA/HIP torch tensor (0 for None): contiguous, or
    a row-major 2-D view with unit column stride (its row stride is passed as
    the leading dimension)."""
    if t is None:
        return 0
    if not t.is_cuda:
        raise ValueError("tinygnn_amd expects device (cuda) tensors")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"expected {dtype}, got {t.dtype}")
    if not (t.is_contiguous() or (t.dim() == 2 and t.stride(1) == 1)):
        raise ValueError("tinygnn_amd expects contiguous tensors or row-major 2-D views")
    return int(t.data_ptr())


@dataclass
class DeviceCSR:
    """CSR matrix resident on the device (row = source node)."""
    n_rows: int
    n_cols: int
    row_ptr: "object"   # torch.int32 [n_rows + 1]
    col_ind: "object"   # torch.int32 [nnz]
    val: "object"       # torch.float32 [nnz]

    @property
    def nnz(self) -> int:
        return int(self.col_ind.numel())

    @staticmethod
    def from_numpy(n_rows, n_cols, row_ptr, col_ind, val, device="cuda"):
        torch = _torch()
        return DeviceCSR(n_rows, n_cols,
                         torch.from_numpy(row_ptr).to(device=device, dtype=torch.int32),
                         torch.from_numpy(col_ind).to(device=device, dtype=torch.int32),
                         torch.from_numpy(val).to(device=device, dtype=torch.float32))

    def to_numpy(self):
        return (self.row_ptr.cpu().numpy(), self.col_ind.cpu().numpy(), self.val.cpu().numpy())


class SpmmPlan:
    """Degree-binned row schedule of one CSR structure (tg_spmm_plan_*)."""

    def __init__(self, row_ptr, n_rows: int, nnz_bound: int, max_f: int, chunk_nnz: int = 0,
                 stream=None, precision: int = PRECISION_EXACT):
        h = C.c_void_p()
        lib.check(lib.tg_spmm_plan_create(n_rows, nnz_bound, dptr(row_ptr), max_f, chunk_nnz,
                                          _on(stream), C.byref(h)))
        self.h = h
        self.row_ptr = row_ptr
        self.n_rows = n_rows
        if precision != PRECISION_EXACT:
            self.set_precision(precision)

    def set_precision(self, precision: int) -> None:
        """PRECISION_EXACT: every row one fma chain in nonzero order (the
        reference's order, bit-identical output); PRECISION_FAST: rows longer
        than the chunk summed from per-chunk partials."""
        lib.check(lib.tg_spmm_plan_set_precision(self.h, precision))

    @property
    def handle(self):
        return self.h

    def info(self):
        a, b, c = C.c_int64(), C.c_int64(), C.c_int64()
        lib.check(lib.tg_spmm_plan_info(self.h, C.byref(a), C.byref(b), C.byref(c)))
        return dict(n_chunks=a.value, n_split_rows=b.value, n_partials=c.value)

    def close(self):
        if getattr(self, "h", None) and self.h.value:
            lib.tg_spmm_plan_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _check_spmm_shapes(a: DeviceCSR, b):
    # ops.cpp:219-229
    if a.n_cols != b.shape[0]:
        raise InvalidArgument(1, f"spmm: dimension mismatch — A is ({a.n_rows}×{a.n_cols}, "
                                 f"SparseCSR) but B is ({b.shape[0]}×{b.shape[1]}, Dense). "
                                 f"Required: A.cols() == B.rows() ({a.n_cols} vs {b.shape[0]}).")


def spmm_epilogue(a: DeviceCSR, b, plan: SpmmPlan, bias=None, epilogue: int = EPI_NONE,
                  out=None, stream=None):
    """act(A * B + bias) in one pass (tg_spmm_execute_epilogue): the SpMM of
    GCNLayer::forward with add_bias and the activation fused into its store
    (reference layers.cpp:319-336); bit-identical to spmm, add_bias_, then
    relu_ / elu_."""
    torch = _torch()
    _check_spmm_shapes(a, b)
    f = b.shape[1]
    if out is None:
        out = torch.empty((a.n_rows, f), dtype=torch.float32, device=b.device)
    lib.check(lib.tg_spmm_execute_epilogue(plan.h, a.n_cols, f, dptr(a.row_ptr),
                                           dptr(a.col_ind), dptr(a.val), dptr(b), b.stride(0),
                                           dptr(out), out.stride(0), dptr(bias), epilogue,
                                           _on(stream)))
    return out


def spmm(a: DeviceCSR, b, plan: SpmmPlan | None = None, out=None, stream=None,
         precision: int = PRECISION_EXACT):
    """C = A * B (reference ops.cpp:198-297).  With a plan, the plan's
    precision applies; without one, `precision`: PRECISION_EXACT (the
    default) is the reference's summation order, bit-identical;
    PRECISION_FAST sums rows longer than 1,024 nonzeros from per-chunk
    partials."""
    torch = _torch()
    _check_spmm_shapes(a, b)
    f = b.shape[1]
    if out is None:
        out = torch.empty((a.n_rows, f), dtype=torch.float32, device=b.device)
    s = _on(stream)
    if plan is None:
        lib.check(lib.tg_spmm_ex(a.n_rows, a.n_cols, f, a.nnz, dptr(a.row_ptr), dptr(a.col_ind),
                                 dptr(a.val), dptr(b), b.stride(0), dptr(out), out.stride(0),
                                 precision, s))
    else:
        lib.check(lib.tg_spmm_execute(plan.h, a.n_cols, f, dptr(a.row_ptr), dptr(a.col_ind),
                                      dptr(a.val), dptr(b), b.stride(0), dptr(out),
                                      out.stride(0), s))
    return out


# ---------------------------------------------------------------------------
# Graph preprocessing
# ---------------------------------------------------------------------------
def edge_list_to_csr(src, dst, n_nodes: int, stream=None) -> DeviceCSR:
    """GraphLoader::edge_list_to_csr (graph_loader.cpp:211-281) on the device.
    Given a `stream` that is not the current one, returns finished arrays."""
    torch = _torch()
    dev = src.device
    e = int(src.numel())
    rp = torch.empty(n_nodes + 1, dtype=torch.int32, device=dev)
    ci = torch.empty(max(e, 1), dtype=torch.int32, device=dev)[:e]
    v = torch.empty(max(e, 1), dtype=torch.float32, device=dev)[:e]
    lib.check(lib.tg_edge_list_to_csr(n_nodes, e, dptr(src, torch.int32), dptr(dst, torch.int32),
                                      dptr(rp), ci.data_ptr(), v.data_ptr(), None, 0,
                                      _on(stream)))
    _finish(stream)
    return DeviceCSR(n_nodes, n_nodes, rp, ci, v)


def csr_validate(a: DeviceCSR, stream=None) -> None:
    """The checks of Tensor::sparse_csr (tensor.cpp:46-86); raises InvalidArgument."""
    lib.check(lib.tg_csr_validate(a.n_rows, a.n_cols, a.nnz, dptr(a.row_ptr),
                                  a.col_ind.data_ptr() if a.nnz else None, _on(stream)))


def _require_square(a: DeviceCSR, fn: str):
    if a.n_rows != a.n_cols:
        raise InvalidArgument(1, f"{fn}: A must be square — got ({a.n_rows}×{a.n_cols}).")


def _self_loop_outputs(a: DeviceCSR):
    torch = _torch()
    dev = a.row_ptr.device
    cap = a.nnz + a.n_rows
    return (torch.empty(a.n_rows + 1, dtype=torch.int32, device=dev),
            torch.empty(max(cap, 1), dtype=torch.int32, device=dev),
            torch.empty(max(cap, 1), dtype=torch.float32, device=dev))


def _trim(a: DeviceCSR, rp, ci, v, stream) -> DeviceCSR:
    _finish(stream)
    nnz = int(rp[-1].item()) if a.n_rows else 0
    return DeviceCSR(a.n_rows, a.n_cols, rp, ci[:nnz], v[:nnz])


def add_self_loops(a: DeviceCSR, stream=None) -> DeviceCSR:
    """add_self_loops (layers.cpp:71-144): A + I, bit-identical structure/values.
    Waits for `stream`, whose result's size it reads."""
    _require_square(a, "add_self_loops")
    rp, ci, v = _self_loop_outputs(a)
    lib.check(lib.tg_add_self_loops(a.n_rows, a.nnz, dptr(a.row_ptr), a.col_ind.data_ptr(),
                                    a.val.data_ptr(), dptr(rp), dptr(ci), dptr(v), None, 0,
                                    _on(stream)))
    return _trim(a, rp, ci, v, stream)


def gcn_norm(a: DeviceCSR, with_degrees: bool = False, stream=None):
    """gcn_norm (layers.cpp:158-208): D^-1/2 (A+I) D^-1/2.  Waits for `stream`,
    whose result's size it reads."""
    torch = _torch()
    _require_square(a, "gcn_norm")
    rp, ci, v = _self_loop_outputs(a)
    deg = torch.empty(max(a.n_rows, 1), dtype=torch.float32, device=rp.device)
    dis = torch.empty_like(deg)
    lib.check(lib.tg_gcn_norm(a.n_rows, a.nnz, dptr(a.row_ptr), a.col_ind.data_ptr(),
                              a.val.data_ptr(), dptr(rp), dptr(ci), dptr(v), dptr(deg), dptr(dis),
                              None, 0, _on(stream)))
    out = _trim(a, rp, ci, v, stream)
    return (out, deg[:a.n_rows], dis[:a.n_rows]) if with_degrees else out


def edge_softmax(a: DeviceCSR, stream=None) -> DeviceCSR:
    """edge_softmax (layers.cpp:768-822)."""
    torch = _torch()
    v = torch.zeros_like(a.val)
    lib.check(lib.tg_edge_softmax(a.n_rows, dptr(a.row_ptr), a.val.data_ptr(), v.data_ptr(),
                                  _on(stream)))
    return DeviceCSR(a.n_rows, a.n_cols, a.row_ptr, a.col_ind, v)


# ---------------------------------------------------------------------------
# Dense ops
# ---------------------------------------------------------------------------
def matmul(a, b, bias=None, epilogue: int = EPI_NONE, algo: int = GEMM_AUTO, out=None,
           stream=None):
    """matmul (ops.cpp:70-162) with an optional fused bias + activation."""
    torch = _torch()
    if a.shape[1] != b.shape[0]:
        # ops.cpp:90-97, the reference's text
        raise InvalidArgument(1, f"matmul: dimension mismatch — A is ({a.shape[0]}×{a.shape[1]})"
                                 f" but B is ({b.shape[0]}×{b.shape[1]}). Required: A.cols() == "
                                 f"B.rows() (both = {a.shape[1]} vs {b.shape[0]}).")
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    lib.check(lib.tg_matmul(m, k, n, dptr(a), a.stride(0), dptr(b), b.stride(0), dptr(out),
                            out.stride(0), dptr(bias), epilogue, algo, _on(stream)))
    return out


def _unary(name, x, *extra, stream=None):
    lib.check(getattr(lib, name)(x.numel(), dptr(x), *extra, _on(stream)))
    return x


def relu_(x, stream=None):
    return _unary("tg_relu", x, stream=stream)


def leaky_relu_(x, alpha: float = 0.01, stream=None):
    return _unary("tg_leaky_relu", x, alpha, stream=stream)


def elu_(x, alpha: float = 1.0, stream=None):
    return _unary("tg_elu", x, alpha, stream=stream)


def sigmoid_(x, stream=None):
    return _unary("tg_sigmoid", x, stream=stream)


def tanh_(x, stream=None):
    return _unary("tg_tanh", x, stream=stream)


def gelu_(x, stream=None):
    return _unary("tg_gelu", x, stream=stream)


def softmax_(x, stream=None):
    lib.check(lib.tg_softmax(x.shape[0], x.shape[1], dptr(x), _on(stream)))
    return x


def log_softmax_(x, stream=None):
    lib.check(lib.tg_log_softmax(x.shape[0], x.shape[1], dptr(x), _on(stream)))
    return x


def add_bias_(x, bias, stream=None):
    n = x.shape[1]
    if bias.dim() != 2 or bias.shape[0] != 1 or bias.shape[1] != n:
        shp = tuple(bias.shape) if bias.dim() == 2 else (1, bias.numel())
        raise InvalidArgument(1, f"add_bias: bias must be shape (1×{n}) to match X columns, "
                                 f"but got ({shp[0]}×{shp[1]}).")
    lib.check(lib.tg_add_bias(x.shape[0], n, dptr(x), dptr(bias), _on(stream)))
    return x


# ---------------------------------------------------------------------------
# Layers
# ---------------------------------------------------------------------------
def sage_aggregate(plan: SpmmPlan, a: DeviceCSR, h, agg: int = AGG_MEAN, stream=None):
    torch = _torch()
    out = torch.empty((a.n_rows, h.shape[1]), dtype=torch.float32, device=h.device)
    lib.check(lib.tg_sage_aggregate(plan.h, a.n_rows, h.shape[1], agg, dptr(a.row_ptr),
                                    a.col_ind.data_ptr(), dptr(h), h.stride(0), dptr(out),
                                    out.stride(0), _on(stream)))
    return out


def sage_forward(plan: SpmmPlan, a: DeviceCSR, h, w_neigh, w_self, bias=None,
                 act: int = ACT_RELU, post: int = POST_NONE, agg: int = AGG_MEAN,
                 dataflow: int = SAGE_AUTO, stream=None):
    """SAGELayer::forward (layers.cpp:538-752).  Given a `stream` that is not
    the current one, returns a finished result."""
    torch = _torch()
    f_in, f_out = w_neigh.shape
    out = torch.empty((a.n_rows, f_out), dtype=torch.float32, device=h.device)
    lib.check(lib.tg_sage_forward(plan.h, a.n_rows, f_in, f_out, agg, dptr(a.row_ptr),
                                  a.col_ind.data_ptr(), dptr(h), dptr(w_neigh), dptr(w_self),
                                  dptr(bias), act, post, dataflow, dptr(out), None, 0,
                                  _on(stream)))
    _finish(stream)
    return out


def gat_scores(wh, heads: int, f: int, att_l, att_r, stream=None):
    torch = _torch()
    n = wh.shape[0]
    src = torch.empty((n, heads), dtype=torch.float32, device=wh.device)
    dst = torch.empty_like(src)
    lib.check(lib.tg_gat_scores(n, heads, f, dptr(wh), wh.stride(0), dptr(att_l), dptr(att_r),
                                dptr(src), dptr(dst), _on(stream)))
    return src, dst


def gat_aggregate(plan: SpmmPlan, a_sl: DeviceCSR, wh, heads: int, f: int, src, dst,
                  slope: float = 0.2, bias=None, act: int = ACT_NONE, post: int = POST_NONE,
                  concat: bool = True, stream=None):
    """All heads of GATLayer::forward's fused edge pass (layers.cpp:1052-1112).
    Given a `stream` that is not the current one, returns a finished result."""
    torch = _torch()
    cols = heads * f if (concat or heads == 1) else f
    out = torch.empty((a_sl.n_rows, cols), dtype=torch.float32, device=wh.device)
    lib.check(lib.tg_gat_aggregate(plan.h, a_sl.n_rows, heads, f, dptr(a_sl.row_ptr),
                                   a_sl.col_ind.data_ptr(), dptr(wh), wh.stride(0), dptr(src),
                                   dptr(dst), slope, dptr(bias), act, post, int(concat),
                                   dptr(out), out.stride(0), None, 0, _on(stream)))
    _finish(stream)
    return out


# ---------------------------------------------------------------------------
# Expert layers: norm, routing, grouped and 8-bit products.  Tensors are
# float32, bfloat16 or float16 on one device, rows contiguous (any row stride).
# A call runs on `stream`, or on the current stream of its tensors' device;
# given a `stream` that is not the current one, it runs after what is queued on
# the current one and returns finished results.
# Outputs and workspaces are torch memory, so the calls can be captured.
# (Small calls are bound by this code: messages are made when they are needed.)
# ---------------------------------------------------------------------------
class _Torch:
    """What the calls below use of torch, looked up once."""

    def __init__(self):
        torch = _torch()
        self.torch = torch
        self.empty = torch.empty
        self.f32, self.i32, self.u8 = torch.float32, torch.int32, torch.uint8
        self.f8 = torch.float8_e4m3fn
        self.types = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16,
                      torch.float16: TYPE_F16}
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


_pt: _Torch | None = None


def _refuse(what: str, message: str):
    raise InvalidArgument(1, f"{what}: {message}")


def _device_call(fn):
    """The GPU of the first argument, or of the first tensor where that is None,
    is the current device for the call."""
    import functools
    name = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kwargs):
        global _pt
        if _pt is None:
            _pt = _Torch()
        first = args[0] if args else kwargs.get(name)
        if first is None:
            for first in (*args, *kwargs.values()):
                if hasattr(first, "get_device"):
                    break
            else:
                return fn(*args, **kwargs)   # Python's own message
        index = getattr(first, "q", first).get_device()
        if index < 0:
            raise ValueError("tinygnn_amd expects device (cuda) tensors")
        cuda = _pt.torch.cuda
        if index != cuda.current_device():
            with cuda.device(index):
                return fn(*args, **kwargs)
        return fn(*args, **kwargs)

    return call


def _stream_of(what: str, stream, first, *others) -> int:
    """The stream's handle; every tensor must be on the first one's GPU."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            if t.get_device() < 0:
                raise ValueError("tinygnn_amd expects device (cuda) tensors")
            _refuse(what, f"tensors on {first.device} and {t.device}.")
    if stream is not None or _pt.raw_stream is None:
        return _on(stream)
    return _pt.raw_stream(index)


def _type_of(what: str, t) -> int:
    code = _pt.types.get(t.dtype)
    if code is None:
        _refuse(what, f"float32, bfloat16 or float16 tensors expected, got {t.dtype}.")
    return code


def _rows_of(what: str, name: str, t):
    """Pointer and leading dimension of a matrix whose rows are contiguous."""
    if t.dim() != 2:
        _refuse(what, f"{name} must be a matrix, got {tuple(t.shape)}.")
    ld, step = t.stride()
    rows, cols = t.shape
    if step == 1 and ld >= cols:
        return t.data_ptr(), ld
    if step != 1 and cols > 1 and rows > 0:
        _refuse(what, f"{name} must have contiguous rows, got strides {t.stride()}.")
    if rows > 1 and cols > 0 and ld < cols:
        _refuse(what, f"{name} has overlapping rows (strides {t.stride()}).")
    return t.data_ptr(), max(ld, cols, 1) if rows > 1 else max(cols, 1)


def _flat(what: str, name: str, t, shape, dtype):
    """Pointer of a contiguous tensor of a given shape and type; None's."""
    if t is None:
        return None
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        _refuse(what, f"{name} must be contiguous, {tuple(shape)} {dtype}, got {tuple(t.shape)} "
                      f"{t.dtype}, strides {t.stride()}.")
    return t.data_ptr()


def _out(what: str, name: str, t, shape, like, dtype):
    """An output: `t` if it fits, or new memory; with pointer and leading
    dimension."""
    if t is None:
        t = _pt.empty(shape, dtype=dtype, device=like.device)
        return t, t.data_ptr(), max(shape[1], 1)
    if t.shape != shape or t.dtype is not dtype:
        _refuse(what, f"{name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}.")
    return (t, *_rows_of(what, name, t))


def _workspace(size: int, like):
    """`size` bytes of torch memory: the tensor and its pointer (0: none)."""
    if not size:
        return None, None
    t = _pt.empty(size, dtype=_pt.u8, device=like.device)
    return t, t.data_ptr()


def _norm_weights(what: str, x, gamma, beta):
    """gamma's and beta's pointers and type: both x's type, or both float32."""
    given = gamma if gamma is not None else beta
    kind = x.dtype if given is None else given.dtype
    if kind is not x.dtype and kind is not _pt.f32:
        _refuse(what, f"gamma and beta must be {x.dtype} or torch.float32, got {kind}.")
    cols = (x.shape[1],)
    return (_flat(what, "gamma", gamma, cols, kind), _flat(what, "beta", beta, cols, kind), kind)


@_device_call
def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5, with_stats: bool = False, out=None,
               stream=None):
    """The rows of x [rows, cols] to mean 0 and variance 1, times gamma, plus
    beta (tg_layer_norm).  gamma / beta: [cols] of x's type or float32.
    with_stats: (y, mean, rstd), float32 [rows], for layer_norm_backward."""
    what = "layer_norm"
    s = _stream_of(what, stream, x, gamma, beta, out)
    kind = _type_of(what, x)
    px, ldx = _rows_of(what, "x", x)
    rows, cols = x.shape
    pg, pb, wk = _norm_weights(what, x, gamma, beta)
    y, py, ldy = _out(what, "out", out, x.shape, x, x.dtype)
    mean = rstd = pm = pr = None
    if with_stats:
        mean = _pt.empty(rows, dtype=_pt.f32, device=x.device)
        rstd = _pt.empty(rows, dtype=_pt.f32, device=x.device)
        pm, pr = mean.data_ptr(), rstd.data_ptr()
    lib.check(lib.tg_layer_norm(rows, cols, kind, px, ldx, pg, pb, _pt.types[wk], eps, py, ldy,
                                pm, pr, s))
    _finish(stream)
    return (y, mean, rstd) if with_stats else y


@_device_call
def layer_norm_backward(dy, x, mean, rstd, gamma=None, out=None, stream=None):
    """(dx, dgamma, dbeta) of layer_norm from dy, its x, mean and rstd
    (tg_layer_norm_backward); dgamma and dbeta have gamma's type (x's without
    gamma).  out takes dx (it may be dy)."""
    what = "layer_norm_backward"
    s = _stream_of(what, stream, dy, x, mean, rstd, gamma, out)
    kind = _type_of(what, x)
    px, ldx = _rows_of(what, "x", x)
    rows, cols = x.shape
    if dy.shape != x.shape or dy.dtype is not x.dtype:
        _refuse(what, f"dy must be {tuple(x.shape)} {x.dtype}, got {tuple(dy.shape)} {dy.dtype}.")
    pdy, lddy = _rows_of(what, "dy", dy)
    pg, _, wk = _norm_weights(what, x, gamma, None)
    pm = _flat(what, "mean", mean, (rows,), _pt.f32)
    pr = _flat(what, "rstd", rstd, (rows,), _pt.f32)
    dx, pdx, lddx = _out(what, "out", out, x.shape, x, x.dtype)
    dgamma = _pt.empty(cols, dtype=wk, device=x.device)
    dbeta = _pt.empty(cols, dtype=wk, device=x.device)
    size = lib.tg_layer_norm_backward_workspace_size(rows, cols)
    ws, pws = _workspace(size, x)
    lib.check(lib.tg_layer_norm_backward(rows, cols, kind, pdy, lddy, px, ldx, pg, _pt.types[wk],
                                         pm, pr, pdx, lddx, dgamma.data_ptr(), dbeta.data_ptr(),
                                         pws, size, s))
    _finish(stream)
    return dx, dgamma, dbeta


@dataclass
class RoutePlan:
    """Rows in group order (tg_route, tg_route_plan).  Group g holds the
    places [offsets[g], offsets[g + 1]); rows[p] is the row at place p (-1 past
    the last group), position[t, j] the place of row t's j-th choice (-1: none)."""
    offsets: object
    rows: object
    position: object


@_device_call
def route(logits, k: int, renormalize: bool = False, stream=None):
    """Softmax of each row of logits [tokens, experts] and its k largest, with
    the plan of the rows by expert (tg_route): (weights float32 [tokens, k],
    experts int32 [tokens, k], RoutePlan).  A logit of -inf masks its expert;
    places without an expert hold -1 and weight 0."""
    what = "route"
    s = _stream_of(what, stream, logits)
    kind = _type_of(what, logits)
    pl, ld = _rows_of(what, "logits", logits)
    tokens, experts = logits.shape
    if not (1 <= k <= 32 and k <= experts <= 1024):
        _refuse(what, f"k must be between 1 and min(32, experts) and experts at most 1024, got "
                      f"k={k} of {experts}.")
    dev = logits.device
    weights = _pt.empty((tokens, k), dtype=_pt.f32, device=dev)
    ids = _pt.empty((tokens, k), dtype=_pt.i32, device=dev)
    offsets = _pt.empty(experts + 1, dtype=_pt.i32, device=dev)
    rows = _pt.empty(tokens * k, dtype=_pt.i32, device=dev)
    position = _pt.empty((tokens, k), dtype=_pt.i32, device=dev)
    size = lib.tg_route_workspace_size(tokens, experts, k)
    ws, pws = _workspace(size, logits)
    lib.check(lib.tg_route(tokens, experts, k, kind, pl, ld, 1 if renormalize else 0,
                           weights.data_ptr(), ids.data_ptr(), offsets.data_ptr(),
                           rows.data_ptr(), position.data_ptr(), pws, size, s))
    _finish(stream)
    return weights, ids, RoutePlan(offsets, rows, position)


@_device_call
def route_plan(ids, groups: int, stream=None) -> RoutePlan:
    """The plan of rows whose groups are known (tg_route_plan): ids int32
    [rows] (node types) or [rows, k]; an id outside [0, groups) is in none."""
    what = "route_plan"
    s = _stream_of(what, stream, ids)
    if ids.dim() not in (1, 2) or ids.dtype is not _pt.i32 or not ids.is_contiguous():
        _refuse(what, f"ids must be a contiguous int32 vector or matrix, got {tuple(ids.shape)} "
                      f"{ids.dtype}.")
    if not 1 <= groups <= 1024:
        _refuse(what, f"between 1 and 1024 groups, got {groups}.")
    n, k, dev = ids.numel(), ids.shape[1] if ids.dim() == 2 else 1, ids.device
    offsets = _pt.empty(groups + 1, dtype=_pt.i32, device=dev)
    rows = _pt.empty(n, dtype=_pt.i32, device=dev)
    position = _pt.empty(ids.shape, dtype=_pt.i32, device=dev)
    size = lib.tg_route_plan_workspace_size(n, groups)
    ws, pws = _workspace(size, ids)
    lib.check(lib.tg_route_plan(n, groups, max(k, 1), ids.data_ptr(), offsets.data_ptr(),
                                rows.data_ptr(), position.data_ptr(), pws, size, s))
    _finish(stream)
    return RoutePlan(offsets, rows, position)


@_device_call
def route_backward(dweights, logits, weights, experts, renormalize: bool = False, stream=None):
    """dlogits of route from the gradient of its weights (tg_route_backward)."""
    what = "route_backward"
    s = _stream_of(what, stream, dweights, logits, weights, experts)
    kind = _type_of(what, logits)
    pl, ld = _rows_of(what, "logits", logits)
    tokens, n = logits.shape
    if weights.dim() != 2:
        _refuse(what, f"weights must be [tokens, k], got {tuple(weights.shape)}.")
    k = weights.shape[1]
    shape = (tokens, k)
    pw = _flat(what, "weights", weights, shape, _pt.f32)
    pe = _flat(what, "experts", experts, shape, _pt.i32)
    pd = _flat(what, "dweights", dweights, shape, _pt.f32)
    out = _pt.empty((tokens, n), dtype=logits.dtype, device=logits.device)
    lib.check(lib.tg_route_backward(tokens, n, k, kind, pl, ld, 1 if renormalize else 0, pw, pe,
                                    pd, out.data_ptr(), n, s))
    _finish(stream)
    return out


def _places(what: str, position):
    if position.dim() != 2:
        _refuse(what, f"position must be [tokens, k], got {tuple(position.shape)}.")
    return _flat(what, "position", position, position.shape, _pt.i32)


@_device_call
def route_combine(y, position, weights=None, out=None, stream=None):
    """out[t] = sum over j of weights[t, j] * y[position[t, j]], weights of 1
    if None (tg_route_combine); a position of -1 adds nothing."""
    what = "route_combine"
    s = _stream_of(what, stream, y, position, weights, out)
    kind = _type_of(what, y)
    py, ldy = _rows_of(what, "y", y)
    pp = _places(what, position)
    tokens, k = position.shape
    rows, cols = y.shape
    pw = _flat(what, "weights", weights, position.shape, _pt.f32)
    o, po, ldo = _out(what, "out", out, (tokens, cols), y, y.dtype)
    lib.check(lib.tg_route_combine(tokens, k, cols, kind, py, rows, ldy, pp, pw, po, ldo, s))
    _finish(stream)
    return o


@_device_call
def route_combine_backward(dout, y, position, weights=None, out=None, stream=None):
    """(dy, dweights) of route_combine (tg_route_combine_backward).  out takes
    dy; rows of dy that no position names (those in no group of the plan) are
    not written."""
    what = "route_combine_backward"
    s = _stream_of(what, stream, dout, y, position, weights, out)
    kind = _type_of(what, y)
    py, ldy = _rows_of(what, "y", y)
    pp = _places(what, position)
    tokens, k = position.shape
    rows, cols = y.shape
    if dout.shape != (tokens, cols) or dout.dtype is not y.dtype:
        _refuse(what, f"dout must be {(tokens, cols)} {y.dtype}, got {tuple(dout.shape)} "
                      f"{dout.dtype}.")
    pd, lddo = _rows_of(what, "dout", dout)
    pw = _flat(what, "weights", weights, position.shape, _pt.f32)
    dy, pdy, lddy = _out(what, "out", out, y.shape, y, y.dtype)
    dw = _pt.empty((tokens, k), dtype=_pt.f32, device=y.device)
    lib.check(lib.tg_route_combine_backward(tokens, k, cols, kind, pd, lddo, py, rows, ldy, pp,
                                            pw, pdy, lddy, dw.data_ptr(), s))
    _finish(stream)
    return dy, dw


def _offsets(what: str, offsets):
    if offsets.dim() != 1 or offsets.numel() < 1:
        _refuse(what, f"offsets must be [groups + 1], got {tuple(offsets.shape)}.")
    return _flat(what, "offsets", offsets, offsets.shape, _pt.i32), offsets.numel() - 1


def _row_index(what: str, rows, x):
    """The rows' pointer and the number of rows of the product."""
    if rows is None:
        return None, x.shape[0]
    if rows.dim() != 1:
        _refuse(what, f"rows must be a vector, got {tuple(rows.shape)}.")
    return _flat(what, "rows", rows, rows.shape, _pt.i32), rows.numel()


def _matrices(what: str, w):
    """Leading dimension and stride of matrices [groups, rows, cols]."""
    groups, rows, cols = w.shape
    each, ld, step = w.stride()
    if w.numel():
        if step != 1 and cols > 1:
            _refuse(what, f"w must have contiguous rows, got strides {w.stride()}.")
        if rows > 1 and ld < cols:
            _refuse(what, f"w has overlapping rows (strides {w.stride()}).")
    return max(ld if rows > 1 else 0, cols, 1), each if groups > 1 else 0


@_device_call
def grouped_matmul(x, w, offsets, rows=None, bias=None, epilogue: int = EPI_NONE,
                   transpose: bool = False, out=None, stream=None):
    """y[p] = epilogue(x[p] @ w[g] + bias[g]) for the rows p of group g, those
    in [offsets[g], offsets[g + 1]) (tg_grouped_matmul); with rows, x[rows[p]]
    in the place of x[p].  w: [groups, k, n], or [groups, n, k] with transpose
    (the gradient of x: grouped_matmul(dy, w, offsets, transpose=True)).  Rows
    in no group are not written."""
    what = "grouped_matmul"
    s = _stream_of(what, stream, x, w, offsets, rows, bias, out)
    kind = _type_of(what, x)
    px, ldx = _rows_of(what, "x", x)
    po, groups = _offsets(what, offsets)
    pr, m = _row_index(what, rows, x)
    if w.dim() != 3 or w.dtype is not x.dtype or w.shape[0] != groups:
        _refuse(what, f"w must be [{groups}, k, n] {x.dtype}, got {tuple(w.shape)} {w.dtype}.")
    n, k = (w.shape[1], w.shape[2]) if transpose else (w.shape[2], w.shape[1])
    if x.shape[1] != k:
        _refuse(what, f"dimension mismatch: x has {x.shape[1]} columns, w {k}.")
    ldw, each = _matrices(what, w)
    pb = _flat(what, "bias", bias, (groups, n), x.dtype)
    y, py, ldy = _out(what, "out", out, (m, n), x, x.dtype)
    lib.check(lib.tg_grouped_matmul(m, k, n, groups, kind, px, x.shape[0], ldx, pr, po,
                                    w.data_ptr(), ldw, each, 1 if transpose else 0, pb, epilogue,
                                    py, ldy, s))
    _finish(stream)
    return y


@_device_call
def grouped_matmul_wgrad(x, dy, offsets, rows=None, bias: bool = False, stream=None):
    """(dw, dbias) of grouped_matmul from x (and rows) and the gradient before
    its epilogue (tg_grouped_matmul_wgrad): dw [groups, k, n], dbias [groups,
    n] or None."""
    what = "grouped_matmul_wgrad"
    s = _stream_of(what, stream, x, dy, offsets, rows)
    kind = _type_of(what, x)
    px, ldx = _rows_of(what, "x", x)
    po, groups = _offsets(what, offsets)
    pr, m = _row_index(what, rows, x)
    if dy.dim() != 2 or dy.shape[0] != m or dy.dtype is not x.dtype:
        _refuse(what, f"dy must be [{m}, n] {x.dtype}, got {tuple(dy.shape)} {dy.dtype}.")
    pd, lddy = _rows_of(what, "dy", dy)
    k, n = x.shape[1], dy.shape[1]
    dw = _pt.empty((groups, k, n), dtype=x.dtype, device=x.device)
    db = _pt.empty((groups, n), dtype=x.dtype, device=x.device) if bias else None
    size = lib.tg_grouped_matmul_wgrad_workspace_size(m, k, n, groups, kind)
    ws, pws = _workspace(size, x)
    lib.check(lib.tg_grouped_matmul_wgrad(m, k, n, groups, kind, px, x.shape[0], ldx, pr, pd,
                                          lddy, po, dw.data_ptr(),
                                          db.data_ptr() if bias else None, pws, size, s))
    _finish(stream)
    return dw, db


@dataclass
class BlockRows:
    """Rows in e4m3 with a scale for each 128 columns (tg_quantize): q
    float8_e4m3fn [rows, columns rounded up to 128], scale float32 [blocks,
    rows], and the columns they stand for."""
    q: object
    scale: object
    cols: int


@dataclass
class BlockWeight:
    """Weights in e4m3 with a scale for each 128 x 128 (tg_quantize_weight): q
    float8_e4m3fn [n, k rounded up to 128] and scale float32 [blocks of n,
    blocks of k], or [groups, ...] of both, and k."""
    q: object
    scale: object
    k: int


def _blocks(n: int) -> int:
    return -(-n // 128)


@_device_call
def quantize(x, stream=None) -> BlockRows:
    """x [rows, cols] in e4m3 with a scale for each row and 128 columns."""
    what = "quantize"
    s = _stream_of(what, stream, x)
    kind = _type_of(what, x)
    px, ldx = _rows_of(what, "x", x)
    rows, cols = x.shape
    blocks = _blocks(cols)
    q = _pt.empty((rows, blocks * 128), dtype=_pt.f8, device=x.device)
    scale = _pt.empty((blocks, rows), dtype=_pt.f32, device=x.device)
    lib.check(lib.tg_quantize(rows, cols, kind, px, ldx, q.data_ptr(), scale.data_ptr(), s))
    _finish(stream)
    return BlockRows(q, scale, cols)


@_device_call
def quantize_weight(w, transpose: bool = False, stream=None) -> BlockWeight:
    """w [k, n] or [groups, k, n] (transpose: [.., n, k]) in e4m3 with a scale
    for each 128 x 128 block, laid out for matmul_fp8 once."""
    what = "quantize_weight"
    s = _stream_of(what, stream, w)
    kind = _type_of(what, w)
    if w.dim() not in (2, 3):
        _refuse(what, f"w must be [k, n] or [groups, k, n], got {tuple(w.shape)}.")
    many = w.dim() == 3
    w3 = w if many else w[None]
    groups = w3.shape[0]
    n, k = (w3.shape[1], w3.shape[2]) if transpose else (w3.shape[2], w3.shape[1])
    ldw, each = _matrices(what, w3)
    q = _pt.empty((groups, n, _blocks(k) * 128), dtype=_pt.f8, device=w.device)
    scale = _pt.empty((groups, _blocks(n), _blocks(k)), dtype=_pt.f32, device=w.device)
    lib.check(lib.tg_quantize_weight(groups, k, n, kind, w.data_ptr(), ldw, each,
                                     1 if transpose else 0, q.data_ptr(), scale.data_ptr(), s))
    _finish(stream)
    return BlockWeight(q if many else q[0], scale if many else scale[0], k)


@_device_call
def matmul_fp8(x: BlockRows, w: BlockWeight, offsets=None, rows=None, bias=None,
               epilogue: int = EPI_NONE, dtype=None, out=None, stream=None):
    """The product of quantised rows and weights (tg_matmul_fp8), rounded once
    to `dtype` (float32 if None, or out's).  With offsets, w and bias [groups,
    n] are one for each group, as in grouped_matmul (rows too)."""
    what = "matmul_fp8"
    q, wq = x.q, w.q
    s = _stream_of(what, stream, q, x.scale, wq, w.scale, offsets, rows, bias, out)
    cols = x.cols
    kb = _blocks(cols)
    if cols != w.k:
        _refuse(what, f"dimension mismatch: x has {cols} columns, w {w.k}.")
    x_rows = q.shape[0]
    pq = _flat(what, "x.q", q, (x_rows, kb * 128), _pt.f8)
    ps = _flat(what, "x.scale", x.scale, (kb, x_rows), _pt.f32)
    if wq.dim() != (2 if offsets is None else 3):
        _refuse(what, f"w.q must be {'[n, k]' if offsets is None else '[groups, n, k]'}, got "
                      f"{tuple(wq.shape)}.")
    n = wq.shape[-2]
    if offsets is None:
        po, groups, lead = None, 1, ()
    else:
        po, groups = _offsets(what, offsets)
        lead = (groups,)
    pw = _flat(what, "w.q", wq, (*lead, n, kb * 128), _pt.f8)
    pws = _flat(what, "w.scale", w.scale, (*lead, _blocks(n), kb), _pt.f32)
    pr, m = _row_index(what, rows, q)
    kind = dtype or (out.dtype if out is not None else _pt.f32)
    code = _pt.types.get(kind)
    if code is None:
        _refuse(what, f"float32, bfloat16 or float16 results expected, got {kind}.")
    pb = _flat(what, "bias", bias, (*lead, n), kind)
    y, py, ldy = _out(what, "out", out, (m, n), q, kind)
    lib.check(lib.tg_matmul_fp8(m, cols, n, groups, pq, ps, x_rows, pr, po, pw, pws, code, pb,
                                epilogue, py, ldy, s))
    _finish(stream)
    return y


# ---------------------------------------------------------------------------
# Dense layers, and what a classifier answers and learns from: the conventions
# of the expert layers' calls above.
# ---------------------------------------------------------------------------
def _linear_weight(what: str, x, w, transpose: bool):
    """(n, k, pointer, leading dimension) of linear's w."""
    if w.dim() != 2 or w.dtype is not x.dtype:
        _refuse(what, f"w must be a {x.dtype} matrix, got {tuple(w.shape)} {w.dtype}.")
    n, k = w.shape if transpose else w.shape[::-1]
    if x.dim() != 2 or x.shape[1] != k:
        _refuse(what, f"dimension mismatch: x is {tuple(x.shape)}, w has {k} rows of x's columns.")
    return n, k, *_rows_of(what, "w", w)


def _like(what: str, name: str, t, shape, dtype):
    """Pointer and leading dimension of an input matrix of a given shape and
    type; None's."""
    if t is None:
        return None, 0
    if t.shape != shape or t.dtype is not dtype:
        _refuse(what, f"{name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}.")
    return _rows_of(what, name, t)


@_device_call
def linear(x, w, bias=None, epilogue: int = EPI_NONE, residual=None, transpose: bool = False,
           with_pre: bool = False, out=None, stream=None):
    """y = residual + epilogue(x @ w + bias) (tg_linear).  w: [k, n], or [n, k]
    with transpose; bias: [n]; residual: [rows, n]; epilogue: EPI_NONE, EPI_RELU,
    EPI_ELU, EPI_GELU or EPI_SILU.  All of x's type; rounded once.  with_pre:
    (y, pre), pre = x @ w + bias for linear_backward.  out may be the residual."""
    what = "linear"
    s = _stream_of(what, stream, x, w, bias, residual, out)
    kind = _type_of(what, x)
    n, k, pw, ldw = _linear_weight(what, x, w, transpose)
    px, ldx = _rows_of(what, "x", x)
    m = x.shape[0]
    pb = _flat(what, "bias", bias, (n,), x.dtype)
    pr, ldr = _like(what, "residual", residual, (m, n), x.dtype)
    y, py, ldy = _out(what, "out", out, (m, n), x, x.dtype)
    pre, pp, ldp = _out(what, "pre", None, (m, n), x, x.dtype) if with_pre else (None, None, 0)
    size = lib.tg_linear_workspace_size(m, k, n, kind)
    ws, pws = _workspace(size, x)
    lib.check(lib.tg_linear(m, k, n, kind, px, ldx, pw, ldw, 1 if transpose else 0, pb, epilogue,
                            pr, ldr, py, ldy, pp, ldp, pws, size, s))
    _finish(stream)
    return (y, pre) if with_pre else y


@_device_call
def linear_backward(dy, x, w, pre=None, epilogue: int = EPI_NONE, bias: bool = False,
                    transpose: bool = False, stream=None):
    """(dx, dw, dbias) of linear from dy, its x, w and, with an epilogue, pre
    (tg_linear_backward); dw in w's layout, dbias None unless bias.  The
    residual's gradient is dy."""
    what = "linear_backward"
    s = _stream_of(what, stream, dy, x, w, pre)
    kind = _type_of(what, x)
    n, k, pw, ldw = _linear_weight(what, x, w, transpose)
    px, ldx = _rows_of(what, "x", x)
    m = x.shape[0]
    pd, lddy = _like(what, "dy", dy, (m, n), x.dtype)
    if epilogue != EPI_NONE and pre is None:
        _refuse(what, "an epilogue's gradient needs pre (linear's with_pre).")
    pp, ldp = _like(what, "pre", pre, (m, n), x.dtype)
    dx = _pt.empty((m, k), dtype=x.dtype, device=x.device)
    dw = _pt.empty(w.shape, dtype=x.dtype, device=x.device)
    db = _pt.empty(n, dtype=x.dtype, device=x.device) if bias else None
    size = lib.tg_linear_backward_call_workspace_size(m, k, n, kind, epilogue, 1 if bias else 0)
    ws, pws = _workspace(size, x)
    lib.check(lib.tg_linear_backward(m, k, n, kind, pd, lddy, px, ldx, pw, ldw,
                                     1 if transpose else 0, pp, ldp, epilogue, dx.data_ptr(),
                                     max(k, 1), dw.data_ptr(), db.data_ptr() if bias else None,
                                     pws, size, s))
    _finish(stream)
    return dx, dw, db


@dataclass
class LogProbs:
    """What log_probs returns: value float32 [rows] (None without labels),
    entropy float32 [rows] or None, top_values float32 and top_ids int32 [rows,
    top] or None, and for log_probs_backward stats float32 [rows, 2] and the
    temperature."""
    value: object
    entropy: object
    top_values: object
    top_ids: object
    stats: object
    temperature: float


@_device_call
def log_probs(logits, labels=None, top: int = 0, entropy: bool = False, temperature: float = 1.0,
              stream=None) -> LogProbs:
    """Log probabilities of the classes labels (int32 [rows]; outside [0,
    classes): none, 0) under softmax(logits / temperature), the rows' entropy
    and their `top` likeliest classes (tg_log_probs)."""
    what = "log_probs"
    s = _stream_of(what, stream, logits, labels)
    kind = _type_of(what, logits)
    pl, ld = _rows_of(what, "logits", logits)
    rows, classes = logits.shape
    if not 0 <= top <= min(64, classes):
        _refuse(what, f"top must be between 0 and min(64, classes), got {top} of {classes}.")
    dev = logits.device
    py = _flat(what, "labels", labels, (rows,), _pt.i32)
    value = ent = top_values = top_ids = None
    pv = pe = ptv = pti = None
    if labels is not None:
        value = _pt.empty(rows, dtype=_pt.f32, device=dev)
        pv = value.data_ptr()
    if entropy:
        ent = _pt.empty(rows, dtype=_pt.f32, device=dev)
        pe = ent.data_ptr()
    if top:
        top_values = _pt.empty((rows, top), dtype=_pt.f32, device=dev)
        top_ids = _pt.empty((rows, top), dtype=_pt.i32, device=dev)
        ptv, pti = top_values.data_ptr(), top_ids.data_ptr()
    stats = _pt.empty((rows, 2), dtype=_pt.f32, device=dev)
    size = lib.tg_log_probs_workspace_size(rows, classes, top, kind)
    ws, pws = _workspace(size, logits)
    lib.check(lib.tg_log_probs(rows, classes, kind, pl, ld, py, temperature, top, pv, pe, ptv, pti,
                               stats.data_ptr(), pws, size, s))
    _finish(stream)
    return LogProbs(value, ent, top_values, top_ids, stats, temperature)


@_device_call
def log_probs_backward(dvalue, logits, labels, result: LogProbs, dentropy=None,
                       temperature: float | None = None, out=None, stream=None):
    """dlogits of log_probs from the gradients of its value (float32 [rows]; None:
    of none, labels None too) and of its entropy (tg_log_probs_backward).  out takes
    dlogits (it may be logits)."""
    what = "log_probs_backward"
    first = logits if dvalue is None else dvalue
    s = _stream_of(what, stream, first, logits, labels, result.stats, result.entropy, dentropy, out)
    kind = _type_of(what, logits)
    pl, ld = _rows_of(what, "logits", logits)
    rows, classes = logits.shape
    if temperature is not None and temperature != result.temperature:
        _refuse(what, f"temperature {temperature} is not log_probs' {result.temperature}.")
    if (dvalue is None) != (labels is None):
        _refuse(what, "dvalue and labels go together.")
    pd = _flat(what, "dvalue", dvalue, (rows,), _pt.f32)
    py = _flat(what, "labels", labels, (rows,), _pt.i32)
    pst = _flat(what, "stats", result.stats, (rows, 2), _pt.f32)
    ph = _flat(what, "dentropy", dentropy, (rows,), _pt.f32)
    if ph is not None and result.entropy is None:
        _refuse(what, "dentropy needs log_probs' entropy.")
    pe = _flat(what, "entropy", result.entropy, (rows,), _pt.f32) if ph is not None else None
    d, po, ldo = _out(what, "out", out, logits.shape, logits, logits.dtype)
    lib.check(lib.tg_log_probs_backward(rows, classes, kind, pl, ld, py, result.temperature, pst,
                                        pe, pd, ph, po, ldo, s))
    _finish(stream)
    return d


@_device_call
def distill(logits, teacher, ids, temperature: float = 1.0, dloss=None, out=None, stream=None):
    """The divergence of softmax(logits / temperature) from a teacher's k top
    logits [rows, k] of the classes ids (int32; outside [0, classes): no place),
    softmax(teacher / temperature) over them: loss float32 [rows] (tg_distill).
    With dloss (float32 [rows], the gradient of each row's loss): (loss,
    dlogits); out takes dlogits (it may be logits)."""
    what = "distill"
    s = _stream_of(what, stream, logits, teacher, ids, dloss, out)
    kind = _type_of(what, logits)
    pl, ld = _rows_of(what, "logits", logits)
    rows, classes = logits.shape
    tk = _type_of(what, teacher)
    if teacher.dim() != 2 or teacher.shape[0] != rows or not 1 <= teacher.shape[1] <= 256:
        _refuse(what, f"teacher must be [{rows}, k] with k between 1 and 256, got "
                      f"{tuple(teacher.shape)}.")
    pt = _flat(what, "teacher", teacher, teacher.shape, teacher.dtype)
    pi = _flat(what, "ids", ids, teacher.shape, _pt.i32)
    pd = _flat(what, "dloss", dloss, (rows,), _pt.f32)
    d, po, ldo = None, None, 0
    if dloss is not None:
        d, po, ldo = _out(what, "out", out, logits.shape, logits, logits.dtype)
    elif out is not None:
        _refuse(what, "out takes the gradient, which needs dloss.")
    loss = _pt.empty(rows, dtype=_pt.f32, device=logits.device)
    k = teacher.shape[1]
    size = lib.tg_distill_workspace_size(rows, classes, k, kind)
    ws, pws = _workspace(size, logits)
    lib.check(lib.tg_distill(rows, classes, k, kind, pl, ld, tk, pt, pi, temperature,
                             loss.data_ptr(), pd, po, ldo, pws, size, s))
    _finish(stream)
    return loss if dloss is None else (loss, d)


# ---------------------------------------------------------------------------
# Model
# ---------------------------------------------------------------------------
class Model:
    """tinygnn::Model (model.hpp:89-164) on the device, over tg_model_*."""

    def __init__(self):
        h = C.c_void_p()
        lib.check(lib.tg_model_create(C.byref(h)))
        self.h = h

    def add_gcn_layer(self, in_f, out_f, bias=True, act=ACT_RELU, post=POST_NONE) -> int:
        i = C.c_int64()
        lib.check(lib.tg_model_add_gcn_layer(self.h, in_f, out_f, int(bias), act, post,
                                             C.byref(i)))
        return i.value

    def add_sage_layer(self, in_f, out_f, agg=AGG_MEAN, bias=True, act=ACT_RELU,
                       post=POST_NONE) -> int:
        i = C.c_int64()
        lib.check(lib.tg_model_add_sage_layer(self.h, in_f, out_f, agg, int(bias), act, post,
                                              C.byref(i)))
        return i.value

    def add_gat_layer(self, in_f, out_f, num_heads=1, concat=True, neg_slope=0.2, bias=True,
                      act=ACT_NONE, post=POST_NONE) -> int:
        i = C.c_int64()
        lib.check(lib.tg_model_add_gat_layer(self.h, in_f, out_f, num_heads, int(concat),
                                             neg_slope, int(bias), act, post, C.byref(i)))
        return i.value

    def num_layers(self) -> int:
        n = C.c_int64()
        lib.check(lib.tg_model_num_layers(self.h, C.byref(n)))
        return n.value

    def output_cols(self) -> int:
        n = C.c_int64()
        lib.check(lib.tg_model_output_cols(self.h, C.byref(n)))
        return n.value

    def set_tensor(self, name: str, array) -> None:
        import numpy as np
        a = np.ascontiguousarray(array, dtype=np.float32)
        if a.ndim == 1:
            a = a.reshape(1, -1)
        lib.check(lib.tg_model_set_tensor(self.h, name.encode(), a.shape[0], a.shape[1],
                                          a.ctypes.data_as(C.c_void_p)))

    def load_weights(self, weights=None) -> None:
        """Model::load_weights (model.cpp:252-305).  ``weights`` is a dict of
        name -> array, a :class:`WeightFile`, or the path of a TGNN weight
        file (model.cpp:252-255).  Only the given tensors are looked up, as
        the reference looks up only the WeightFile it is given."""
        if isinstance(weights, (str, bytes)) or hasattr(weights, "__fspath__"):
            weights = load_weight_file(weights)
        if isinstance(weights, WeightFile):
            weights = weights.tensors
        lib.check(lib.tg_model_clear_tensors(self.h))
        for k, v in (weights or {}).items():
            self.set_tensor(k, v)
        lib.check(lib.tg_model_load_weights(self.h))

    def set_sage_dataflow(self, dataflow: int) -> None:
        lib.check(lib.tg_model_set_sage_dataflow(self.h, dataflow))

    def set_precision(self, precision: int) -> None:
        """PRECISION_FAST (default) or PRECISION_EXACT (the reference's
        operation order: bit-identical GCN / SAGE outputs)."""
        lib.check(lib.tg_model_set_precision(self.h, precision))

    def set_blocking(self, rows_per_block: int = -1) -> None:
        """Column blocking of the GCN / SAGE-mean / GAT aggregations (both
        forward modes; exact precision: only for rows in column order, keeping
        the reference's summation order): rows_per_block source nodes per
        block, 0 = off, -1 = the default (equal blocks of at most 23552 rows
        for weighted passes over A + I -- GAT, exact or weighted GCN -- and
        38912 for passes without values -- SAGE's mean over A, fast GCN over a
        unit-valued A + I -- on graphs dense enough to pay)."""
        lib.check(lib.tg_model_set_blocking(self.h, rows_per_block))

    def blocking_info(self) -> dict:
        """The column blocking the last forward used (tg_model_blocking_info):
        blocks and lane-group columns of A + I's and A's blocked copies,
        whether A + I's was split from A directly (sl_direct), and whether
        each copy is prepared for the output-resident passes (resident_sl,
        resident_raw)."""
        v = [C.c_int64() for _ in range(6)]
        lib.check(lib.tg_model_blocking_info(self.h, *[C.byref(x) for x in v]))
        return dict(blocks_sl=v[0].value, cols_sl=v[1].value, blocks_raw=v[2].value,
                    cols_raw=v[3].value, sl_direct=bool(v[4].value),
                    resident_sl=bool(v[5].value & 1), resident_raw=bool(v[5].value & 2))

    def set_self_loop_split(self, direct: bool = True) -> None:
        """Whether a fast GCN-only model splits its blocked A + I from A
        directly when A allows it (tg_model_set_self_loop_split; the same
        outputs bit for bit either way).  Drops the cached state."""
        self._adj_key = None
        lib.check(lib.tg_model_set_self_loop_split(self.h, 1 if direct else 0))

    def set_resident_passes(self, on: bool = True) -> None:
        """Whether the fast blocked aggregations without values (SAGE mean,
        the factored GCN) run as output-resident passes, one launch with the
        output tile in LDS, or one pass per column block
        (tg_model_set_resident_passes).  Drops the cached state."""
        self._adj_key = None
        lib.check(lib.tg_model_set_resident_passes(self.h, 1 if on else 0))

    def invalidate(self) -> None:
        """Forgets the cached adjacency state (tg_model_invalidate)."""
        self._adj_key = None
        lib.check(lib.tg_model_invalidate(self.h))

    @staticmethod
    def _adjacency_key(adj: DeviceCSR):
        return (adj.n_rows, adj.row_ptr, adj.col_ind, adj.val, adj.row_ptr._version,
                adj.col_ind._version, adj.val._version)

    def _cache_valid(self, key) -> bool:
        old = getattr(self, "_adj_key", None)
        if old is None:
            return False
        return (old[0] == key[0] and all(a is b for a, b in zip(old[1:4], key[1:4]))
                and old[4:] == key[4:])

    def forward(self, adj: DeviceCSR, x, mode: int = FORWARD_REFERENCE, out=None, stream=None):
        """Model::forward (model.cpp:359-439).

        ``mode=FORWARD_REFERENCE`` (the default) recomputes gcn_norm /
        add_self_loops and the row plans on every call, as the reference
        does (model.cpp:373-381).  ``mode=FORWARD_CACHED`` reuses them when
        ``adj`` holds the same ``row_ptr`` / ``col_ind`` / ``val`` tensor
        objects as the previous forward, at the same torch versions (an
        in-place edit through torch bumps the version; a new tensor is a
        different object).  The model keeps references to those three
        tensors, so their memory cannot be handed to another graph while the
        cache refers to it.  Writes that torch does not track (through raw
        device pointers) must be followed by :meth:`invalidate`."""
        torch = _torch()
        if out is None:
            out = torch.empty((adj.n_rows, self.output_cols()), dtype=torch.float32,
                              device=x.device)
        key = self._adjacency_key(adj)
        if mode == FORWARD_CACHED and not self._cache_valid(key):
            lib.check(lib.tg_model_invalidate(self.h))
        self._adj_key = None
        lib.check(lib.tg_model_forward(self.h, adj.n_rows, adj.nnz, dptr(adj.row_ptr),
                                       adj.col_ind.data_ptr(), adj.val.data_ptr(), x.shape[1],
                                       dptr(x), dptr(out), mode, _on(stream)))
        self._adj_key = key
        return out

    @staticmethod
    def from_spec(spec, weights: dict | None = None) -> "Model":
        """Builds a model from layer dicts (see tinygnn_amd.synth.spec_*)."""
        m = Model()
        for l in spec:
            t = l["type"]
            if t == "gcn":
                m.add_gcn_layer(l["in"], l["out"], l.get("bias", True), l.get("act", ACT_RELU),
                                l.get("post", POST_NONE))
            elif t == "sage":
                m.add_sage_layer(l["in"], l["out"], l.get("agg", AGG_MEAN), l.get("bias", True),
                                 l.get("act", ACT_RELU), l.get("post", POST_NONE))
            elif t == "gat":
                m.add_gat_layer(l["in"], l["out"], l.get("heads", 1), l.get("concat", True),
                                l.get("slope", 0.2), l.get("bias", True), l.get("act", ACT_NONE),
                                l.get("post", POST_NONE))
            else:
                raise ValueError(t)
        if weights is not None:
            m.load_weights(weights)
        return m

    def close(self):
        if getattr(self, "h", None) and self.h.value:
            lib.tg_model_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------------------
# Ingestion: CSV graphs (GraphLoader, graph_loader.cpp:61-326), the TGNN
# weight file (model.cpp:134-185) and the Cora binary (model.cpp:49-129).
# ---------------------------------------------------------------------------
class CsvText:
    """A CSV text indexed into lines on the device (tg_csv_open / tg_csv_index).

    ``CsvText.open(path)`` reads the file into device memory;
    ``CsvText.from_device(u8_tensor, name)`` indexes bytes already there (the
    tensor is kept alive with the handle)."""

    def __init__(self, handle, keep=None):
        self.h = handle
        self._keep = keep
        n, hdr = C.c_int64(), C.c_int()
        lib.check(lib.tg_csv_info(self.h, C.byref(n), C.byref(hdr)))
        self.n_lines, self.has_header = int(n.value), bool(hdr.value)

    @classmethod
    def open(cls, path, stream=None) -> "CsvText":
        h = C.c_void_p()
        lib.check(lib.tg_csv_open(os.fsencode(path), C.byref(h), _on(stream)))
        return cls(h)

    @classmethod
    def from_device(cls, text, name: str = "", stream=None) -> "CsvText":
        torch = _torch()
        if text.dtype != torch.uint8 or not text.is_contiguous():
            raise ValueError("CsvText.from_device expects a contiguous uint8 device tensor")
        h = C.c_void_p()
        lib.check(lib.tg_csv_index(dptr(text), text.numel(), name.encode(), C.byref(h),
                                   _on(stream)))
        return cls(h, keep=text)

    @property
    def n_data(self) -> int:
        return self.n_lines - int(self.has_header)

    def parse_edges(self, device=None, stream=None):
        """GraphLoader::parse_edges (graph_loader.cpp:61-107): (src, dst,
        max_id) with int32 device tensors of one entry per data line."""
        torch = _torch()
        device = device or torch.device("cuda", torch.cuda.current_device())
        n = max(self.n_data, 0)
        src = torch.empty(max(n, 1), dtype=torch.int32, device=device)[:n]
        dst = torch.empty(max(n, 1), dtype=torch.int32, device=device)[:n]
        mx = C.c_int64()
        lib.check(lib.tg_csv_parse_edges(self.h, src.data_ptr(), dst.data_ptr(), C.byref(mx),
                                         _on(stream)))
        return src, dst, int(mx.value)

    def feature_shape(self, stream=None):
        rows, cols = C.c_int64(), C.c_int64()
        lib.check(lib.tg_csv_feature_shape(self.h, C.byref(rows), C.byref(cols),
                                           _on(stream)))
        return int(rows.value), int(cols.value)

    def parse_features(self, n_rows: int | None = None, device=None, stream=None):
        """GraphLoader::parse_features (graph_loader.cpp:112-206): a
        [rows x cols] float32 device tensor (``n_rows`` > rows zero-pads)."""
        torch = _torch()
        device = device or torch.device("cuda", torch.cuda.current_device())
        rows, cols = self.feature_shape(stream)
        n_rows = rows if n_rows is None else int(n_rows)
        out = torch.empty((n_rows, cols), dtype=torch.float32, device=device)
        lib.check(lib.tg_csv_parse_features(self.h, out.data_ptr() if out.numel() else None,
                                            n_rows, cols, _on(stream)))
        return out

    def close(self):
        if getattr(self, "h", None) and self.h.value:
            lib.tg_csv_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def parse_edges(path, stream=None):
    """GraphLoader::parse_edges on the device: (src, dst) int32 tensors."""
    t = CsvText.open(path, stream)
    try:
        src, dst, _ = t.parse_edges(stream=stream)
        return src, dst
    finally:
        t.close()


def parse_features(path, stream=None):
    """GraphLoader::parse_features on the device: [rows x cols] float32."""
    t = CsvText.open(path, stream)
    try:
        return t.parse_features(stream=stream)
    finally:
        t.close()


@dataclass
class GraphData:
    """GraphData (graph_loader.hpp:17-23): adjacency (values 1.0) and
    features, both on the device."""
    adjacency: DeviceCSR
    node_features: object
    num_nodes: int
    num_edges: int
    num_features: int


def load_graph(edges_path, features_path, stream=None) -> GraphData:
    """GraphLoader::load (graph_loader.cpp:286-326): edges, then features,
    num_nodes = max(largest endpoint + 1, feature rows), the CSR built on the
    device and the features zero-padded to num_nodes rows."""
    te = CsvText.open(edges_path, stream)
    try:
        src, dst, max_id = te.parse_edges(stream=stream)
    finally:
        te.close()
    tf = CsvText.open(features_path, stream)
    try:
        rows, cols = tf.feature_shape(stream)
        n_edges = int(src.numel())
        num_nodes = max(max_id + 1 if n_edges else 0, rows)
        x = tf.parse_features(n_rows=num_nodes, stream=stream)
    finally:
        tf.close()
    adj = edge_list_to_csr(src, dst, num_nodes, stream=stream)
    return GraphData(adj, x, num_nodes, n_edges, cols)


@dataclass
class WeightFile:
    """WeightFile (model.hpp:76-79): test accuracy and named host tensors."""
    test_accuracy: float
    tensors: dict


def load_weight_file(path) -> WeightFile:
    """load_weight_file (model.cpp:134-185), read by the native library."""
    import numpy as np
    h = C.c_void_p()
    lib.check(lib.tg_weights_open(os.fsencode(path), C.byref(h)))
    try:
        n, acc = C.c_int64(), C.c_float()
        lib.check(lib.tg_weights_info(h, C.byref(n), C.byref(acc)))
        tensors = {}
        for i in range(n.value):
            name, nlen, rows, cols, data = (C.c_void_p(), C.c_int64(), C.c_int64(), C.c_int64(),
                                            C.c_void_p())
            lib.check(lib.tg_weights_tensor(h, i, C.byref(name), C.byref(nlen), C.byref(rows),
                                            C.byref(cols), C.byref(data)))
            key = C.string_at(name.value, nlen.value).decode("utf-8", "surrogateescape")
            count = rows.value * cols.value
            arr = np.empty((rows.value, cols.value), np.float32)
            if count:
                C.memmove(arr.ctypes.data, data.value, count * 4)
            tensors[key] = arr
        return WeightFile(float(acc.value), tensors)
    finally:
        lib.tg_weights_destroy(h)


def save_weight_file(path, tensors: dict, test_accuracy: float = 0.0) -> None:
    """Writes a TGNN weight file, version 1 (model.hpp:22-33): the format
    load_weight_file reads.  Tensors are 2-D float32 (1-D arrays are written
    as one row), in the dict's order."""
    import struct
    import numpy as np
    with open(path, "wb") as f:
        f.write(b"TGNN")
        f.write(struct.pack("<IfI", 1, float(test_accuracy), len(tensors)))
        for name, arr in tensors.items():
            a = np.ascontiguousarray(arr, dtype="<f4")
            if a.ndim == 1:
                a = a.reshape(1, -1)
            if a.ndim != 2:
                raise ValueError(f"{name}: expected a 1-D or 2-D array")
            nb = name.encode("utf-8", "surrogateescape")
            f.write(struct.pack("<I", len(nb)) + nb + struct.pack("<II", *a.shape))
            f.write(a.tobytes())


@dataclass
class CoraData:
    """CoraData (model.hpp:50-62): the graph on the device, labels and masks
    on the host."""
    num_nodes: int
    num_features: int
    num_classes: int
    num_edges: int
    adjacency: DeviceCSR
    features: object
    labels: object
    train_mask: object
    val_mask: object
    test_mask: object


def load_cora_binary(path, stream=None) -> CoraData:
    """load_cora_binary (model.cpp:49-129): the file read by the native
    library, features uploaded, adjacency built on the device."""
    import numpy as np
    torch = _torch()
    dev = torch.device("cuda", torch.cuda.current_device())
    h = C.c_void_p()
    lib.check(lib.tg_cora_open(os.fsencode(path), C.byref(h)))
    try:
        n, f, c, e = C.c_int64(), C.c_int64(), C.c_int64(), C.c_int64()
        lib.check(lib.tg_cora_info(h, C.byref(n), C.byref(f), C.byref(c), C.byref(e)))
        n, f, c, e = n.value, f.value, c.value, e.value
        x = torch.empty((n, f), dtype=torch.float32, device=dev)
        rp = torch.empty(n + 1, dtype=torch.int32, device=dev)
        ci = torch.empty(max(e, 1), dtype=torch.int32, device=dev)[:e]
        v = torch.empty(max(e, 1), dtype=torch.float32, device=dev)[:e]
        lib.check(lib.tg_cora_upload(h, x.data_ptr() if x.numel() else None, rp.data_ptr(),
                                     ci.data_ptr(), v.data_ptr(), _on(stream)))
        ptrs = [C.c_void_p() for _ in range(4)]
        lib.check(lib.tg_cora_host(h, *[C.byref(p) for p in ptrs]))
        labels = np.empty(n, np.int32)
        masks = [np.empty(n, np.uint8) for _ in range(3)]
        if n:
            C.memmove(labels.ctypes.data, ptrs[0].value, n * 4)
            for m, p in zip(masks, ptrs[1:]):
                C.memmove(m.ctypes.data, p.value, n)
        return CoraData(n, f, c, e, DeviceCSR(n, n, rp, ci, v), x, labels, *masks)
    finally:
        lib.tg_cora_destroy(h)
