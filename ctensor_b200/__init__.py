"""ctensor_b200 — B200 (sm_100a) elementwise / broadcast / reduction operators behind a C ABI.

The product is ``libctb200.so`` (sources in ``ctensor_b200/csrc``, interface in
``include/ctb200.h``).  This module is the thin Python binding used by the tests and the
benchmark: it loads the library with ctypes, wraps device memory held by torch tensors in
``ctb_view`` structs and calls the C entry points on torch's current CUDA stream.  torch only
provides memory, streams and process groups; no torch operator computes a result here.

There is no CPU fallback: importing works anywhere, but every operator call needs the built
library and a CUDA device and raises otherwise.
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG_DIR, "libctb200.so")
MAX_DIMS = 8

# dtypes (reference DType numbering)
F32, I32, F64, U8, U16, U32, U64, I8, I16, I64, BOOL = range(11)        # the reference's DType numbering
# binary operators
ADD, SUB, MUL, DIV, LT, LE, GT, GE, EQ, NE, POW = range(11)
# unary operators
(ADD_S, SUB_S, RSUB_S, MUL_S, DIV_S, RDIV_S, POW_S, RPOW_S, LT_S, LE_S, GT_S, GE_S, EQ_S, NE_S,
 ABS, RELU, EXP, LOG, TANH, SIGMOID, SQRT, GELU_TANH,
 SIN, COS, TAN, ASIN, ACOS, ATAN, SINH, COSH, SOFTPLUS) = range(31)
# reductions
SUM, MEAN, MAX, MIN, VAR, ARGMAX = range(6)
DIM_FULL = -1
# norms of residual_norm
NORM_NONE, NORM_LAYER, NORM_RMS = range(3)

STATUS_NAMES = {0: "CTB_OK", 1: "CTB_ERR_NULL", 2: "CTB_ERR_SHAPE", 3: "CTB_ERR_DTYPE",
                4: "CTB_ERR_DIM", 5: "CTB_ERR_ARG", 6: "CTB_ERR_CUDA", 7: "CTB_ERR_WORKSPACE",
                8: "CTB_ERR_LIMIT"}

# every symbol include/ctb200.h declares
EXPORTED_SYMBOLS = [
    "ctb_abi_version", "ctb_last_error", "ctb_device_count", "ctb_alloc", "ctb_free", "ctb_sync",
    "ctb_alloc_managed", "ctb_free_managed", "ctb_set_device", "ctb_device_sync",
    "ctb_binary", "ctb_unary", "ctb_copy_strided", "ctb_reduce", "ctb_reduce_workspace_bytes",
    "ctb_reduce_ws", "ctb_reduce_dim_noalloc", "ctb_reduce_full_partial", "ctb_finalize_full", "ctb_softmax_lastdim",
    "ctb_layernorm_lastdim", "ctb_binary_host", "ctb_unary_host", "ctb_reduce_host",
    "ctb_log_softmax_lastdim", "ctb_gather", "ctb_accumulate_grad", "ctb_sgd_step", "ctb_adam_step",
    "ctb_copy_into", "ctb_cat", "ctb_channel_moments", "ctb_batchnorm_apply",
    "ctb_matmul", "ctb_optimizer_step",
    "ctb_pool_alloc_managed", "ctb_pool_free_managed", "ctb_pool_trim", "ctb_pool_set_limit", "ctb_pool_stats",
    "ctb_prefetch_managed",
    "ctb_div_backward", "ctb_tanh_backward", "ctb_cross_entropy", "ctb_cross_entropy_backward",
    "ctb_shard_range", "ctb_comm_init_all", "ctb_comm_size", "ctb_comm_device", "ctb_comm_stream", "ctb_comm_sync",
    "ctb_comm_destroy", "ctb_allreduce", "ctb_full_reduce_sharded", "ctb_matmul_tc",
    "ctb_score_softmax", "ctb_score_softmax_workspace_bytes", "ctb_score_softmax_backward",
    "ctb_residual_norm", "ctb_residual_norm_workspace_bytes", "ctb_residual_norm_backward",
    "ctb_grad_norm_workspace_bytes", "ctb_grad_norm", "ctb_clip_grad_norm",
]


class CtbError(RuntimeError):
    """A C-ABI call returned a non-zero status.  ``code`` is the ctb_status value; the message
    is the library's, which equals the reference's exception text for the same mistake."""

    def __init__(self, code: int, message: str):
        super().__init__(f"{STATUS_NAMES.get(code, code)}: {message}")
        self.code = code
        self.message = message


class OptimizerHyper(ctypes.Structure):
    """struct ctb_optimizer_hyper."""
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "alpha")]


(OPT_SGD, OPT_ADAM, OPT_ADAMW, OPT_ADAMAX, OPT_NADAM, OPT_RADAM, OPT_RMSPROP, OPT_ADAGRAD, OPT_LION) = range(9)


class CScoreRules(ctypes.Structure):
    """struct ctb_score_rules."""
    _fields_ = [("scale", ctypes.c_double), ("cap", ctypes.c_double), ("causal", ctypes.c_int32), ("reserved", ctypes.c_int32)] + [
        (n, ctypes.c_void_p) for n in ("query_start", "key_lengths", "prefix", "query_docs", "key_docs", "slopes")]


class CResidualNormParams(ctypes.Structure):
    """struct ctb_residual_norm_params."""
    _fields_ = [("post_kind", ctypes.c_int32), ("pre_kind", ctypes.c_int32), ("post_eps", ctypes.c_double),
                ("pre_eps", ctypes.c_double), ("scale", ctypes.c_double)] + [
        (n, ctypes.c_void_p) for n in ("post_weight", "post_bias", "pre_weight", "pre_bias")]


class CResidualNormGrads(ctypes.Structure):
    """struct ctb_residual_norm_grads."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")]


class PoolInfo(ctypes.Structure):
    """struct ctb_pool_info."""
    _fields_ = [("live_bytes", ctypes.c_size_t), ("cached_bytes", ctypes.c_size_t), ("cached_blocks", ctypes.c_size_t),
                ("hits", ctypes.c_uint64), ("misses", ctypes.c_uint64), ("trims", ctypes.c_uint64)]


class View(ctypes.Structure):
    """struct ctb_view."""
    _fields_ = [("base", ctypes.c_void_p), ("offset", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("ndim", ctypes.c_int32),
                ("shape", ctypes.c_int64 * MAX_DIMS), ("stride", ctypes.c_int64 * MAX_DIMS)]


def make_view(base: int, dtype: int, shape: Sequence[int], strides: Sequence[int], offset: int = 0) -> View:
    if len(shape) > MAX_DIMS:
        raise CtbError(5, f"ndim {len(shape)} not in 0..{MAX_DIMS}")
    v = View()
    v.base = base
    v.offset = offset
    v.dtype = dtype
    v.ndim = len(shape)
    for i, (s, st) in enumerate(zip(shape, strides)):
        v.shape[i] = s
        v.stride[i] = st
    return v


_lib = None


def lib() -> ctypes.CDLL:
    """Load libctb200.so (built in-tree by ``ctensor_b200.build``)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it first (python -c 'import __graft_entry__ as g; g.build()' "
            "or python -m ctensor_b200.build).  There is no CPU fallback.")
    L = ctypes.CDLL(LIB_PATH)
    vp, vd, i32, i64 = ctypes.POINTER(View), ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    L.ctb_abi_version.restype = i32
    L.ctb_last_error.restype = ctypes.c_char_p
    L.ctb_device_count.restype = i32
    L.ctb_alloc.argtypes = [ctypes.POINTER(vd), ctypes.c_size_t, i32, vd]
    L.ctb_free.argtypes = [vd, vd]
    L.ctb_sync.argtypes = [vd]
    L.ctb_alloc_managed.argtypes = [ctypes.POINTER(vd), ctypes.c_size_t, i32]
    L.ctb_free_managed.argtypes = [vd]
    L.ctb_pool_alloc_managed.argtypes = [ctypes.POINTER(vd), ctypes.c_size_t, i32, i32, vd]
    L.ctb_pool_free_managed.argtypes = [vd]
    L.ctb_pool_trim.argtypes = [i32]
    L.ctb_pool_set_limit.argtypes = [i32, ctypes.c_size_t]
    L.ctb_pool_stats.argtypes = [i32, ctypes.POINTER(PoolInfo)]
    L.ctb_prefetch_managed.argtypes = [vd, ctypes.c_size_t, i32, vd]
    L.ctb_shard_range.argtypes = [i64, i32, i32, ctypes.POINTER(i64), ctypes.POINTER(i64)]
    L.ctb_comm_init_all.argtypes = [i32, ctypes.POINTER(i32)]
    L.ctb_comm_device.argtypes = [i32]
    L.ctb_comm_stream.argtypes = [i32]
    L.ctb_comm_stream.restype = vd
    L.ctb_allreduce.argtypes = [ctypes.POINTER(vd), ctypes.c_size_t, i32, i32]
    L.ctb_full_reduce_sharded.argtypes = [i32, ctypes.POINTER(vp), i64, ctypes.POINTER(vp)]
    L.ctb_div_backward.argtypes = [vp, vp, vp, vp, vp, i32, vd]
    L.ctb_tanh_backward.argtypes = [vp, vp, vp, i32, vd]
    L.ctb_cross_entropy.argtypes = [vp, vp, i32, vp, vd, vd]
    L.ctb_cross_entropy_backward.argtypes = [vp, vp, ctypes.c_double, vp, i32, vd, vd]
    L.ctb_binary.argtypes = [i32, vp, vp, vp, vd]
    L.ctb_unary.argtypes = [i32, vp, ctypes.c_double, vp, vd]
    L.ctb_copy_strided.argtypes = [vp, vp, vd]
    L.ctb_reduce.argtypes = [i32, vp, i32, vp, vd]
    L.ctb_reduce_workspace_bytes.restype = ctypes.c_size_t
    L.ctb_reduce_workspace_bytes.argtypes = [vp, i32]
    L.ctb_reduce_ws.argtypes = [i32, vp, i32, vp, vd, ctypes.c_size_t, vd]
    L.ctb_reduce_dim_noalloc.argtypes = [i32, vp, i32, vp, vd]
    L.ctb_reduce_full_partial.argtypes = [i32, vp, vd, vd]
    L.ctb_finalize_full.argtypes = [i32, vd, i64, vp, vd]
    L.ctb_softmax_lastdim.argtypes = [vp, vp, i32, vp, vd]
    L.ctb_layernorm_lastdim.argtypes = [vp, vp, vp, ctypes.c_double, vp, vd]
    L.ctb_log_softmax_lastdim.argtypes = [vp, vp, vp, vd]
    L.ctb_gather.argtypes = [vp, i32, vp, vp, vd, vd]
    L.ctb_accumulate_grad.argtypes = [vp, vp, vd]
    L.ctb_sgd_step.argtypes = [vp, vp, ctypes.c_double, vd]
    L.ctb_copy_into.argtypes = [vp, vp, vd]
    L.ctb_matmul.argtypes = [vp, vp, vp, vd]
    L.ctb_matmul_tc.argtypes = [vp, vp, vp, vd, vd]
    L.ctb_optimizer_step.argtypes = [i32, vp, vp, vd, vd, ctypes.POINTER(OptimizerHyper), i32, vd]
    L.ctb_channel_moments.argtypes = [vp, vp, vp, vd]
    L.ctb_batchnorm_apply.argtypes = [vp, vp, vp, vp, vp, ctypes.c_double, vp, vd]
    L.ctb_cat.argtypes = [ctypes.POINTER(vp), i32, i32, vp, vd]
    L.ctb_adam_step.argtypes = [vp, vp, vd, vd] + [ctypes.c_double] * 4 + [i32, ctypes.c_double, i32, vd]
    sz, rules_p, params_p = ctypes.c_size_t, ctypes.POINTER(CScoreRules), ctypes.POINTER(CResidualNormParams)
    L.ctb_score_softmax.argtypes = [vp, rules_p, vp, vd]
    L.ctb_score_softmax_workspace_bytes.argtypes = [vp]
    L.ctb_score_softmax_workspace_bytes.restype = sz
    L.ctb_score_softmax_backward.argtypes = [vp, vp, vp, rules_p, vp, vp, vd, sz, vd]
    L.ctb_residual_norm.argtypes = [vp, vp, vp, params_p, vp, vp, vp, vd]
    L.ctb_residual_norm_workspace_bytes.argtypes = [vp, vp]
    L.ctb_residual_norm_workspace_bytes.restype = sz
    L.ctb_residual_norm_backward.argtypes = [vp, vp, vp, vp, params_p, vp, vp, ctypes.POINTER(CResidualNormGrads), vd, sz, vd]
    L.ctb_grad_norm_workspace_bytes.argtypes = [i32]
    L.ctb_grad_norm_workspace_bytes.restype = sz
    L.ctb_grad_norm.argtypes = [ctypes.POINTER(vp), i32, ctypes.c_double, vp, vd, sz, vd]
    L.ctb_clip_grad_norm.argtypes = [ctypes.POINTER(vp), i32, ctypes.c_double, ctypes.c_double, ctypes.POINTER(vp), vp, vd, sz, vd]
    L.ctb_binary_host.argtypes = [i32, vp, vp, vp, i32]
    L.ctb_unary_host.argtypes = [i32, vp, ctypes.c_double, vp, i32]
    L.ctb_reduce_host.argtypes = [i32, vp, i32, vp, i32]
    for name in EXPORTED_SYMBOLS:      # AttributeError here = the library lacks a declared symbol
        getattr(L, name)
    _lib = L
    return L


def check(status: int) -> None:
    if status != 0:
        raise CtbError(status, lib().ctb_last_error().decode())


# ---- torch plumbing (device memory + streams) -------------------------------------------------------
def _torch():
    import torch
    return torch


def _dtype_code(t) -> int:
    torch = _torch()
    try:
        return _TORCH_CODES[t.dtype] if _TORCH_CODES else _torch_codes()[t.dtype]
    except KeyError:
        raise CtbError(3, f"unsupported dtype {t.dtype}")


_TORCH_CODES: dict = {}


def _torch_codes() -> dict:
    """torch dtype -> element-type code (the reference's DType numbering)."""
    torch = _torch()
    _TORCH_CODES.update({torch.float32: F32, torch.int32: I32, torch.float64: F64, torch.uint8: U8, torch.int8: I8,
                         torch.int16: I16, torch.int64: I64, torch.bool: BOOL})
    for name, code in (("uint16", U16), ("uint32", U32), ("uint64", U64)):      # copy-only types; newer torch has them
        if hasattr(torch, name):
            _TORCH_CODES[getattr(torch, name)] = code
    return _TORCH_CODES


def _torch_dtype(code: int):
    return {v: k for k, v in _torch_codes().items()}[code]


@dataclass
class DView:
    """A strided view of a torch storage buffer: the (Storage, offset, shape, strides) quadruple
    of the reference's Tensorimpl.  ``buf`` is a 1-d torch tensor (CUDA for the device entry
    points, CPU — ideally pinned — for the ``*_host`` ones)."""
    buf: "object"
    shape: tuple
    strides: tuple
    offset: int = 0

    @staticmethod
    def of(t) -> "DView":
        """View of a torch tensor as it is (its own strides; offset folded into data_ptr)."""
        if any(s < 0 for s in t.stride()):
            raise CtbError(5, "negative strides are not supported")
        return DView(t, tuple(t.shape), tuple(t.stride()), 0)

    @property
    def dtype(self) -> int:
        return _dtype_code(self.buf)

    @property
    def numel(self) -> int:
        n = 1
        for s in self.shape:
            n *= s
        return n

    def cview(self) -> View:
        """The C descriptor of this view; built once per DView (a view never changes), so a caller that
        keeps its DViews pays the ctypes marshalling once, not per call."""
        cv = self.__dict__.get("_cv")
        if cv is None:
            cv = make_view(self.buf.data_ptr(), self.dtype, self.shape, self.strides, self.offset)
            self.__dict__["_cv"] = cv
        return cv

    def permute(self, dims: Sequence[int]) -> "DView":
        return DView(self.buf, tuple(self.shape[d] for d in dims), tuple(self.strides[d] for d in dims), self.offset)


def _as_dview(x) -> DView:
    return x if isinstance(x, DView) else DView.of(x)


def _stream_ptr(x: DView) -> int:
    torch = _torch()
    if not x.buf.is_cuda:
        raise CtbError(6, "device entry point called with host memory (use the *_host functions)")
    return torch.cuda.current_stream(x.buf.device).cuda_stream


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def _device_guard(x: DView):
    """Makes the tensor's device current for the call; free when it already is."""
    cuda = _torch().cuda
    dev = x.buf.device
    if dev.type == "cuda" and dev.index == cuda.current_device():
        return _NO_GUARD
    return cuda.device(dev)


def broadcast_shape(a: Sequence[int], b: Sequence[int]) -> tuple:
    nd = max(len(a), len(b))
    out = []
    for i in range(nd):
        da = 1 if i < nd - len(a) else a[i - (nd - len(a))]
        db = 1 if i < nd - len(b) else b[i - (nd - len(b))]
        if da != db and da != 1 and db != 1:
            raise CtbError(2, "Shape mismatch in binary op")
        out.append(db if da == 1 else da)
    return tuple(out)


def reduced_shape(shape: Sequence[int], dim: int) -> tuple:
    if dim == DIM_FULL:
        return (1,)
    s = tuple(x for i, x in enumerate(shape) if i != dim)
    return s if s else (1,)


def _new_out(like: DView, shape, dtype_code=None):
    torch = _torch()
    return torch.empty(shape, dtype=_torch_dtype(like.dtype if dtype_code is None else dtype_code),
                       device=like.buf.device)


# ---- operators (device memory) ------------------------------------------------------------------------
def binary(op: int, a, b, out=None):
    """out = a (op) b with broadcasting; a, b: torch CUDA tensors or DViews."""
    a, b = _as_dview(a), _as_dview(b)
    if out is None:
        out = _new_out(a, broadcast_shape(a.shape, b.shape))
    with _device_guard(a):
        check(lib().ctb_binary(op, a.cview(), b.cview(), _as_dview(out).cview(), _stream_ptr(a)))
    return out


def unary(op: int, a, scalar: float = 0.0, out=None):
    a = _as_dview(a)
    if out is None:
        out = _new_out(a, a.shape)
    with _device_guard(a):
        check(lib().ctb_unary(op, a.cview(), float(scalar), _as_dview(out).cview(), _stream_ptr(a)))
    return out


def contiguous(a, out=None):
    """Strided gather into fresh row-major storage (Tensor::contiguous / clone)."""
    a = _as_dview(a)
    if out is None:
        out = _new_out(a, a.shape)
    with _device_guard(a):
        check(lib().ctb_copy_strided(a.cview(), _as_dview(out).cview(), _stream_ptr(a)))
    return out


def reduce(op: int, a, dim: int = DIM_FULL, out=None, workspace=None):
    """sum/mean/max/min/var/argmax along ``dim`` (DIM_FULL = everything)."""
    a = _as_dview(a)
    if out is None:
        out = _new_out(a, reduced_shape(a.shape, dim), I32 if op == ARGMAX else None)
    with _device_guard(a):
        if workspace is None:
            check(lib().ctb_reduce(op, a.cview(), dim, _as_dview(out).cview(), _stream_ptr(a)))
        else:
            check(lib().ctb_reduce_ws(op, a.cview(), dim, _as_dview(out).cview(), workspace.data_ptr(),
                                      workspace.numel() * workspace.element_size(), _stream_ptr(a)))
    return out


NOALLOC_SCRATCH_BYTES = 4 * 1024 * 1024 + 64 * 1024


def reduce_dim_noalloc(op: int, a, dim: int, out):
    """ctb_reduce_dim_noalloc: the dim-wise reduction for callers that must not allocate device
    memory (allocator callbacks, fully budgeted or real-time processes).  Scratch comes from a
    fixed array inside the library; `out` must be provided; shapes that need more than
    NOALLOC_SCRATCH_BYTES of scratch raise CtbError(CTB_ERR_LIMIT).  Calls on one device share
    that array: keep them stream-ordered, and make the first call outside stream capture."""
    a = _as_dview(a)
    with _device_guard(a):
        check(lib().ctb_reduce_dim_noalloc(op, a.cview(), dim, _as_dview(out).cview(), _stream_ptr(a)))
    return out


def reduce_workspace_bytes(a, dim: int) -> int:
    return int(lib().ctb_reduce_workspace_bytes(_as_dview(a).cview(), dim))


def reduce_full_partial(op: int, a, partial=None):
    """fp64 partial of a full reduction over this shard (device tensor with one double)."""
    torch = _torch()
    a = _as_dview(a)
    if partial is None:
        partial = torch.empty(1, dtype=torch.float64, device=a.buf.device)
    with _device_guard(a):
        check(lib().ctb_reduce_full_partial(op, a.cview(), partial.data_ptr(), _stream_ptr(a)))
    return partial


def finalize_full(op: int, partial, total_count: int, out=None, dtype_code: int = F32):
    torch = _torch()
    if out is None:
        out = torch.empty(1, dtype=_torch_dtype(dtype_code), device=partial.device)
    with torch.cuda.device(partial.device):
        check(lib().ctb_finalize_full(op, partial.data_ptr(), int(total_count), _as_dview(out).cview(),
                                      torch.cuda.current_stream(partial.device).cuda_stream))
    return out


def softmax(x, mask=None, causal: bool = False, out=None):
    x = _as_dview(x)
    m = None if mask is None else _as_dview(mask)
    if out is None:
        out = _new_out(x, x.shape)
    with _device_guard(x):
        check(lib().ctb_softmax_lastdim(x.cview(), None if m is None else m.cview(), int(causal),
                                        _as_dview(out).cview(), _stream_ptr(x)))
    return out


def log_softmax(x, mask=None, out=None):
    """(t - max t) - ln(sum exp(t - max t)) over the last dim, t = x (+ mask)."""
    x = _as_dview(x)
    m = None if mask is None else _as_dview(mask)
    if out is None:
        out = _new_out(x, x.shape)
    with _device_guard(x):
        check(lib().ctb_log_softmax_lastdim(x.cview(), None if m is None else m.cview(),
                                            _as_dview(out).cview(), _stream_ptr(x)))
    return out


def gather(x, dim: int, index, out=None):
    """Tensor::gather: out[i] = x[i with coordinate ``dim`` replaced by index[i]]; the index may hold
    any integer dtype (src/core/tensor.cpp:352-356 of the reference refuses the floating ones: so does
    this binding; the library itself also takes them, as the first generation's gather does).
    Raises CtbError(CTB_ERR_DIM) with the reference's text when an index is out of bounds."""
    torch = _torch()
    x, idx = _as_dview(x), _as_dview(index)
    if idx.dtype in (F32, F64):
        raise CtbError(3, "Index tensor must be integer type")
    if out is None:
        out = _new_out(x, idx.shape)
    bad = torch.zeros(1, dtype=torch.int32, device=x.buf.device)
    with _device_guard(x):
        check(lib().ctb_gather(x.cview(), dim, idx.cview(), _as_dview(out).cview(), bad.data_ptr(),
                               _stream_ptr(x)))
    if int(bad.item()):
        raise CtbError(4, "Gather index out of bounds")
    return out


def accumulate_grad(grad, src):
    """grad += src with the broadcast dims of src summed first and non-finite values skipped
    (accumulate_grad of the reference's autograd); ``grad`` is updated in place."""
    g, s = _as_dview(grad), _as_dview(src)
    with _device_guard(g):
        check(lib().ctb_accumulate_grad(g.cview(), s.cview(), _stream_ptr(g)))
    return grad


def div_backward(grad, a, b, want_a=True, want_b=True, out_a=None, out_b=None, accumulate=False):
    """ctb_div_backward: (grad / b, -((grad * a) / ((b * b) + 1e-6))) over the broadcast shape; with
    ``accumulate`` the results are added into out_a / out_b (existing gradient buffers)."""
    g, a, b = _as_dview(grad), _as_dview(a), _as_dview(b)
    shape = broadcast_shape(g.shape, broadcast_shape(a.shape, b.shape))
    if want_a and out_a is None:
        out_a = _new_out(g, shape)
    if want_b and out_b is None:
        out_b = _new_out(g, shape)
    with _device_guard(g):
        check(lib().ctb_div_backward(g.cview(), a.cview(), b.cview(), _as_dview(out_a).cview() if want_a else None,
                                     _as_dview(out_b).cview() if want_b else None, int(accumulate), _stream_ptr(g)))
    return out_a, out_b


def tanh_backward(grad, t, out=None, accumulate=False):
    """ctb_tanh_backward: grad * (1 / (cosh t * cosh t))."""
    g, t = _as_dview(grad), _as_dview(t)
    if out is None:
        out = _new_out(g, broadcast_shape(g.shape, t.shape))
    with _device_guard(g):
        check(lib().ctb_tanh_backward(g.cview(), t.cview(), _as_dview(out).cview(), int(accumulate), _stream_ptr(g)))
    return out


def cross_entropy(logits, labels, mean=True, out=None, bad=None):
    """ctb_cross_entropy: mean | sum over the rows of -(log_softmax(logits)[row, label])."""
    x, lab = _as_dview(logits), _as_dview(labels)
    if out is None:
        out = _new_out(x, (1,))
    with _device_guard(x):
        check(lib().ctb_cross_entropy(x.cview(), lab.cview(), int(mean), _as_dview(out).cview(),
                                      None if bad is None else bad.data_ptr(), _stream_ptr(x)))
    return out


def cross_entropy_backward(logits, labels, grad_scale, out=None, accumulate=False, bad=None):
    """ctb_cross_entropy_backward: (softmax(logits) - onehot(labels)) * grad_scale."""
    x, lab = _as_dview(logits), _as_dview(labels)
    if out is None:
        out = _new_out(x, x.shape)
    with _device_guard(x):
        check(lib().ctb_cross_entropy_backward(x.cview(), lab.cview(), float(grad_scale), _as_dview(out).cview(),
                                               int(accumulate), None if bad is None else bad.data_ptr(), _stream_ptr(x)))
    return out


def matmul(a, b, out=None):
    """matmul_mp: 2-d operands, or 3-d with one leading batch dim."""
    av, bv = _as_dview(a), _as_dview(b)
    if out is None:
        batch = max(av.shape[0] if len(av.shape) == 3 else 1, bv.shape[0] if len(bv.shape) == 3 else 1)
        shape = (av.shape[-2], bv.shape[-1]) if len(av.shape) < 3 and len(bv.shape) < 3 else (batch, av.shape[-2], bv.shape[-1])
        out = _new_out(av, shape)
    with _device_guard(av):
        check(lib().ctb_matmul(av.cview(), bv.cview(), _as_dview(out).cview(), _stream_ptr(av)))
    return out


def matmul_tc(a, b, out=None, status=None):
    """ctb_matmul_tc: the product on the tensor cores (TF32 products, fp32 accumulation).  `status`: an
    int32 CUDA tensor of one element that is non-zero afterwards if the kernel gave up a wait."""
    a, b = _as_dview(a), _as_dview(b)
    if out is None:
        out = _new_out(a, tuple(a.shape[:-1]) + (b.shape[-1],))
    with _device_guard(a):
        check(lib().ctb_matmul_tc(a.cview(), b.cview(), _as_dview(out).cview(),
                                  None if status is None else status.data_ptr(), _stream_ptr(a)))
    return out


def channel_moments(x):
    """Per-channel (dim 1) mean and biased variance of a contiguous x[N, C, ...]: (mean, var)."""
    xv = _as_dview(x)
    c = xv.shape[1] if len(xv.shape) > 1 else 0
    mean, var = _new_out(xv, (c,)), _new_out(xv, (c,))
    with _device_guard(xv):
        check(lib().ctb_channel_moments(xv.cview(), DView.of(mean).cview(), DView.of(var).cview(), _stream_ptr(xv)))
    return mean, var


def batchnorm_apply(x, mean, var, gamma=None, beta=None, eps: float = 1e-5, out=None):
    """((x - mean[c]) * (var[c] + eps)^-0.5) * gamma[c] + beta[c] for a contiguous x[N, C, ...]."""
    xv = _as_dview(x)
    opt = lambda t: None if t is None else _as_dview(t).cview()
    if out is None:
        out = _new_out(xv, xv.shape)
    with _device_guard(xv):
        check(lib().ctb_batchnorm_apply(xv.cview(), _as_dview(mean).cview(), _as_dview(var).cview(),
                                        opt(gamma), opt(beta), float(eps), _as_dview(out).cview(), _stream_ptr(xv)))
    return out


def copy_into(src, dst):
    """dst[...] = src (broadcast allowed); dst may be any strided view."""
    s, d = _as_dview(src), _as_dview(dst)
    with _device_guard(d):
        check(lib().ctb_copy_into(s.cview(), d.cview(), _stream_ptr(d)))
    return dst


def cat(tensors, dim: int = 0, out=None):
    """cat_mp: concatenate along ``dim``."""
    vs = [_as_dview(t) for t in tensors]
    if out is None and vs:
        shape = list(vs[0].shape)
        if 0 <= dim < len(shape):
            shape[dim] = sum(v.shape[dim] if len(v.shape) == len(shape) else 0 for v in vs)
        out = _new_out(vs[0], tuple(shape))
    cviews = [v.cview() for v in vs]
    arr = (ctypes.POINTER(View) * max(1, len(cviews)))(*[ctypes.pointer(c) for c in cviews])
    if not vs:
        check(lib().ctb_cat(arr, 0, dim, None, None))       # raises "cat_mp: empty list"
        return None
    with _device_guard(vs[0]):
        check(lib().ctb_cat(arr, len(cviews), dim, _as_dview(out).cview(), _stream_ptr(vs[0])))
    return out


def sgd_step(param, grad, lr: float):
    """param -= lr * grad in place (SGD::step of the reference)."""
    p, g = _as_dview(param), _as_dview(grad)
    with _device_guard(p):
        check(lib().ctb_sgd_step(p.cview(), g.cview(), float(lr), _stream_ptr(p)))
    return param


def adam_step(param, grad, m, v, lr: float, step: int, beta1: float = 0.9, beta2: float = 0.999,
              eps: float = 1e-8, weight_decay=None):
    """One Adam step in place (AdamW when ``weight_decay`` is given); m, v: fp32 CUDA tensors."""
    p, g = _as_dview(param), _as_dview(grad)
    with _device_guard(p):
        check(lib().ctb_adam_step(p.cview(), g.cview(), m.data_ptr(), v.data_ptr(), float(lr), float(beta1),
                                  float(beta2), float(eps), int(step),
                                  0.0 if weight_decay is None else float(weight_decay),
                                  0 if weight_decay is None else 1, _stream_ptr(p)))
    return param


def optimizer_step(kind: int, param, grad, state1, state2, step: int, lr: float, beta1: float = 0.9,
                   beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.0, alpha: float = 0.99):
    """One in-place step of any of the reference's optimizers (OPT_* codes)."""
    p, g = _as_dview(param), _as_dview(grad)
    h = OptimizerHyper(lr, beta1, beta2, eps, weight_decay, alpha)
    with _device_guard(p):
        check(lib().ctb_optimizer_step(kind, p.cview(), g.cview(), None if state1 is None else state1.data_ptr(),
                                       None if state2 is None else state2.data_ptr(), ctypes.byref(h), int(step),
                                       _stream_ptr(p)))
    return param


def layernorm(x, gamma=None, beta=None, eps: float = 1e-5, out=None):
    x = _as_dview(x)
    g = None if gamma is None else _as_dview(gamma)
    b = None if beta is None else _as_dview(beta)
    if out is None:
        out = _new_out(x, x.shape)
    with _device_guard(x):
        check(lib().ctb_layernorm_lastdim(x.cview(), None if g is None else g.cview(),
                                          None if b is None else b.cview(), float(eps),
                                          _as_dview(out).cview(), _stream_ptr(x)))
    return out


# ---- a transformer block's steps between its matrix products ------------------------------------------------
# These calls take several tensors and return several, often around kernels of a few microseconds, so their
# descriptors are packed in one go and results take their descriptor from an input of the same shape.
_VIEW_PACK = [struct.Struct(f"=qqii{n}q{8 * (MAX_DIMS - n)}x{n}q{8 * (MAX_DIMS - n)}x") for n in range(MAX_DIMS + 1)]


def _raw_view(x):
    """The C descriptor of a tensor or DView (None stays None)."""
    if x is None:
        return None
    if isinstance(x, DView):
        return x.cview()
    shape, n = x.shape, x.dim()
    if n > MAX_DIMS:
        raise CtbError(5, f"ndim {n} not in 0..{MAX_DIMS}")
    return View.from_buffer_copy(_VIEW_PACK[n].pack(x.data_ptr(), 0, _dtype_code(x), n, *shape, *x.stride()))


def _device_of(x) -> int:
    """Index of the CUDA device that holds ``x``."""
    index = (x.buf if isinstance(x, DView) else x).get_device()
    if index < 0:
        raise CtbError(6, "device entry point called with host memory")
    return index


def _on_device(index: int, what: str, tensors) -> None:
    for t in tensors:
        if t is not None and (t.buf if isinstance(t, DView) else t).get_device() != index:
            raise CtbError(5, f"{what}: tensors on different devices")


def _device_scope(index: int):
    cuda = _torch().cuda
    return _NO_GUARD if cuda.current_device() == index else cuda.device(index)


def _stream_of(index: int) -> int:
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # without a Stream object: 1.2 us less per call
    return raw(index) if raw is not None else torch.cuda.current_stream(index).cuda_stream


def _new_like(x, view):
    """A fresh contiguous tensor of x's shape and dtype, and its descriptor."""
    torch = _torch()
    if isinstance(x, DView):
        out = _new_out(x, x.shape)
        return out, _raw_view(out)
    if not x.is_contiguous():
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        return out, _raw_view(out)
    out = torch.empty_like(x)
    v = View.from_buffer_copy(view)
    v.base = out.data_ptr()
    return out, v


def _address(cview):
    """A pointer member of a C struct; the struct's owner keeps the view alive."""
    return None if cview is None else ctypes.addressof(cview)


@functools.lru_cache(maxsize=None)
def _cuda_device(index: int):
    return _torch().device("cuda", index)


def _scratch(nbytes: int, index: int):
    """(tensor, address, size) of one call's scratch, from torch's allocator: ordered on the current stream,
    and a captured graph's own when the call is captured."""
    if not nbytes:
        return None, None, 0
    torch = _torch()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=_cuda_device(index))
    return ws, ws.data_ptr(), nbytes


class ScoreRules:
    """What ``score_softmax`` does to attention scores: scale, tanh ``cap`` (0: none), ``causal``, and per
    sequence ``query_start`` (position of its first query; default: keys - queries), ``key_lengths``,
    ``prefix`` (keys every query may look at) — int32 [batch] —, ``query_docs`` / ``key_docs`` (document
    numbers, int32 [batch, queries] / [batch, keys]) and ``slopes`` (float32 [heads], bias
    -slope * |distance|).  Holds its tensors; their contents may change between calls, their memory may not."""
    _TABLES = ("query_start", "key_lengths", "prefix", "query_docs", "key_docs", "slopes")

    def __init__(self, scale: float = 1.0, cap: float = 0.0, causal: bool = False, query_start=None, key_lengths=None,
                 prefix=None, query_docs=None, key_docs=None, slopes=None):
        self.tables = (query_start, key_lengths, prefix, query_docs, key_docs, slopes)
        self._views = [_raw_view(t) for t in self.tables]
        self.c = CScoreRules(float(scale), float(cap), int(bool(causal)), 0, *(_address(v) for v in self._views))


def score_softmax(scores, rules: ScoreRules, out=None):
    """Attention probabilities of ``scores`` [batch, heads, queries, keys] over the keys that ``rules``
    admit; zeros elsewhere and in the rows of queries that are admitted to nothing."""
    dev = _device_of(scores)
    _on_device(dev, "score_softmax", rules.tables)
    sv = _raw_view(scores)
    with _device_scope(dev):
        if out is None:
            out, ov = _new_like(scores, sv)
        else:
            _on_device(dev, "score_softmax", (out,))
            ov = _raw_view(out)
        check(lib().ctb_score_softmax(sv, rules.c, ov, _stream_of(dev)))
    return out


def score_softmax_backward(grad, probs, rules: ScoreRules, scores=None, want_slopes: bool = False, out=None):
    """(gradient of the scores, gradient of ``rules``' slopes or None) from the gradient of the
    probabilities; ``scores`` (the forward's input) is needed when the rules have a cap."""
    dev = _device_of(probs)
    _on_device(dev, "score_softmax_backward", (grad, scores, out) + rules.tables)
    pv = _raw_view(probs)
    slopes = slopes_view = None
    with _device_scope(dev):
        if out is None:
            out, ov = _new_like(probs, pv)
        else:
            ov = _raw_view(out)
        ws, at, nbytes = None, None, 0
        if want_slopes and pv.ndim == 4:
            slopes = _torch().empty(pv.shape[1], dtype=_torch().float32, device=out.device if not isinstance(out, DView) else out.buf.device)
            slopes_view = _raw_view(slopes)
            ws, at, nbytes = _scratch(lib().ctb_score_softmax_workspace_bytes(pv), dev)
        check(lib().ctb_score_softmax_backward(_raw_view(grad), pv, _raw_view(scores), rules.c, ov, slopes_view, at, nbytes, _stream_of(dev)))
    return out, slopes


class ResidualNorm:
    """The weights and kinds of ``residual_norm``: y = x + scale * gate * N_post(f), h = N_pre(y), each norm
    NORM_NONE, NORM_LAYER or NORM_RMS with an optional float32 weight and bias of the row length.  Holds
    its tensors; their contents may change between calls, their memory may not."""
    _VECTORS = ("post_weight", "post_bias", "pre_weight", "pre_bias")

    def __init__(self, pre: int = NORM_LAYER, pre_weight=None, pre_bias=None, pre_eps: float = 1e-5, post: int = NORM_NONE,
                 post_weight=None, post_bias=None, post_eps: float = 1e-5, scale: float = 1.0):
        self.pre, self.post = pre, post
        self.vectors = (post_weight, post_bias, pre_weight, pre_bias)
        self._views = [_raw_view(t) for t in self.vectors]
        self.c = CResidualNormParams(int(post), int(pre), float(post_eps), float(pre_eps), float(scale),
                                     *(_address(v) for v in self._views))


def residual_norm(x, f, params: ResidualNorm, gate=None):
    """(y, h, stats): the residual stream after a block's output ``f`` is added, its norm for the next block,
    and the rows' statistics [..., 4] for the backward pass.  ``f`` None: y is ``x`` itself; h is None when
    ``params`` has no pre norm."""
    dev = _device_of(x)
    _on_device(dev, "residual_norm", (f, gate) + params.vectors)
    xv = _raw_view(x)
    y, yv, h, hv = x, None, None, None
    with _device_scope(dev):
        if f is not None:
            y, yv = _new_like(x, xv)
        if params.pre != NORM_NONE:
            h, hv = _new_like(x, xv)
        like = x.buf if isinstance(x, DView) else x
        stats = like.new_empty(tuple(x.shape[:-1]) + (4,))
        check(lib().ctb_residual_norm(xv, _raw_view(f), _raw_view(gate), params.c, yv, hv, _raw_view(stats), _stream_of(dev)))
    return y, h, stats


@dataclass
class ResidualNormGrads:
    """Gradients of ``residual_norm``'s inputs; None where there was no such input."""
    x: "object" = None
    f: "object" = None
    gate: "object" = None
    post_weight: "object" = None
    post_bias: "object" = None
    pre_weight: "object" = None
    pre_bias: "object" = None


def residual_norm_backward(f, y, stats, params: ResidualNorm, grad_y=None, grad_h=None, gate=None) -> ResidualNormGrads:
    """The gradients of x, f, the gate, the weights and the biases, from the forward's f, y and stats and
    the gradients of y and h (``grad_y`` None: zero; ``grad_h`` goes with a pre norm)."""
    dev = _device_of(y)
    _on_device(dev, "residual_norm_backward", (f, stats, grad_y, grad_h, gate) + params.vectors)
    yv, gv = _raw_view(y), _raw_view(gate)
    with _device_scope(dev):
        outs = [_new_like(y, yv), (None, None) if f is None else _new_like(y, yv), (None, None) if gate is None else _new_like(gate, gv)]
        outs += [(None, None) if t is None else _new_like(t, v) for t, v in zip(params.vectors, params._views)]
        c = CResidualNormGrads(*(_address(v) for _, v in outs))
        ws, at, nbytes = _scratch(lib().ctb_residual_norm_workspace_bytes(yv, gv), dev)
        check(lib().ctb_residual_norm_backward(_raw_view(f), yv, gv, _raw_view(stats), params.c, _raw_view(grad_y), _raw_view(grad_h), c,
                                               at, nbytes, _stream_of(dev)))
    return ResidualNormGrads(*(t for t, _ in outs))


class TensorList:
    """A list of CUDA tensors (a model's gradients) with the C descriptors built once.  It holds the tensors;
    a tensor that is given other memory afterwards needs a new list."""

    def __init__(self, tensors):
        self.tensors = list(tensors)
        self.device = _device_of(self.tensors[0]) if self.tensors else None
        if self.tensors:
            _on_device(self.device, "TensorList", self.tensors)
        self._views = [_raw_view(t) for t in self.tensors]
        self.has_f64 = any(v.dtype == F64 for v in self._views)
        self.c = (ctypes.POINTER(View) * max(1, len(self._views)))(*[ctypes.pointer(v) for v in self._views])

    def __len__(self):
        return len(self.tensors)


def _grad_norm(grads, max_norm, p, out, norm):
    torch = _torch()
    grads = grads if isinstance(grads, TensorList) else TensorList(grads)
    if out is not None:
        out = out if isinstance(out, TensorList) else TensorList(out)
        if len(out) != len(grads):
            raise CtbError(2, "clip_grad_norm: as many outputs as gradients are needed")
    dev = grads.device
    if dev is None:
        if norm is None:
            raise CtbError(5, "grad_norm: an empty list needs `norm`, which says where the result goes")
        dev = _device_of(norm)
    if out is not None and out.device is not None and out.device != dev:
        raise CtbError(5, "clip_grad_norm: tensors on different devices")
    _on_device(dev, "grad_norm", (norm,))
    with _device_scope(dev):
        if norm is None:
            norm = torch.empty(1, dtype=torch.float64 if grads.has_f64 else torch.float32, device=_cuda_device(dev))
        ws, at, nbytes = _scratch(lib().ctb_grad_norm_workspace_bytes(len(grads)), dev)
        if max_norm is None:
            check(lib().ctb_grad_norm(grads.c, len(grads), float(p), _raw_view(norm), at, nbytes, _stream_of(dev)))
        else:
            check(lib().ctb_clip_grad_norm(grads.c, len(grads), float(max_norm), float(p), None if out is None else out.c,
                                           _raw_view(norm), at, nbytes, _stream_of(dev)))
    return norm


def grad_norm(grads, p: float = 2.0, norm=None):
    """(sum |g|^p)^(1/p) over all tensors of ``grads`` (a list or a TensorList), p = 1, 2 or inf, as a
    one-element CUDA tensor (float64 if any gradient is, else float32)."""
    return _grad_norm(grads, None, p, None, norm)


def clip_grad_norm(grads, max_norm: float, p: float = 2.0, out=None, norm=None):
    """Scales all of ``grads`` by max_norm / norm when max_norm < norm < inf — in place, or into the tensors
    of ``out``, which get the values as they are otherwise — and returns the norm (a CUDA tensor: no
    synchronisation)."""
    return _grad_norm(grads, max_norm, p, out, norm)


# ---- operators (host memory in, host memory out) --------------------------------------------------------
def binary_host(op: int, a, b, out, device: int = 0):
    a, b, o = _as_dview(a), _as_dview(b), _as_dview(out)
    check(lib().ctb_binary_host(op, a.cview(), b.cview(), o.cview(), device))
    return out


def unary_host(op: int, a, out, scalar: float = 0.0, device: int = 0):
    a, o = _as_dview(a), _as_dview(out)
    check(lib().ctb_unary_host(op, a.cview(), float(scalar), o.cview(), device))
    return out


def reduce_host(op: int, a, dim: int, out, device: int = 0):
    a, o = _as_dview(a), _as_dview(out)
    check(lib().ctb_reduce_host(op, a.cview(), dim, o.cview(), device))
    return out
