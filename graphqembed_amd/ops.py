"""Operators on plain device tensors (include/gqe_ops.h): training and scoring queries against a WHOLE entity table.

The reference trains with one sampled negative per query (netquery/model.py:112-127); these are what training against every
entity needs next to it:

    softmax_xent, softmax_xent_loss, softmax_xent_grads   cross entropy of a softmax over all rows of a table, logits never kept
    grad_norm, clip_grad_norm_                            global gradient norm over many tensors, clipping in place
    layer_norm, layer_norm_forward, layer_norm_backward   layer normalisation of query rows
    chain_rows, chain_rows_backward                       query embeddings of a bilinear-diag relation chain

``softmax_xent`` and ``layer_norm`` are differentiable by torch's autograd; the others are the calls a fused training step makes.
All work is enqueued on ``torch.cuda.current_stream()`` of the tensors' device (which need not be the current device); nothing
synchronises and nothing is kept between calls, so every call can be captured into a graph, but for ``softmax_xent`` and
``layer_norm`` where autograd would record them (they raise: capture the calls they are made of).  float32 and bfloat16; sums are
float32 (the norm: float64).  There is no CPU fallback: without libgqe.so or a HIP device the calls raise ``GqeLibraryError``.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from collections import OrderedDict
from itertools import chain, repeat
from operator import attrgetter

import torch

from . import engine as _engine
from .engine import MAX_DIM, GqeError, GqeLibraryError

F32, BF16 = 0, 1
XENT_LOSS, XENT_DQ, XENT_DTABLE = 1, 2, 4
MAX_CHAIN_QUERIES = 65536
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}
_P = C.c_void_p
_DEVICE_OF, _DTYPE_OF = torch.Tensor.get_device, attrgetter("dtype")


class gqe_xent_args(C.Structure):
    _fields_ = [("device", C.c_int32), ("phase", C.c_int32), ("dtype", C.c_int32), ("dim", C.c_int32),
                ("n_queries", C.c_int64), ("n_rows", C.c_int64), ("q", _P), ("q_stride", C.c_int64),
                ("table", _P), ("table_stride", C.c_int64), ("target", _P), ("weight", _P),
                ("scale", C.c_float), ("normalize", C.c_int32), ("loss", _P), ("lse", _P), ("stat", _P),
                ("dq", _P), ("dq_stride", C.c_int64), ("dq_f32", C.c_int32), ("accumulate", C.c_int32),
                ("dtable", _P), ("dtable_stride", C.c_int64), ("workspace", _P), ("workspace_bytes", C.c_int64), ("stream", _P)]


class gqe_tensor(C.Structure):
    _fields_ = [("data", _P), ("numel", C.c_int64), ("dtype", C.c_int32), ("reserved", C.c_int32)]


class gqe_layer_norm_args(C.Structure):
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("dim", C.c_int32), ("accumulate", C.c_int32), ("n_rows", C.c_int64),
                ("x", _P), ("x_stride", C.c_int64), ("weight", _P), ("bias", _P), ("eps", C.c_float), ("reserved", C.c_int32),
                ("y", _P), ("y_stride", C.c_int64), ("mean", _P), ("rstd", _P), ("dy", _P), ("dy_stride", C.c_int64),
                ("dx", _P), ("dx_stride", C.c_int64), ("dweight", _P), ("dbias", _P),
                ("workspace", _P), ("workspace_bytes", C.c_int64), ("stream", _P)]


class gqe_chain_args(C.Structure):
    _fields_ = [("device", C.c_int32), ("dim", C.c_int32), ("n", C.c_int64), ("rows", _P), ("table", _P), ("table_stride", C.c_int64),
                ("n_rows", C.c_int64), ("n_rels", C.c_int32), ("reserved", C.c_int32), ("rel", _P * 3), ("q", _P), ("q_stride", C.c_int64),
                ("dq", _P), ("dq_stride", C.c_int64), ("dtable", _P), ("dtable_stride", C.c_int64), ("drel", _P * 3),
                ("workspace", _P), ("workspace_bytes", C.c_int64), ("stream", _P)]


# The same as bytes (a call of 20 us cannot spend 5 of them on setting fields one by one); tests/test_ops_cpu.py holds the two together.
_XENT = struct.Struct("@4i2qPqPqPPfiPPPPqiiPqPqP")
_NORM = struct.Struct("@4iqPqPPfiPqPPPqPqPPPqP")
_TENSOR = struct.Struct("@Pqii")

# every symbol include/gqe_ops.h declares: name -> (restype, argtypes)
OPS_SYMBOLS = OrderedDict([
    ("gqe_ops_last_error", (C.c_char_p, [])),
    ("gqe_softmax_xent_workspace", (C.c_int64, [_P])),
    ("gqe_softmax_xent", (C.c_int, [_P])),
    ("gqe_clip_grads_workspace", (C.c_int64, [_P, C.c_int32])),
    ("gqe_clip_grads", (C.c_int, [C.c_int32, _P, C.c_int32, C.c_float, _P, _P, C.c_int64, _P])),
    ("gqe_layer_norm_workspace", (C.c_int64, [_P])),
    ("gqe_layer_norm_forward", (C.c_int, [_P])),
    ("gqe_layer_norm_backward", (C.c_int, [_P])),
    ("gqe_chain_rows_forward", (C.c_int, [_P])),
    ("gqe_chain_rows_backward", (C.c_int, [_P])),
])

_lib = None


def library():
    """libgqe.so with the operators' entry points typed (no GPU needed)."""
    global _lib
    if _lib is None:
        lib = _engine.load_library()
        for name, (res, args) in OPS_SYMBOLS.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def _check(rc):
    if rc < 0:
        raise GqeError(rc, (library().gqe_ops_last_error() or b"").decode())
    return rc


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _on_gpu(what, *tensors):
    """Index of the HIP device that all tensors are on."""
    index = None
    for t in tensors:
        try:
            i = t.get_device() if t.is_cuda else -1
        except AttributeError:
            raise ValueError("%s: expected a tensor, got %s" % (what, type(t).__name__)) from None
        if i < 0:
            raise GqeLibraryError("%s: the operators run on an MI355X only (got a tensor on %s; there is no CPU fallback)" % (what, t.device))
        if index is None:
            index = i
        elif i != index:
            raise ValueError("%s: tensors on %s and %s" % (what, tensors[0].device, t.device))
    return index


def _recorded(what, forms, *tensors):
    """Whether autograd records a call on these tensors.  Refused in a capture: with an eager graph of the same leaves alive, torch's
    backward makes that graph's stream wait for the captured one, which ends the capture and the process."""
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("%s: autograd's form cannot be captured; capture %s" % (what, forms))
    return True


def _dtype(what, t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s: float32 or bfloat16, not %s" % (what, t.dtype))
    return code


def _rows(t):
    """[n, d] with unit stride along a row and rows that do not overlap (a view of a table keeps its row stride), and that stride."""
    n, d = t.shape
    row, unit = t.stride()
    if (d > 1 and unit != 1) or (n > 1 and row < d):
        t, row = t.contiguous(), d
    return t, max(row, d) if n <= 1 else row


# -- softmax cross entropy over a table ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _xent_space(phase, dtype, dim, n, rows, own_stat):
    """Workspace bytes of a call: its sizes alone say."""
    a = gqe_xent_args(phase=phase, dtype=dtype, dim=dim, n_queries=n, n_rows=rows, stat=1 if own_stat else None)
    return _check(library().gqe_softmax_xent_workspace(C.byref(a)))


def _xent(what, phase, q, table, target, scale, normalize, weight=None, loss=None, lse=None, stat=None, dq=None, dtable=None, accumulate=False):
    """One call of gqe_softmax_xent on checked tensors; returns (q, table, target) as they were handed over."""
    index = _on_gpu(what, q, table, target)
    if q.dim() != 2 or table.dim() != 2 or q.shape[1] != table.shape[1]:
        raise ValueError("%s: q [n, d] and table [rows, d], got %s and %s" % (what, tuple(q.shape), tuple(table.shape)))
    if q.dtype != table.dtype:
        raise ValueError("%s: q is %s, the table %s" % (what, q.dtype, table.dtype))
    n, d = q.shape
    rows = table.shape[0]
    if target.dim() != 1 or target.shape[0] != n or target.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s: target is int32 or int64 [%d], got %s %s" % (what, n, target.dtype, tuple(target.shape)))
    if not 1 <= d <= MAX_DIM:
        raise ValueError("%s: d = %d is not in 1 .. %d" % (what, d, MAX_DIM))
    if rows < 1:
        raise ValueError("%s: an empty table" % what)
    if target.dtype == torch.int64:       # rows beyond int32 (there are none) stay out of range
        target = target.clamp(-1, 0x7fffffff).to(torch.int32)
    dtype = _dtype(what, q)
    q, q_stride = _rows(q)
    table, t_stride = _rows(table)
    target = target.contiguous()
    if weight is not None:
        _on_gpu(what, q, weight)
        if weight.dtype != torch.float32 or weight.dim() != 1 or weight.shape[0] != n:
            raise ValueError("%s: weight is float32 [%d], got %s %s" % (what, n, weight.dtype, tuple(weight.shape)))
        weight = weight.contiguous()
    need = _xent_space(phase, dtype, d, n, rows, stat is not None)
    space = q.new_empty(need, dtype=torch.uint8)
    _check(library().gqe_softmax_xent(_XENT.pack(
        index, phase, dtype, d, n, rows, q.data_ptr(), q_stride, table.data_ptr(), t_stride, target.data_ptr(),
        0 if weight is None else weight.data_ptr(), scale, 1 if normalize else 0, 0 if loss is None else loss.data_ptr(),
        0 if lse is None else lse.data_ptr(), 0 if stat is None else stat.data_ptr(), 0 if dq is None else dq.data_ptr(), d,
        1 if dq is not None and dq.dtype == torch.float32 else 0, 1 if accumulate else 0, 0 if dtable is None else dtable.data_ptr(),
        0 if dtable is None else max(dtable.stride(0), d) if rows <= 1 else dtable.stride(0), space.data_ptr(), need, _stream(index))))
    return q, table, target


# (tensors come from Tensor.new_empty with sizes as arguments: 1.2 us of host time each, against 1.8 us of torch.empty(shape, device=))
def _floats(like, *shape):
    return like.new_empty(*shape, dtype=torch.float32)


def softmax_xent_loss(q, table, target, scale=1.0, normalize=False):
    """(loss[n], lse[n]) in float32: lse = log sum_v exp(scale * q . t_v) over all rows of ``table``, loss = lse - scale * q . t_target.

    ``normalize``: rows count as t / |t| (what the encoder does with the rows it reads; a zero row stays zero), so that unit queries
    score by cosine.  target < 0 ignores a query (loss 0; its lse is still given); target >= rows gives loss NaN."""
    _on_gpu("softmax_xent_loss", q)
    loss, lse = _floats(q, q.shape[0]), _floats(q, q.shape[0])
    _xent("softmax_xent_loss", XENT_LOSS, q, table, target, scale, normalize, loss=loss, lse=lse)
    return loss, lse


def softmax_xent_grads(q, table, target, weight=None, scale=1.0, normalize=False, grad_table=None):
    """(loss[n], lse[n], dq, dtable): ``softmax_xent_loss`` and the gradients of sum_b weight_b loss_b (None: all ones) in one call.

    dq and dtable have the type of q.  ``grad_table`` (float32, the table's shape): dtable is ADDED there instead, and returned."""
    what = "softmax_xent_grads"
    _on_gpu(what, q, table)
    loss, lse = _floats(q, q.shape[0]), _floats(q, q.shape[0])
    dq = q.new_empty(*q.shape)
    accumulate = grad_table is not None
    if not accumulate:
        grad_table = table.new_empty(*table.shape)
    else:
        _on_gpu(what, q, grad_table)
        d = table.shape[-1]
        if grad_table.dtype != torch.float32 or q.dtype != torch.float32 or grad_table.shape != table.shape or \
                (d > 1 and grad_table.stride(1) != 1) or (table.shape[0] > 1 and grad_table.stride(0) < d):
            raise ValueError("%s: grad_table is float32 %s with unit stride along a row (and q float32)" % (what, tuple(table.shape)))
    _xent(what, XENT_LOSS | XENT_DQ | XENT_DTABLE, q, table, target, scale, normalize, weight=weight, loss=loss, lse=lse, dq=dq, dtable=grad_table,
          accumulate=accumulate)
    return loss, lse, dq, grad_table


class _SoftmaxXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, table, target, scale, normalize):
        loss, stat = _floats(q, q.shape[0]), _floats(q, q.shape[0], 2)
        dq, phase = None, XENT_LOSS
        if ctx.needs_input_grad[0]:
            dq, phase = _floats(q, *q.shape), XENT_LOSS | XENT_DQ      # of each query's own loss, scaled in backward
        q, table, target = _xent("softmax_xent", phase, q, table, target, scale, normalize, loss=loss, stat=stat, dq=dq)
        ctx.save_for_backward(q, table, target, stat, dq)
        ctx.scale, ctx.normalize = scale, normalize
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, table, target, stat, dq = ctx.saved_tensors
        grad = grad.to(torch.float32).contiguous()
        gq = gt = None
        if ctx.needs_input_grad[0]:
            gq = (dq * grad.unsqueeze(1)).to(q.dtype)
        if ctx.needs_input_grad[1]:
            gt = table.new_empty(*table.shape)
            _xent("softmax_xent", XENT_DTABLE, q, table, target, ctx.scale, ctx.normalize, weight=grad, stat=stat, dtable=gt)
        return gq, gt, None, None, None


def softmax_xent(q, table, target, scale=1.0, normalize=False, reduction="mean"):
    """Differentiable ``softmax_xent_loss``: the loss of q [n, d] against every row of ``table``, gradients for both.

    reduction: "none" (loss[n]), "sum", "mean" (over the queries whose target is not ignored; 0 if there is none)."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError("softmax_xent: reduction %r" % (reduction,))
    scale, normalize = float(scale), bool(normalize)
    _on_gpu("softmax_xent", q, table, target)
    if _recorded("softmax_xent", "softmax_xent_grads", q, table):
        loss = _SoftmaxXent.apply(q, table, target, scale, normalize)
    else:
        loss = softmax_xent_loss(q, table, target, scale, normalize)[0]
    if reduction == "none":
        return loss
    loss_sum = loss.sum()
    return loss_sum if reduction == "sum" else loss_sum / (target >= 0).sum().clamp(min=1)


# -- gradient norm and clipping ------------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _tensors(n):
    return struct.Struct("@" + n * _TENSOR.format[1:])


def _clip(what, grads, max_norm):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ValueError("%s: no tensors" % what)
    try:
        devices = set(map(_DEVICE_OF, grads))
    except TypeError:
        devices = ()
    index = _on_gpu(what, *grads) if len(devices) != 1 or -1 in devices else devices.pop()      # (names what is wrong)
    for g, contiguous in zip(grads, map(torch.Tensor.is_contiguous, grads)):
        if not contiguous:
            raise ValueError("%s: tensors are contiguous (got shape %s, strides %s)" % (what, tuple(g.shape), g.stride()))
    codes = [_DTYPES.get(t) for t in map(_DTYPE_OF, grads)]
    if None in codes:
        _dtype(what, grads[codes.index(None)])
    n, lib = len(grads), library()
    arr = _tensors(n).pack(*chain.from_iterable(zip(map(torch.Tensor.data_ptr, grads), map(torch.Tensor.numel, grads), codes, repeat(0))))
    need = _check(lib.gqe_clip_grads_workspace(arr, n))
    space, norm = grads[0].new_empty(need, dtype=torch.uint8), grads[0].new_empty((), dtype=torch.float32)
    _check(lib.gqe_clip_grads(index, arr, n, max_norm, norm.data_ptr(), space.data_ptr(), need, _stream(index)))
    return norm


def grad_norm(grads):
    """sqrt(sum over all tensors of g^2) as a 0-dim float32 device tensor (no synchronisation)."""
    return _clip("grad_norm", grads, -1.0)


def clip_grad_norm_(grads, max_norm):
    """Multiply all tensors in place by min(1, max_norm / (norm + 1e-6)); returns the norm before (0-dim float32 device tensor, no
    synchronisation) — torch.nn.utils.clip_grad_norm_ on the gradients themselves.  Nothing is written where the factor is 1."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("clip_grad_norm_: max_norm %r" % (max_norm,))
    return _clip("clip_grad_norm_", grads, max_norm)


# -- layer normalisation -------------------------------------------------------------------------------------------------------

def _ln_vector(what, name, v, index, d):
    if v is None:
        return 0
    if _on_gpu(what, v) != index:
        raise ValueError("%s: %s is on another device" % (what, name))
    if v.dtype != torch.float32 or v.dim() != 1 or v.shape[0] != d or not (v.is_contiguous() or d == 1):
        raise ValueError("%s: %s is float32 [%d], contiguous, got %s %s" % (what, name, d, v.dtype, tuple(v.shape)))
    return v.data_ptr()


@functools.lru_cache(maxsize=256)
def _ln_space(dtype, dim, n):
    """Workspace bytes of a backward call: its sizes alone say."""
    a = gqe_layer_norm_args(dtype=dtype, dim=dim, n_rows=n)
    return _check(library().gqe_layer_norm_workspace(C.byref(a)))


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """(y, mean[n], rstd[n]) of the rows of x [n, d]; weight and bias float32 [d] or None; y has the type of x."""
    what = "layer_norm"
    index = _on_gpu(what, x)
    if x.dim() != 2:
        raise ValueError("%s: rows [n, d], got %s" % (what, tuple(x.shape)))
    n, d = x.shape
    dtype = _dtype(what, x)
    w, b = _ln_vector(what, "weight", weight, index, d), _ln_vector(what, "bias", bias, index, d)
    x, stride = _rows(x)
    y, mean, rstd = x.new_empty(n, d), _floats(x, n), _floats(x, n)
    _check(library().gqe_layer_norm_forward(_NORM.pack(index, dtype, d, 0, n, x.data_ptr(), stride, w, b, eps, 0, y.data_ptr(), d, mean.data_ptr(),
                                                       rstd.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, _stream(index))))
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, grad_weight=None, grad_bias=None):
    """(dx, dweight, dbias) from the forward call's mean and rstd; dx has the type of x, dweight and dbias are float32.

    ``grad_weight`` and ``grad_bias`` (float32 [d], both or neither): the two are ADDED there instead, and returned."""
    what = "layer_norm_backward"
    index = _on_gpu(what, x, dy, mean, rstd)
    if x.dim() != 2 or dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("%s: rows [n, d] of one type, got dy %s %s, x %s %s" % (what, dy.dtype, tuple(dy.shape), x.dtype, tuple(x.shape)))
    n, d = x.shape
    for v in (mean, rstd):
        if v.dtype != torch.float32 or v.dim() != 1 or v.shape[0] != n:
            raise ValueError("%s: mean and rstd are float32 [%d]" % (what, n))
    dtype = _dtype(what, x)
    w = _ln_vector(what, "weight", weight, index, d)
    x, x_stride = _rows(x)
    dy, dy_stride = _rows(dy)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = x.new_empty(n, d)
    accumulate = grad_weight is not None
    if accumulate != (grad_bias is not None):
        raise ValueError("%s: grad_weight and grad_bias come together" % what)
    if accumulate:
        _ln_vector(what, "grad_weight", grad_weight, index, d)
        _ln_vector(what, "grad_bias", grad_bias, index, d)
    dweight, dbias = (grad_weight, grad_bias) if accumulate else (_floats(x, d), _floats(x, d))
    need = _ln_space(dtype, d, n)
    space = x.new_empty(need, dtype=torch.uint8) if need else None
    _check(library().gqe_layer_norm_backward(_NORM.pack(index, dtype, d, 1 if accumulate else 0, n, x.data_ptr(), x_stride, w, 0, 0.0, 0, 0, 0, mean.data_ptr(),
                                                        rstd.data_ptr(), dy.data_ptr(), dy_stride, dx.data_ptr(), d, dweight.data_ptr(),
                                                        dbias.data_ptr(), space.data_ptr() if need else 0, need, _stream(index))))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Differentiable ``layer_norm_forward`` along the last dimension of x."""
    if x.dim() < 1:
        raise ValueError("layer_norm: a 0-dim tensor")
    rows, eps = x.reshape(-1, x.shape[-1]), float(eps)
    if _recorded("layer_norm", "layer_norm_forward and layer_norm_backward", x, weight, bias):
        return _LayerNorm.apply(rows, weight, bias, eps).view(x.shape)
    return layer_norm_forward(rows, weight, bias, eps)[0].view(x.shape)


# -- query side of a relation chain ----------------------------------------------------------------------------------------------

def _chain_args(what, table, rows, rels):
    index = _on_gpu(what, table, rows, *rels)
    d = table.shape[-1]
    if table.dim() != 2 or table.dtype != torch.float32 or not 1 <= d <= MAX_DIM or (d > 1 and table.stride(1) != 1) or table.shape[0] < 1 or \
            (table.shape[0] > 1 and table.stride(0) < d):
        raise ValueError("%s: the table is float32 [rows, d <= %d] with unit stride along a row" % (what, MAX_DIM))
    if rows.dim() != 1 or rows.dtype != torch.int32 or not rows.is_contiguous():
        raise ValueError("%s: rows is int32 [n], contiguous" % what)
    if len(rels) > 3:
        raise ValueError("%s: %d relations" % (what, len(rels)))
    a = gqe_chain_args()
    a.device, a.dim, a.n, a.rows = index, d, rows.shape[0], rows.data_ptr()
    a.table, a.table_stride, a.n_rows, a.n_rels, a.stream = table.data_ptr(), max(table.stride(0), d), table.shape[0], len(rels), _stream(index)
    for j, r in enumerate(rels):
        if r.dtype != torch.float32 or r.dim() != 1 or r.shape[0] != d or not r.is_contiguous():
            raise ValueError("%s: relations are float32 [%d], contiguous" % (what, d))
        a.rel[j] = r.data_ptr()
    return a


def chain_rows(table, rows, rels):
    """q [n, d]: the anchors' table rows over their lengths, times the relation vectors (at most 3) element by element."""
    a = _chain_args("chain_rows", table, rows, rels)
    q = torch.empty((a.n, a.dim), dtype=torch.float32, device=table.device)
    a.q, a.q_stride = q.data_ptr(), a.dim
    _check(library().gqe_chain_rows_forward(C.byref(a)))
    return q


def chain_rows_backward(dq, table, rows, rels, grad_table, grad_rels):
    """ADD the gradients of ``chain_rows`` into grad_table (the table's shape) and grad_rels (one for each relation)."""
    what = "chain_rows_backward"
    a = _chain_args(what, table, rows, rels)
    _on_gpu(what, table, dq, grad_table, *grad_rels)
    if dq.dtype != torch.float32 or dq.dim() != 2 or tuple(dq.shape) != (a.n, a.dim) or grad_table.dtype != torch.float32 or grad_table.shape != table.shape or \
            (a.dim > 1 and grad_table.stride(1) != 1) or (a.n_rows > 1 and grad_table.stride(0) < a.dim) or len(grad_rels) != len(rels):
        raise ValueError("%s: dq is float32 [%d, %d], the gradients have their tensors' shapes" % (what, a.n, a.dim))
    for j, r in enumerate(grad_rels):
        if r.dtype != torch.float32 or r.dim() != 1 or r.shape[0] != a.dim or not r.is_contiguous():
            raise ValueError("%s: gradients of relations are float32 [%d], contiguous" % (what, a.dim))
        a.drel[j] = r.data_ptr()
    dq, stride = _rows(dq)
    need = 8 * a.n * a.dim
    space = torch.empty(max(need, 4), dtype=torch.uint8, device=table.device)
    a.dq, a.dq_stride, a.dtable, a.dtable_stride = dq.data_ptr(), stride, grad_table.data_ptr(), max(grad_table.stride(0), a.dim)
    a.workspace, a.workspace_bytes = space.data_ptr(), need
    _check(library().gqe_chain_rows_backward(C.byref(a)))
