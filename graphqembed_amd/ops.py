"""Operators on plain device tensors (include/gqe_ops.h): training and scoring queries against a WHOLE entity table.

The reference trains with one sampled negative per query (netquery/model.py:112-127); these are what training against every
entity needs next to it:

    softmax_xent, softmax_xent_loss, softmax_xent_grads   cross entropy of a softmax over all rows of a table, logits never kept
    grad_norm, clip_grad_norm_                            global gradient norm over many tensors, clipping in place
    layer_norm, layer_norm_forward, layer_norm_backward   layer normalisation of query rows

``softmax_xent`` and ``layer_norm`` are differentiable by torch's autograd; the others are the calls a fused training step makes.
All work is enqueued on ``torch.cuda.current_stream()`` of the tensors' device (which need not be the current device); nothing
synchronises and nothing is kept between calls, so every call can be captured into a graph.  float32 and bfloat16; sums are
float32 (the norm: float64).  There is no CPU fallback: without libgqe.so or a HIP device the calls raise ``GqeLibraryError``.
"""
from __future__ import annotations

import ctypes as C
from collections import OrderedDict

import torch

from . import engine as _engine
from .engine import MAX_DIM, GqeError, GqeLibraryError

F32, BF16 = 0, 1
XENT_LOSS, XENT_DQ, XENT_DTABLE = 1, 2, 4
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}
_P = C.c_void_p


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


# every symbol include/gqe_ops.h declares: name -> (restype, argtypes)
OPS_SYMBOLS = OrderedDict([
    ("gqe_ops_last_error", (C.c_char_p, [])),
    ("gqe_softmax_xent_workspace", (C.c_int64, [C.POINTER(gqe_xent_args)])),
    ("gqe_softmax_xent", (C.c_int, [C.POINTER(gqe_xent_args)])),
    ("gqe_clip_grads_workspace", (C.c_int64, [C.POINTER(gqe_tensor), C.c_int32])),
    ("gqe_clip_grads", (C.c_int, [C.c_int32, C.POINTER(gqe_tensor), C.c_int32, C.c_float, _P, _P, C.c_int64, _P])),
    ("gqe_layer_norm_workspace", (C.c_int64, [C.POINTER(gqe_layer_norm_args)])),
    ("gqe_layer_norm_forward", (C.c_int, [C.POINTER(gqe_layer_norm_args)])),
    ("gqe_layer_norm_backward", (C.c_int, [C.POINTER(gqe_layer_norm_args)])),
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


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _on_gpu(what, *tensors):
    """All tensors on one HIP device; its index."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s: expected a tensor, got %s" % (what, type(t).__name__))
        if not t.is_cuda:
            raise GqeLibraryError("%s: the operators run on an MI355X only (got a tensor on %s; there is no CPU fallback)" % (what, t.device))
        if t.device != tensors[0].device:
            raise ValueError("%s: tensors on %s and %s" % (what, tensors[0].device, t.device))
    return tensors[0].device


def _dtype(what, t):
    if t.dtype not in _DTYPES:
        raise ValueError("%s: float32 or bfloat16, not %s" % (what, t.dtype))
    return _DTYPES[t.dtype]


def _rows(t):
    """[n, d] with unit stride along a row and rows that do not overlap (a view of a table keeps its row stride)."""
    if t.shape[1] > 1 and t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))


# -- softmax cross entropy over a table ----------------------------------------------------------------------------------------

def _xent_args(what, q, table, target, scale, normalize):
    dev = _on_gpu(what, q, table, target)
    if q.dim() != 2 or table.dim() != 2 or q.shape[1] != table.shape[1]:
        raise ValueError("%s: q [n, d] and table [rows, d], got %s and %s" % (what, tuple(q.shape), tuple(table.shape)))
    if q.dtype != table.dtype:
        raise ValueError("%s: q is %s, the table %s" % (what, q.dtype, table.dtype))
    if target.dim() != 1 or target.shape[0] != q.shape[0] or target.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s: target is int32 or int64 [%d], got %s %s" % (what, q.shape[0], target.dtype, tuple(target.shape)))
    if not 1 <= q.shape[1] <= MAX_DIM:
        raise ValueError("%s: d = %d is not in 1 .. %d" % (what, q.shape[1], MAX_DIM))
    if table.shape[0] < 1:
        raise ValueError("%s: an empty table" % what)
    if target.dtype == torch.int64:       # rows beyond int32 (there are none) stay out of range
        target = target.clamp(-1, 0x7fffffff).to(torch.int32)
    q, table, target = _rows(q), _rows(table), target.contiguous()
    a = gqe_xent_args()
    a.device, a.dtype, a.dim = dev.index, _dtype(what, q), q.shape[1]
    a.n_queries, a.n_rows = q.shape[0], table.shape[0]
    a.q, a.q_stride, a.table, a.table_stride = q.data_ptr(), _row_stride(q), table.data_ptr(), _row_stride(table)
    a.target, a.scale, a.normalize = target.data_ptr(), float(scale), 1 if normalize else 0
    return a, (q, table, target)


def _xent_run(a, device):
    lib = library()
    need = _check(lib.gqe_softmax_xent_workspace(C.byref(a)))
    space = torch.empty(need, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes, a.stream = space.data_ptr(), need, _stream(device)
    _check(lib.gqe_softmax_xent(C.byref(a)))


def _weights(what, weight, q):
    if weight is None:
        return None
    _on_gpu(what, q, weight)
    if weight.dtype != torch.float32 or weight.shape != (q.shape[0],):
        raise ValueError("%s: weight is float32 [%d], got %s %s" % (what, q.shape[0], weight.dtype, tuple(weight.shape)))
    return weight.contiguous()


def softmax_xent_loss(q, table, target, scale=1.0, normalize=False):
    """(loss[n], lse[n]) in float32: lse = log sum_v exp(scale * q . t_v) over all rows of ``table``, loss = lse - scale * q . t_target.

    ``normalize``: rows count as t / |t| (what the encoder does with the rows it reads; a zero row stays zero), so that unit queries
    score by cosine.  target < 0 ignores a query (loss 0; its lse is still given); target >= rows gives loss NaN."""
    a, keep = _xent_args("softmax_xent_loss", q, table, target, scale, normalize)
    loss = torch.empty(q.shape[0], dtype=torch.float32, device=q.device)
    lse = torch.empty_like(loss)
    a.phase, a.loss, a.lse = XENT_LOSS, loss.data_ptr(), lse.data_ptr()
    _xent_run(a, q.device)
    return loss, lse


def softmax_xent_grads(q, table, target, weight=None, scale=1.0, normalize=False, grad_table=None):
    """(loss[n], lse[n], dq, dtable): ``softmax_xent_loss`` and the gradients of sum_b weight_b loss_b (None: all ones) in one call.

    dq and dtable have the type of q.  ``grad_table`` (float32, the table's shape): dtable is ADDED there instead, and returned."""
    a, keep = _xent_args("softmax_xent_grads", q, table, target, scale, normalize)
    n, d = q.shape
    loss = torch.empty(n, dtype=torch.float32, device=q.device)
    lse = torch.empty_like(loss)
    dq = torch.empty((n, d), dtype=q.dtype, device=q.device)
    w = _weights("softmax_xent_grads", weight, q)
    if grad_table is None:
        grad_table = torch.empty(tuple(table.shape), dtype=table.dtype, device=table.device)
    else:
        _on_gpu("softmax_xent_grads", q, grad_table)
        if grad_table.dtype != torch.float32 or q.dtype != torch.float32 or grad_table.shape != table.shape or \
                (d > 1 and grad_table.stride(1) != 1) or (table.shape[0] > 1 and grad_table.stride(0) < d):
            raise ValueError("softmax_xent_grads: grad_table is float32 %s with unit stride along a row (and q float32)" % (tuple(table.shape),))
        a.accumulate = 1
    a.phase, a.loss, a.lse = XENT_LOSS | XENT_DQ | XENT_DTABLE, loss.data_ptr(), lse.data_ptr()
    a.weight = None if w is None else w.data_ptr()
    a.dq, a.dq_stride, a.dtable, a.dtable_stride = dq.data_ptr(), d, grad_table.data_ptr(), _row_stride(grad_table)
    _xent_run(a, q.device)
    return loss, lse, dq, grad_table


class _SoftmaxXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, table, target, scale, normalize):
        a, (qc, tc, tgt) = _xent_args("softmax_xent", q, table, target, scale, normalize)
        n, d = q.shape
        loss = torch.empty(n, dtype=torch.float32, device=q.device)
        stat = torch.empty((n, 2), dtype=torch.float32, device=q.device)
        dq = None
        a.phase, a.loss, a.stat = XENT_LOSS, loss.data_ptr(), stat.data_ptr()
        if ctx.needs_input_grad[0]:
            dq = torch.empty((n, d), dtype=torch.float32, device=q.device)      # of each query's own loss, scaled in backward
            a.phase |= XENT_DQ
            a.dq, a.dq_stride, a.dq_f32 = dq.data_ptr(), d, 1
        _xent_run(a, q.device)
        ctx.save_for_backward(qc, tc, tgt, stat, dq)
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
            a, keep = _xent_args("softmax_xent", q, table, target, ctx.scale, ctx.normalize)
            gt = torch.empty(tuple(table.shape), dtype=table.dtype, device=table.device)
            a.phase, a.stat, a.weight = XENT_DTABLE, stat.data_ptr(), grad.data_ptr()
            a.dtable, a.dtable_stride = gt.data_ptr(), _row_stride(gt)
            _xent_run(a, q.device)
        return gq, gt, None, None, None


def softmax_xent(q, table, target, scale=1.0, normalize=False, reduction="mean"):
    """Differentiable ``softmax_xent_loss``: the loss of q [n, d] against every row of ``table``, gradients for both.

    reduction: "none" (loss[n]), "sum", "mean" (over the queries whose target is not ignored; 0 if there is none)."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError("softmax_xent: reduction %r" % (reduction,))
    loss = _SoftmaxXent.apply(q, table, target, float(scale), bool(normalize))
    if reduction == "none":
        return loss
    loss_sum = loss.sum()
    return loss_sum if reduction == "sum" else loss_sum / (target >= 0).sum().clamp(min=1)


# -- gradient norm and clipping ------------------------------------------------------------------------------------------------

def _clip(what, grads, max_norm):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ValueError("%s: no tensors" % what)
    dev = _on_gpu(what, *grads)
    arr = (gqe_tensor * len(grads))()
    for a, g in zip(arr, grads):
        if not g.is_contiguous():
            raise ValueError("%s: tensors are contiguous (got shape %s, strides %s)" % (what, tuple(g.shape), g.stride()))
        a.data, a.numel, a.dtype = g.data_ptr(), g.numel(), _dtype(what, g)
    lib = library()
    need = _check(lib.gqe_clip_grads_workspace(arr, len(grads)))
    space = torch.empty(need, dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    _check(lib.gqe_clip_grads(dev.index, arr, len(grads), max_norm, norm.data_ptr(), space.data_ptr(), need, _stream(dev)))
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

def _ln_vector(what, name, v, x):
    if v is None:
        return None
    _on_gpu(what, x, v)
    if v.dtype != torch.float32 or v.shape != (x.shape[-1],):
        raise ValueError("%s: %s is float32 [%d], got %s %s" % (what, name, x.shape[-1], v.dtype, tuple(v.shape)))
    return v.contiguous()


def _ln_args(what, x):
    if x.dim() != 2:
        raise ValueError("%s: rows [n, d], got %s" % (what, tuple(x.shape)))
    dev = _on_gpu(what, x)
    a = gqe_layer_norm_args()
    a.device, a.dtype, a.dim, a.n_rows = dev.index, _dtype(what, x), x.shape[1], x.shape[0]
    x = _rows(x)
    a.x, a.x_stride, a.stream = x.data_ptr(), _row_stride(x), _stream(dev)
    return a, x


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """(y, mean[n], rstd[n]) of the rows of x [n, d]; weight and bias float32 [d] or None; y has the type of x."""
    a, x = _ln_args("layer_norm", x)
    weight, bias = _ln_vector("layer_norm", "weight", weight, x), _ln_vector("layer_norm", "bias", bias, x)
    n, d = x.shape
    y = torch.empty((n, d), dtype=x.dtype, device=x.device)
    mean = torch.empty(n, dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    a.weight = None if weight is None else weight.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()
    a.eps, a.y, a.y_stride, a.mean, a.rstd = float(eps), y.data_ptr(), d, mean.data_ptr(), rstd.data_ptr()
    _check(library().gqe_layer_norm_forward(C.byref(a)))
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """(dx, dweight, dbias) from the forward call's mean and rstd; dx has the type of x, dweight and dbias are float32."""
    a, x = _ln_args("layer_norm_backward", x)
    _on_gpu("layer_norm_backward", x, dy, mean, rstd)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("layer_norm_backward: dy is %s %s, x %s %s" % (dy.dtype, tuple(dy.shape), x.dtype, tuple(x.shape)))
    for v in (mean, rstd):
        if v.dtype != torch.float32 or v.shape != (x.shape[0],):
            raise ValueError("layer_norm_backward: mean and rstd are float32 [%d]" % x.shape[0])
    weight = _ln_vector("layer_norm_backward", "weight", weight, x)
    dy, mean, rstd = _rows(dy), mean.contiguous(), rstd.contiguous()
    n, d = x.shape
    dx = torch.empty((n, d), dtype=x.dtype, device=x.device)
    cols = torch.empty((2, d), dtype=torch.float32, device=x.device)
    lib = library()
    need = _check(lib.gqe_layer_norm_workspace(C.byref(a)))
    space = torch.empty(need, dtype=torch.uint8, device=x.device)
    a.weight = None if weight is None else weight.data_ptr()
    a.mean, a.rstd, a.dy, a.dy_stride = mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), _row_stride(dy)
    a.dx, a.dx_stride, a.dweight, a.dbias = dx.data_ptr(), d, cols[0].data_ptr(), cols[1].data_ptr()
    a.workspace, a.workspace_bytes = space.data_ptr(), need
    _check(lib.gqe_layer_norm_backward(C.byref(a)))
    return dx, cols[0], cols[1]


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
    return _LayerNorm.apply(x.reshape(-1, x.shape[-1]), weight, bias, float(eps)).view(x.shape)
