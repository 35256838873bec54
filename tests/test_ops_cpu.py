"""The operators of include/gqe_ops.h where no GPU is needed: every refusal comes from the host side of the C entry points, before
anything is launched; the binding's structures match the header; without a HIP device the Python calls raise."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ops():
    from graphqembed_amd import engine
    if not os.path.exists(engine.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    from graphqembed_amd import ops
    ops.library()
    return ops


def xent_args(ops, **kw):
    """A call that would be accepted, with made-up addresses: only refusals may be asked of it here."""
    a = ops.gqe_xent_args()
    a.phase, a.dtype, a.dim, a.n_queries, a.n_rows = 7, ops.F32, 64, 10, 100
    a.q = a.table = a.target = a.dq = a.dtable = a.stat = a.loss = a.lse = a.workspace = 1 << 20
    a.q_stride = a.table_stride = a.dq_stride = a.dtable_stride = 64
    a.scale, a.workspace_bytes = 1.0, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


XENT_REFUSED = [
    ("phase", dict(phase=0)), ("phase", dict(phase=8)), ("dtype", dict(dtype=2)), ("dtype", dict(dtype=-1)),
    ("dim", dict(dim=0)), ("dim", dict(dim=257)), ("rows", dict(n_rows=0)), ("rows", dict(n_rows=-1)), ("rows", dict(n_rows=1 << 31)),
    ("queries", dict(n_queries=-1)), ("queries", dict(n_queries=1 << 31)),
    ("NULL", dict(q=None)), ("NULL", dict(table=None)), ("NULL", dict(target=None)), ("dq is NULL", dict(dq=None)), ("dtable is NULL", dict(dtable=None)),
    ("stat", dict(phase=4, stat=None)), ("accumulate", dict(dtype=1, accumulate=1)),
    ("scale", dict(scale=float("inf"))), ("scale", dict(scale=float("nan"))),
    ("stride", dict(table_stride=63)), ("stride", dict(q_stride=63)), ("stride", dict(dtable_stride=0)), ("stride", dict(dq_stride=1)),
    ("aligned", dict(q=(1 << 20) + 2)), ("aligned", dict(dtable=(1 << 20) + 1)),
    ("workspace", dict()), ("workspace", dict(workspace=(1 << 20) + 128, workspace_bytes=1 << 40)), ("workspace", dict(workspace=None, workspace_bytes=1 << 40)),
]


@pytest.mark.parametrize("word,change", XENT_REFUSED)
def test_softmax_xent_refusals(ops, word, change):
    lib = ops.library()
    a = xent_args(ops, **change)
    rc = lib.gqe_softmax_xent(C.byref(a))
    assert rc in (-1, -5) and (rc == -5) == (word == "workspace")
    assert word in lib.gqe_ops_last_error().decode()


@pytest.mark.parametrize("change", [dict(dq=1 << 20), dict(dq=2 << 20), dict(dtable=1 << 20), dict(dtable=2 << 20)])
def test_softmax_xent_refuses_gradients_in_the_place_of_inputs(ops, change):
    lib = ops.library()
    a = xent_args(ops, **{**dict(q=1 << 20, table=2 << 20, dq=3 << 20, dtable=4 << 20, workspace_bytes=1 << 40), **change})
    assert lib.gqe_softmax_xent(C.byref(a)) == -1 and "shares memory" in lib.gqe_ops_last_error().decode()


@pytest.mark.parametrize("dx", [1 << 20, 2 << 20])
@pytest.mark.parametrize("n", [10, 5000])
def test_layer_norm_refuses_gradients_in_the_place_of_inputs(ops, n, dx):
    lib = ops.library()
    a = ops.gqe_layer_norm_args()
    a.dim, a.n_rows, a.x, a.dy, a.dx, a.dweight = 64, n, 1 << 20, 2 << 20, dx, 3 << 20
    a.mean = a.rstd = a.workspace = 4 << 20
    a.workspace_bytes, a.x_stride, a.dy_stride, a.dx_stride = 1 << 40, 64, 64, 64
    assert lib.gqe_layer_norm_backward(C.byref(a)) == -1 and "shares memory" in lib.gqe_ops_last_error().decode()


def test_chain_rows_refuse_results_in_the_place_of_inputs(ops):
    lib = ops.library()
    a = ops.gqe_chain_args()
    a.dim, a.n, a.n_rows, a.n_rels, a.rows, a.table, a.table_stride = 64, 4, 9, 2, 8 << 20, 1 << 20, 64
    a.rel[0], a.rel[1], a.drel[0], a.drel[1] = 2 << 20, 3 << 20, 4 << 20, 5 << 20
    a.q, a.q_stride, a.dq, a.dq_stride, a.dtable, a.dtable_stride, a.workspace, a.workspace_bytes = 1 << 20, 64, 6 << 20, 64, 1 << 20, 64, 7 << 20, 1 << 30
    for call in (lib.gqe_chain_rows_forward, lib.gqe_chain_rows_backward):
        assert call(C.byref(a)) == -1 and "shares memory with the table" in lib.gqe_ops_last_error().decode()
    a.dtable, a.drel[1] = 9 << 20, 2 << 20
    assert lib.gqe_chain_rows_backward(C.byref(a)) == -1 and "gradient 1 shares memory with relation 0" in lib.gqe_ops_last_error().decode()


def test_null_arguments(ops):
    lib = ops.library()
    assert lib.gqe_softmax_xent(None) == -1 and lib.gqe_softmax_xent_workspace(None) == -1
    assert lib.gqe_layer_norm_forward(None) == -1 and lib.gqe_layer_norm_backward(None) == -1 and lib.gqe_layer_norm_workspace(None) == -1
    assert lib.gqe_clip_grads(0, None, 3, 1.0, 1 << 20, 1 << 20, 1 << 30, None) == -1 and lib.gqe_clip_grads_workspace(None, 3) == -1


def test_softmax_xent_workspace(ops):
    """No logits are kept: up to 128 queries the workspace is a constant number of partial rows however large the table; beyond, the
    prepared operands come on top (as many bytes as float32 rows padded to 64 columns) with 24 bytes a row."""
    lib = ops.library()
    need = lambda **kw: lib.gqe_softmax_xent_workspace(C.byref(xent_args(ops, **kw)))
    assert need(dim=300) == -1
    parts = (256 + 8) * 128 * 4 * 300                           # (slots + a few) x rows of a workgroup x (d + sums) x 4 bytes
    assert 0 < need(n_rows=10000, n_queries=128, dim=256) < parts
    assert need(n_rows=100000000, n_queries=128, dim=256) < parts
    for dim, padded in ((256, 256), (100, 128), (130, 192), (7, 64)):
        big = need(n_rows=100000000, n_queries=512, dim=dim)
        assert 100000000 * padded * 4 < big < 100000000 * (padded * 4 + 25) + 2 * parts
        assert need(n_rows=100000000, n_queries=512, dim=dim, dtype=1) < 100000000 * (padded * 2 + 25) + 2 * parts
    assert need(n_rows=100000000, n_queries=128, dim=256, phase=1) < 1 << 20
    assert need(n_queries=0) == 256
    assert all(need(n_queries=n, n_rows=rows, dtype=dtype, phase=4, dim=40) > 0 for n in (0, 1, 600, 700) for rows in (1, 10240, 1 << 30) for dtype in (0, 1))
    assert need(n_rows=0x7fffff00, n_queries=0x7fffff00, dim=256, phase=2) > 0       # sizes stay in 64 bits


LN_REFUSED = [
    ("dtype", dict(dtype=3)), ("dim", dict(dim=0)), ("dim", dict(dim=16385)), ("rows", dict(n_rows=-1)), ("rows", dict(n_rows=1 << 31)),
    ("NULL", dict(x=None)), ("NULL", dict(mean=None)), ("NULL", dict(rstd=None)), ("aligned", dict(x=(1 << 20) + 2)), ("stride", dict(x_stride=7)),
]


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("word,change", LN_REFUSED)
def test_layer_norm_refusals(ops, word, change, backward):
    lib = ops.library()
    a = ops.gqe_layer_norm_args()
    a.dim, a.n_rows, a.eps = 64, 10, 1e-5
    a.x = a.y = a.dy = a.dx = a.mean = a.rstd = 1 << 20
    a.x_stride = a.y_stride = a.dy_stride = a.dx_stride = 64
    for k, v in change.items():
        setattr(a, k, v)
    rc = (lib.gqe_layer_norm_backward if backward else lib.gqe_layer_norm_forward)(C.byref(a))
    assert rc == -1 and word in lib.gqe_ops_last_error().decode()


def test_layer_norm_refuses_what_one_direction_needs(ops):
    lib = ops.library()
    a = ops.gqe_layer_norm_args()
    a.dim, a.n_rows, a.eps = 64, 10, float("nan")
    a.x = a.y = a.mean = a.rstd = 1 << 20
    a.x_stride = a.y_stride = a.dy_stride = a.dx_stride = 64
    assert lib.gqe_layer_norm_forward(C.byref(a)) == -1 and "eps" in lib.gqe_ops_last_error().decode()
    a.y, a.eps = None, 1e-5
    assert lib.gqe_layer_norm_forward(C.byref(a)) == -1 and "y is NULL" in lib.gqe_ops_last_error().decode()
    assert lib.gqe_layer_norm_backward(C.byref(a)) == -1 and "dy is NULL" in lib.gqe_ops_last_error().decode()
    a.dy = a.dweight = 1 << 20
    assert lib.gqe_layer_norm_workspace(C.byref(a)) == 0                      # few rows: one launch, no workspace
    a.n_rows = 5000
    assert lib.gqe_layer_norm_workspace(C.byref(a)) > 0
    assert lib.gqe_layer_norm_backward(C.byref(a)) == -5 and "workspace" in lib.gqe_ops_last_error().decode()


def tensors(ops, *spec):
    arr = (ops.gqe_tensor * len(spec))()
    for a, (data, numel, dtype) in zip(arr, spec):
        a.data, a.numel, a.dtype = data, numel, dtype
    return arr


@pytest.mark.parametrize("word,spec,max_norm", [
    ("dtype", [(1 << 20, 5, 7)], 1.0), ("no data", [(None, 5, 0)], 1.0), ("no data", [(1 << 20, -1, 0)], 1.0), ("aligned", [((1 << 20) + 2, 5, 0)], 1.0),
    ("aligned", [((1 << 20) + 1, 5, 1)], 1.0), ("NaN", [(1 << 20, 5, 0)], float("nan")),
    ("share memory", [(1 << 20, 100, 0), ((1 << 20) + 4096, 10, 0), ((1 << 20) + 396, 10, 0)], 1.0),
    ("share memory", [(1 << 20, 10, 0), (1 << 20, 10, 0)], 1.0), ("elements", [(1 << 20, 1 << 62, 1)], 1.0), ("elements", [(1 << 20, 1 << 50, 0)] * 2, -1.0)])
def test_clip_grads_refusals(ops, word, spec, max_norm):
    lib = ops.library()
    rc = lib.gqe_clip_grads(0, tensors(ops, *spec), len(spec), max_norm, 1 << 20, 1 << 20, 1 << 30, None)
    assert rc == -1 and word in lib.gqe_ops_last_error().decode()


def test_clip_grads_refuses_small_workspaces(ops):
    lib = ops.library()
    arr = tensors(ops, (1 << 20, 100, 0))
    need = lib.gqe_clip_grads_workspace(arr, 1)
    assert lib.gqe_clip_grads(0, arr, 1, 1.0, 1 << 20, 1 << 20, need - 1, None) == -5
    assert lib.gqe_clip_grads(0, arr, 1, 1.0, None, 1 << 20, need, None) == -1


CHAIN_REFUSED = [("dim", dict(dim=0)), ("dim", dict(dim=257)), ("queries", dict(n=-1)), ("queries", dict(n=65537)), ("table", dict(n_rows=0)),
                 ("relations", dict(n_rels=4)), ("relations", dict(n_rels=-1)), ("relation 0", dict(n_rels=1, rel=(C.c_void_p * 3)())),
                 ("NULL", dict(table=None)), ("NULL", dict(rows=None)), ("stride", dict(table_stride=63))]


@pytest.mark.parametrize("word,change", CHAIN_REFUSED + [("NULL", dict(q=None)), ("stride", dict(q_stride=3)), ("NULL", dict(dq=None)),
                                                         ("relation 1", dict(drel=(C.c_void_p * 3)(1 << 20, None, None))), ("NULL", dict(dtable=None)),
                                                         ("stride", dict(dtable_stride=1)), ("workspace", dict(workspace_bytes=8 * 10 * 64 - 1)),
                                                         ("workspace", dict(workspace=None))])
def test_chain_rows_refusals(ops, word, change):
    lib = ops.library()
    a = ops.gqe_chain_args(dim=64, n=10, n_rows=100, n_rels=2, workspace_bytes=1 << 20)
    a.rows = a.table = a.q = a.dq = a.dtable = a.workspace = 1 << 20
    a.table_stride = a.q_stride = a.dq_stride = a.dtable_stride = 64
    a.rel = a.drel = (C.c_void_p * 3)(1 << 20, 1 << 20, None)
    for k, v in change.items():
        setattr(a, k, v)
    both = [(lib.gqe_chain_rows_forward, ("q", "q_stride")), (lib.gqe_chain_rows_backward, ("dq", "drel", "dtable", "dtable_stride", "workspace", "workspace_bytes"))]
    only = [fn for fn, fields in both if set(fields) & set(change)]
    for fn in only or [fn for fn, _ in both]:
        assert fn(C.byref(a)) == (-5 if word == "workspace" else -1)
        assert word in lib.gqe_ops_last_error().decode()
    assert lib.gqe_chain_rows_forward(None) == -1 and lib.gqe_chain_rows_backward(None) == -1


def test_the_optimisers_and_the_trainer_refuse(ops):
    """max_grad_norm and the softmax loss need whole gradients and whole tables: refused before anything runs."""
    from graphqembed_amd.model import FusedAdam, FusedSGD
    from graphqembed_amd.trainer import TensorizedTrainer

    class Engine(object):
        world, sharded = 2, False

    class Model(object):
        engine = Engine()
    for kind in (FusedAdam, FusedSGD):
        assert kind(Model(), lr=0.1).max_grad_norm is None
        with pytest.raises(Exception, match="one GPU"):
            kind(Model(), lr=0.1, max_grad_norm=1.0)
        for bad in (-1.0, float("nan")):
            with pytest.raises(ValueError):
                kind(Model(), lr=0.1, max_grad_norm=bad)
    with pytest.raises(Exception, match="loss"):
        TensorizedTrainer(Model(), FusedSGD(Model(), 0.1), {}, {}, loss="softmax")
    with pytest.raises(Exception, match="loss"):
        TensorizedTrainer(Model(), FusedSGD(Model(), 0.1), {}, {}, loss="nce")


def test_the_binding_matches_the_header(ops):
    text = open(os.path.join(ROOT, "include", "gqe_ops.h")).read()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(gqe_\w+)\(", code))
    assert declared == set(ops.OPS_SYMBOLS)
    for struct in ("gqe_xent_args", "gqe_tensor", "gqe_layer_norm_args", "gqe_chain_args"):
        body = re.search(r"typedef struct \{([^{}]*)\} %s;" % struct, code).group(1)
        names = []
        for line in body.split(";"):
            line = line.strip()
            if line:
                kind = re.match(r"(?:const )?(int32_t|int64_t|float|void)\b", line).group(1)
                for part in line[line.index(kind) + len(kind):].split(","):
                    name, count = re.match(r"(\w+)(?:\[(\d+)\])?$", part.strip().lstrip("* ")).groups()
                    names.append((name, ("p" if "*" in line else kind) + (count or "")))
        types = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float, "p": C.c_void_p, "p3": C.c_void_p * 3}
        assert [(n, types[k]) for n, k in names] == getattr(ops, struct)._fields_
    for struct, packed in (("gqe_xent_args", ops._XENT), ("gqe_tensor", ops._TENSOR), ("gqe_layer_norm_args", ops._NORM)):
        kind = getattr(ops, struct)
        values = [i + 1 for i in range(len(kind._fields_))]
        a = kind.from_buffer_copy(packed.pack(*values))
        assert C.sizeof(kind) == packed.size and [getattr(a, n) for n, _ in kind._fields_] == values


def test_cpu_tensors_are_refused(ops):
    import torch
    from graphqembed_amd.engine import GqeLibraryError
    q, t, tgt = torch.randn(3, 8), torch.randn(5, 8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.softmax_xent_loss(q, t, tgt), lambda: ops.softmax_xent_grads(q, t, tgt), lambda: ops.softmax_xent(q, t, tgt),
                 lambda: ops.clip_grad_norm_([q], 1.0), lambda: ops.grad_norm([q]), lambda: ops.layer_norm(q), lambda: ops.layer_norm_forward(q),
                 lambda: ops.chain_rows(t, tgt, [t[0]]), lambda: ops.chain_rows_backward(q, t, tgt, [], t, [])):
        with pytest.raises(GqeLibraryError):
            call()
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([q], -1.0)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([], 1.0)
    with pytest.raises(ValueError):
        ops.softmax_xent(q, t, tgt, reduction="max")
