"""The operators of include/gqe_ops.h against the formulas in 64 bits.

Bounds.  u = 2^-24 is half a step of float32, 2^-8 of bfloat16.  With Z = |scale| |q| |t| (largest over the rows) a logit computed in
float32 arithmetic is off by at most  dz = 12 u Z:  splitting loses 2^-22 = 4 u of each factor's product twice over (the split and
the dropped lo lo), the products' sum over d <= 256 in blocks of 16 rounds 16 times at no more than Z, and the scaling, the
unit length and the base-2 exponent round 3 times more - 8 u + 19 u at the very worst, 12 u with signs as they fall (and the
exponent's own rounding, u (|z| + |lse| + 16) log2 e, is added for e = dz + 2 u (Z + |lse| + 16)).
  lse, loss:  e + u (|lse| + 8)
  a softmax share, and 1 - the target's:  relative 2 e + 8 u;   every gradient is a sum of shares times inputs, so it is off by that
  times the sum of the magnitudes M = sum |share| |input| (computed in 64 bits), plus 64 u M for the sums, plus 2^-8 M where shares
  are rounded to bfloat16 and 2^-8 |result| where the result is."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dev():
    return torch.device("cuda", 0)


def xent_inputs(B, V, d, dtype, seed=0, normalize=False, ignored=0.0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    table = n(V, d) * spread / math.sqrt(d)
    target = torch.randint(0, V, (B,), generator=g, device="cuda")
    q = (n(B, d) + (2.0 * table[target] if B else 0.0)) * (1.0 / math.sqrt(d) if normalize else 1.0)
    if ignored:
        target = torch.where(torch.rand(B, generator=g, device="cuda") < ignored, -torch.randint(1, 9, (B,), generator=g, device="cuda"), target)
    weight = torch.rand(B, generator=g, device="cuda") + 0.1
    return q.to(dtype), table.to(dtype), target.to(torch.int32), weight


def xent_exact(q, table, target, weight, scale, normalize):
    """The formulas in 64 bits: values and, for the bounds, the magnitudes that each sum runs over."""
    Q, W = q.double(), table.double()
    length = W.norm(dim=1, keepdim=True)
    T = torch.where(length > 0, W / length, torch.zeros_like(W)) if normalize else W
    z = scale * (Q @ T.t().contiguous())
    lse = torch.logsumexp(z, 1)
    ok = target >= 0
    at = target.long().clamp(min=0)
    rest = torch.logsumexp(z.scatter(1, at[:, None], -math.inf), 1)
    diff = rest - z.gather(1, at[:, None])[:, 0]
    # log(1 + e^diff): lse - z_target itself cancels below 1e-16, in 64 bits too
    loss = torch.where(ok, diff.clamp(min=0) + torch.log1p(torch.exp(-diff.abs())), torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    c = p.clone()
    c.scatter_(1, at[:, None], -torch.exp(rest - lse)[:, None])
    c = c * (weight.double() * ok)[:, None] * scale
    dq = c @ T
    dt = c.t().contiguous() @ Q
    mag_dq, mag_dt = c.abs() @ T.abs(), c.abs().t().contiguous() @ Q.abs()
    if normalize:
        inv = torch.where(length > 0, 1 / length, torch.zeros_like(length))
        dt = (dt - T * (T * dt).sum(1, keepdim=True)) * inv
        mag_dt = (mag_dt + T.abs() * (T.abs() * mag_dt).sum(1, keepdim=True)) * inv
    Z = abs(scale) * float(Q.norm(dim=1).max() if len(Q) else 0.0) * float(T.norm(dim=1).max())
    return dict(loss=loss, lse=lse, dq=dq, dtable=dt, mag_dq=mag_dq, mag_dt=mag_dt, Z=Z)


def check_xent(got, e, dtype, normalize, what=""):
    loss, lse, dq, dtable = got
    big = float(e["lse"].abs().max()) if e["lse"].numel() else 0.0
    err = 12 * U * e["Z"] + 2 * U * (e["Z"] + big + 16)
    for name, x in (("loss", loss), ("lse", lse)):
        if x is not None and x.numel():
            off = (x.double() - e[name]).abs().max().item()
            assert off <= err + U * (big + 8), (what, name, off, err)
    rel = 2 * err + 8 * U + 64 * U + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    for name, x, mag in (("dq", dq, "mag_dq"), ("dtable", dtable, "mag_dt")):
        if x is None or not x.numel():
            continue
        tol = rel * e[mag] + (2.0 ** -8 if x.dtype == torch.bfloat16 else 4 * U) * e[name].abs() + 1e-37
        off = (x.double() - e[name]).abs()
        worst = (off / tol).max().item()
        assert worst <= 1.0, (what, name, worst)


XENT_SHAPES = [(1, 1, 1), (1, 64, 16), (3, 2, 5), (37, 1001, 48), (128, 128, 64), (129, 127, 65), (31, 33, 100), (200, 3001, 128), (300, 999, 130),
               (65, 2049, 192), (513, 700, 200), (64, 515, 255), (130, 1500, 256), (1500, 65, 96), (5000, 31, 33), (2, 60001, 24)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("B,V,d", XENT_SHAPES)
def test_softmax_xent_grads(B, V, d, normalize, dtype):
    from graphqembed_amd import ops
    scale = 20.0 if normalize else 1.0
    q, table, target, weight = xent_inputs(B, V, d, dtype, seed=B + V + d, normalize=normalize, ignored=0.15 if B > 8 else 0.0)
    got = ops.softmax_xent_grads(q, table, target, weight=weight, scale=scale, normalize=normalize)
    e = xent_exact(q, table, target, weight, scale, normalize)
    check_xent(got, e, dtype, normalize)
    again = ops.softmax_xent_grads(q, table, target, weight=weight, scale=scale, normalize=normalize)
    assert all(torch.equal(a, b) for a, b in zip(got, again))          # no atomics: the same bits
    loss, lse = ops.softmax_xent_loss(q, table, target, scale=scale, normalize=normalize)
    check_xent((loss, lse, None, None), e, dtype, normalize)
    assert got[2].dtype == got[3].dtype == dtype and loss.dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,d", [(333, 75842, 206), (700, 30001, 256), (1500, 9000, 100), (260, 60000, 48)])
def test_softmax_xent_losses_of_long_streams(B, V, d, dtype):
    """Losses alone take a tile's place for the next but one: many tiles to a workgroup, call after call the same bits."""
    from graphqembed_amd import ops
    for seed in range(6):
        q, table, target, weight = xent_inputs(B, V, d, dtype, seed=seed)
        loss, lse = ops.softmax_xent_loss(q, table, target)
        e = xent_exact(q, table, target, weight, 1.0, False)
        check_xent((loss, lse, None, None), e, dtype, False, seed)
        for _ in range(20):
            again = ops.softmax_xent_loss(q, table, target)
            assert torch.equal(again[0], loss) and torch.equal(again[1], lse), seed


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_softmax_xent_strided_and_unaligned(dtype):
    """Views: rows 1 .. n of a wider buffer at an odd element offset, 64-bit targets, weights of every sign, a negative scale."""
    from graphqembed_amd import ops
    B, V, d = 70, 513, 72
    q, table, target, weight = xent_inputs(B, V, d, dtype, seed=5, ignored=0.1)
    weight = weight - 0.6
    weight[3] = 0.0
    for pad, off in ((1, 1), (8, 8), (3, 0), (24, 4)):
        qw = torch.full((B + 1, d + pad), float("nan"), dtype=dtype, device=dev())
        tw = torch.full((V + 2, d + pad), float("nan"), dtype=dtype, device=dev())
        qv, tv = qw.view(-1)[off:off + B * (d + pad)].view(B, d + pad)[:, :d], tw[1:V + 1].reshape(-1)[:V * (d + pad)].view(V, d + pad)[:, :d]
        tv = tw[1:V + 1, pad:] if pad != 24 else tw[1:V + 1, :d]
        qv.copy_(q)
        tv.copy_(table)
        got = ops.softmax_xent_grads(qv, tv, target.long(), weight=weight, scale=-0.5)
        check_xent(got, xent_exact(q, table, target, weight, -0.5, False), dtype, False, (pad, off))
    qt = q.t().contiguous().t()                                          # column-major queries: copied by the call
    got = ops.softmax_xent_grads(qt, table, target, weight=weight)
    check_xent(got, xent_exact(q, table, target, weight, 1.0, False), dtype, False, "transposed")


@pytest.mark.parametrize("normalize", [False, True])
def test_softmax_xent_accumulates(normalize):
    from graphqembed_amd import ops
    for B, V, d in ((40, 300, 64), (600, 90, 33), (0, 50, 16)):          # direct, split along the queries, none
        q, table, target, weight = xent_inputs(B, V, d, torch.float32, seed=9)
        base = torch.randn(V + 1, d + 7, device=dev())
        into = base.clone()[1:, 3:3 + d]
        want = base[1:, 3:3 + d].double()
        out = ops.softmax_xent_grads(q, table, target, weight=weight, normalize=normalize, grad_table=into)
        assert out[3] is into
        if B:
            e = xent_exact(q, table, target, weight, 1.0, normalize)
            e["dtable"] = e["dtable"] + want
            check_xent(out, e, torch.float32, normalize)
            ops.softmax_xent_grads(q, table, target, weight=weight, normalize=normalize, grad_table=into)     # the same place twice
            e["dtable"] = 2 * e["dtable"] - want
            e["mag_dt"] = 2 * e["mag_dt"]
            check_xent((None, None, None, into), e, torch.float32, normalize)
        else:
            assert torch.equal(into.double(), want)


def test_softmax_xent_no_queries():
    from graphqembed_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        table = torch.randn(100, 48, device=dev()).to(dtype)
        q = torch.empty(0, 48, device=dev(), dtype=dtype)
        loss, lse, dq, dt = ops.softmax_xent_grads(q, table, torch.empty(0, dtype=torch.int32, device=dev()))
        assert loss.shape == lse.shape == (0,) and dq.shape == (0, 48) and not dt.any()
        loss = ops.softmax_xent(q.requires_grad_(), table, torch.empty(0, dtype=torch.int64, device=dev()))
        assert loss.item() == 0.0


def test_softmax_xent_targets_that_do_not_count():
    """All ignored: loss 0, gradients 0, lse as ever.  A target behind the table: NaN loss, no gradient, the others unharmed."""
    from graphqembed_amd import ops
    q, table, target, weight = xent_inputs(50, 300, 64, torch.float32, seed=3)
    none = torch.full_like(target, -1)
    loss, lse, dq, dt = ops.softmax_xent_grads(q, table, none, weight=weight)
    e = xent_exact(q, table, target, weight, 1.0, False)
    assert not loss.any() and not dq.any() and not dt.any()
    check_xent((None, lse, None, None), e, torch.float32, False)
    bad = target.clone()
    bad[7], bad[20] = 300, 2 ** 31 - 1
    loss, lse, dq, dt = ops.softmax_xent_grads(q, table, bad, weight=weight)
    kept = target.clone()
    kept[7] = kept[20] = -1
    e = xent_exact(q, table, kept, weight, 1.0, False)
    assert torch.isnan(loss[[7, 20]]).all()
    loss[7] = loss[20] = 0.0
    check_xent((loss, lse, dq, dt), e, torch.float32, False)
    ref = ops.softmax_xent(q, table, none)
    assert ref.item() == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_softmax_xent_answers_that_are_certain(dtype):
    """A query answered with probability 1 - 1e-9 .. 1 - 1e-30: loss and gradients keep their relative precision (the target's own
    term does not cancel), and with one row in the table everything is 0."""
    from graphqembed_amd import ops
    d, V = 64, 400
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(V, d, generator=g, device="cuda").to(dtype)
    target = torch.arange(0, 40, device="cuda", dtype=torch.int32) * 7
    q = (table[target.long()].float() * torch.linspace(0.3, 1.2, 40, device="cuda")[:, None]).to(dtype)
    w = torch.ones(40, device="cuda")
    got = ops.softmax_xent_grads(q, table, target, weight=w)
    e = xent_exact(q, table, target, w, 1.0, False)
    assert e["loss"].min() < 1e-20 and e["loss"].max() > 1e-9
    err = 12 * U * e["Z"] + 2 * U * (e["Z"] + float(e["lse"].abs().max()) + 16)
    assert ((got[0].double() - e["loss"]).abs() / e["loss"]).max().item() <= 2 * err + 8 * U
    check_xent(got, e, dtype, False)          # (the magnitudes are sums of the shares of the OTHER rows)
    got = ops.softmax_xent_grads(q, table[:1].contiguous(), torch.zeros_like(target))
    assert not got[0].any() and not got[2].any() and not got[3].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
def test_softmax_xent_rows_of_every_size(normalize, dtype):
    """Rows between 2^-40 and 2^40 times the others (and a row of zeros): each counts with its own precision."""
    from graphqembed_amd import ops
    B, V, d = 40, 260, 80
    q, table, target, weight = xent_inputs(B, V, d, dtype, seed=11, normalize=normalize)
    factor = 2.0 ** torch.randint(-40, 41 if normalize else 1, (V, 1), device="cuda").float()
    factor[::3] = 1.0
    table = (table.float() * factor).to(dtype)
    table[5] = 0
    qf = (q.float() * 2.0 ** torch.randint(-30, 1, (B, 1), device="cuda").float()).to(dtype)
    for qq in (q, qf):
        got = ops.softmax_xent_grads(qq, table, target, weight=weight, scale=4.0, normalize=normalize)
        assert all(torch.isfinite(x).all() for x in got)
        check_xent(got, xent_exact(qq, table, target, weight, 4.0, normalize), dtype, normalize)


def test_softmax_xent_large_logits():
    """Logits of +-3000 (no overflow of the exponentials) against the bound that their own rounding leaves."""
    from graphqembed_amd import ops
    q, table, target, weight = xent_inputs(64, 800, 96, torch.float32, seed=2, spread=3.0)
    got = ops.softmax_xent_grads(q, table, target, weight=weight, scale=60.0)
    e = xent_exact(q, table, target, weight, 60.0, False)
    assert float(e["lse"].max()) > 1000
    check_xent(got, e, torch.float32, False)


def test_softmax_xent_not_a_number():
    """A NaN in a query stays with that query's outputs (and its share of the table's gradient); a NaN row reaches every query."""
    from graphqembed_amd import ops
    q, table, target, weight = xent_inputs(70, 200, 48, torch.float32, seed=4)
    q[33, 5] = float("nan")
    loss, lse, dq, dt = ops.softmax_xent_grads(q, table, target, weight=weight)
    keep = torch.arange(70, device="cuda") != 33
    assert torch.isnan(loss[33]) and torch.isnan(lse[33]) and torch.isfinite(loss[keep]).all() and torch.isfinite(dq[keep]).all()
    assert torch.isnan(dt).any()
    q, table, target, weight = xent_inputs(70, 200, 48, torch.float32, seed=4)
    table[11, 0] = float("nan")
    loss, lse, dq, dt = ops.softmax_xent_grads(q, table, target, weight=weight)
    assert torch.isnan(loss).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("normalize", [False, True])
def test_softmax_xent_autograd_against_differences(normalize):
    from graphqembed_amd import ops
    q, table, target, _ = xent_inputs(33, 150, 40, torch.float32, seed=6, normalize=normalize, ignored=0.2)
    scale = 5.0
    q.requires_grad_()
    table.requires_grad_()
    ops.softmax_xent(q, table, target, scale=scale, normalize=normalize).backward()

    def value(Q, W):
        e = xent_exact(Q, W, target, torch.ones(33, device="cuda"), scale, normalize)
        return e["loss"].sum() / (target >= 0).sum()
    for x, grad, f in ((q, q.grad, lambda h, v: value(q.detach().double() + h * v, table.detach())),
                       (table, table.grad, lambda h, v: value(q.detach(), table.detach().double() + h * v))):
        v = torch.randn(x.shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(1))
        h = 1e-6
        want = ((f(h, v) - f(-h, v)) / (2 * h)).item()
        # differences: O(h^2) and 1e-16 / h; the gradient: float32 shares
        assert abs((grad.double() * v).sum().item() - want) <= 1e-5 * (grad.double() * v).abs().sum().item() + 1e-8
    # every reduction, and a loss that is used twice
    per = ops.softmax_xent(q, table, target, scale=scale, normalize=normalize, reduction="none")
    g1 = torch.autograd.grad((per * torch.arange(33, device="cuda")).sum() + per.sum(), (q, table))
    w = torch.arange(33, device="cuda", dtype=torch.float32) + 1
    _, _, dq, dt = ops.softmax_xent_grads(q.detach(), table.detach(), target, weight=w, scale=scale, normalize=normalize)
    e = xent_exact(q.detach(), table.detach(), target, w, scale, normalize)
    check_xent((None, None, g1[0], g1[1]), e, torch.float32, normalize)
    total = ops.softmax_xent(q, table, target, scale=scale, normalize=normalize, reduction="sum")
    assert abs(total.item() - per.sum().item()) <= 64 * U * per.abs().sum().item()


def test_softmax_xent_autograd_needs_only_one_side():
    from graphqembed_amd import ops
    q, table, target, _ = xent_inputs(33, 150, 40, torch.bfloat16, seed=6)
    ops.softmax_xent(q.requires_grad_(), table, target).backward()
    a = q.grad.clone()
    q = q.detach()
    ops.softmax_xent(q, table.requires_grad_(), target).backward()
    e = xent_exact(q, table.detach(), target, torch.full((33,), 1 / 33.0, device="cuda"), 1.0, False)
    check_xent((None, None, a, table.grad), e, torch.bfloat16, False)
    with torch.no_grad():
        assert torch.isfinite(ops.softmax_xent(q, table, target))


def test_softmax_xent_refusals():
    from graphqembed_amd import ops
    q, table, target, weight = xent_inputs(10, 20, 32, torch.float32)
    for call in (lambda: ops.softmax_xent_loss(q.half(), table.half(), target), lambda: ops.softmax_xent_loss(q, table.bfloat16(), target),
                 lambda: ops.softmax_xent_loss(q, table[:, :16], target), lambda: ops.softmax_xent_loss(q, table, target.float()),
                 lambda: ops.softmax_xent_loss(q, table, target[:9]), lambda: ops.softmax_xent_loss(q, table[:0], target),
                 lambda: ops.softmax_xent_grads(q, table, target, weight=weight.double()),
                 lambda: ops.softmax_xent_grads(q, table, target, weight=weight[:3]),
                 lambda: ops.softmax_xent_grads(q, table, target, grad_table=table[:10]),
                 lambda: ops.softmax_xent_grads(q, table, target, grad_table=table.bfloat16()),
                 lambda: ops.softmax_xent_loss(torch.randn(3, 257, device="cuda"), torch.randn(3, 257, device="cuda"), target[:3]),
                 lambda: ops.softmax_xent_loss(q[0], table, target)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops.GqeError):
        ops.softmax_xent_loss(q, table, target, scale=float("nan"))
    with pytest.raises(ops.GqeLibraryError):
        ops.softmax_xent_loss(q, table, target.cpu())


def test_softmax_xent_on_other_streams_and_in_a_graph():
    """Two streams at once; then a captured training step replayed between eager steps, each replay checked."""
    from graphqembed_amd import ops
    q, table, target, weight = xent_inputs(140, 2000, 64, torch.float32, seed=8)
    want = ops.softmax_xent_grads(q, table, target, weight=weight)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([ops.softmax_xent_grads(q, table, target, weight=weight) for _ in range(3)])
    torch.cuda.synchronize()
    for o in outs:
        for r in o:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.softmax_xent_grads(q, table, target, weight=weight)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse, dq, dt = ops.softmax_xent_grads(q, table, target, weight=weight)
        norm = ops.clip_grad_norm_([dq, dt], 0.01)
    for k in range(4):
        q2, t2, tg2, w2 = xent_inputs(140, 2000, 64, torch.float32, seed=20 + k)
        q.copy_(q2); table.copy_(t2); target.copy_(tg2); weight.copy_(w2)
        graph.replay()
        e = ops.softmax_xent_grads(q2, t2, tg2, weight=w2)
        n = ops.clip_grad_norm_([e[2], e[3]], 0.01)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, lse, dq, dt, norm), e + (n,)))


def test_softmax_xent_beyond_32_bit_offsets():
    """A table of more than 2^32 bytes' worth of elements: the last rows are reached (rows beyond 2^31 elements)."""
    from graphqembed_amd import ops
    V, d = 9_000_000, 256                        # 2.3e9 elements
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    table = torch.zeros(V, d, dtype=torch.bfloat16, device="cuda")
    table[-3:] = 0.25
    q = torch.ones(2, d, dtype=torch.bfloat16, device="cuda")
    target = torch.tensor([V - 1, 4], dtype=torch.int32, device="cuda")
    loss, lse, dq, dt = ops.softmax_xent_grads(q, table, target)
    want = math.log(3 * math.exp(64.0) + (V - 3))
    assert abs(lse[0].item() - want) < 64 * 32 * U and abs(loss[0].item() - (want - 64.0)) < 64 * 32 * U and abs(loss[1].item() - want) < 64 * 32 * U
    # row V - 1 is query 0's target (share 1/3 - 1) and a candidate of query 1 (share 1/3)
    assert abs(dt[-1, 0].item() - (2.0 / 3 - 1)) < 2.0 ** -8 and abs(dt[-2, 7].item() - 2.0 / 3) < 2.0 ** -7 and abs(dt[4, 1].item() + 1) < 2.0 ** -7
    assert float(dt[5:-3].abs().max()) < 1e-20


# -- gradient norm and clipping --------------------------------------------------------------------------------------------------

def clip_check(grads, max_norm, dtype):
    from graphqembed_amd import ops
    G = [g.double() for g in grads]
    want = math.sqrt(math.fsum(float((g * g).sum()) for g in G))
    norm = ops.clip_grad_norm_(grads, max_norm)
    assert abs(norm.item() - want) <= 2 * U * want + 1e-45
    c = min(1.0, max_norm / (want + 1e-6))
    step = 2.0 ** -8 if dtype == torch.bfloat16 else U
    for g, x in zip(G, grads):          # the factor rounds once, the product once
        assert ((x.double() - g * c).abs() <= (step + 2 * U) * (g * c).abs() + 1e-37).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5, 0], [63] * 5, [8191, 8192, 8193, 1, 16385], [3, 100000, 17], [2_000_003, 11], list(range(1, 230))])
def test_clip_grad_norm(sizes, dtype):
    for max_norm, factor in ((0.5, 1.0), (1e9, 1.0), (0.0, 1.0), (3.0, 1e-30), (1.0, 1e18)):
        if dtype == torch.bfloat16 and factor != 1.0:
            continue
        g = torch.Generator(device="cuda").manual_seed(len(sizes))
        clip_check([(torch.randn(n, generator=g, device="cuda") * factor).to(dtype) for n in sizes], max_norm, dtype)


def test_clip_grad_norm_views_and_mixed_types():
    """Tensors at every alignment inside one buffer, both types, neighbours left alone."""
    from graphqembed_amd import ops
    base = torch.randn(40000, device="cuda")
    half = torch.randn(40000, device="cuda").to(torch.bfloat16)
    b0, h0 = base.clone(), half.clone()
    views = [base[1:4], base[5:5000], base[5003:5003], base[6002:6003], base[7001:39999], half[3:4], half[5:20001], half[20002:39997]]
    c0 = [v.clone() for v in views]
    want = math.sqrt(sum(float((v.double() ** 2).sum()) for v in views))
    norm = ops.clip_grad_norm_(views, 1.0)
    assert abs(norm.item() - want) <= 2 * U * want
    c = 1.0 / (want + 1e-6)
    for v, o in zip(views, c0):
        step = 2.0 ** -8 if v.dtype == torch.bfloat16 else U
        assert ((v.double() - o.double() * c).abs() <= (step + 2 * U) * (o.double() * c).abs()).all()
    out = torch.ones(40000, dtype=torch.bool, device="cuda")
    for a, b in ((1, 4), (5, 5000), (6002, 6003), (7001, 39999)):
        out[a:b] = False
    assert torch.equal(base[out], b0[out])
    out[:] = True
    for a, b in ((3, 4), (5, 20001), (20002, 39997)):
        out[a:b] = False
    assert torch.equal(half[out], h0[out])


def test_clip_grad_norm_not_finite():
    """As the formula gives it: an infinite norm multiplies by 0 (inf * 0 = NaN), a NaN norm makes everything NaN."""
    from graphqembed_amd import ops
    a, b = torch.ones(100, device="cuda"), torch.ones(50, device="cuda").to(torch.bfloat16)
    a[7] = float("inf")
    assert ops.clip_grad_norm_([a, b], 1.0).item() == float("inf")
    assert torch.isnan(a[7]) and not a[:7].any() and not b.any()
    a[7] = float("nan")
    assert torch.isnan(ops.grad_norm([a, b]))
    assert torch.isnan(ops.clip_grad_norm_([a, b], 1.0)) and torch.isnan(a).all() and torch.isnan(b).all()
    z = torch.zeros(10, device="cuda")
    assert ops.clip_grad_norm_([z], 1.0).item() == 0.0 and not z.any()
    assert ops.grad_norm([torch.empty(0, device="cuda")]).item() == 0.0
    assert ops.clip_grad_norm_([torch.empty(0, device="cuda")], 1.0).item() == 0.0


def test_clip_grad_norm_refusals_and_bits():
    from graphqembed_amd import ops
    a = torch.randn(5, 8, device="cuda")
    for call in (lambda: ops.clip_grad_norm_([a.t()], 1.0), lambda: ops.clip_grad_norm_([a.double()], 1.0), lambda: ops.clip_grad_norm_([a], float("nan"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops.GqeError):
        ops.clip_grad_norm_([a, a], 1.0)
    with pytest.raises(ops.GqeError):
        ops.clip_grad_norm_([a, a[2]], 1.0)
    assert ops.grad_norm([a, a]).item() > 0.0           # reading twice is fine
    big = torch.randn(3_000_001, device="cuda")
    assert len({ops.grad_norm([big, a]).item() for _ in range(5)}) == 1


# -- layer normalisation -----------------------------------------------------------------------------------------------------------

def norm_exact(x, w, b, dy, eps):
    X, D = x.double(), dy.double()
    W, Bi = (1.0 if w is None else w.double()), (0.0 if b is None else b.double())
    mu = X.mean(1, keepdim=True)
    inv = 1 / torch.sqrt(((X - mu) ** 2).mean(1, keepdim=True) + eps)
    H = (X - mu) * inv
    A = D * W
    return dict(y=H * W + Bi, dx=inv * (A - A.mean(1, keepdim=True) - H * (A * H).mean(1, keepdim=True)), dw=(D * H).sum(0), db=D.sum(0), mu=mu, inv=inv, H=H, A=A, X=X, D=D)


LN_SHAPES = [(1, 1), (1, 2), (5, 3), (7, 31), (33, 32), (100, 64), (257, 100), (512, 128), (63, 200), (1000, 256), (77, 257), (40, 511), (9, 512), (50, 513),
             (31, 1000), (20, 1024), (11, 1025), (300, 2500), (6, 4096), (5, 4097), (3, 16384), (70000, 16), (9001, 48)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", LN_SHAPES)
def test_layer_norm(n, d, dtype):
    """Sums of d terms in float32 are off by at most 2 (4 + log2 d) u of their terms' magnitude here (lanes and halvings); xhat by
    that in the mean (times |mean| + spread over the spread) and in the variance.  Outputs round once more."""
    from graphqembed_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n + d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dy = (r(n, d) * 2 + 1).to(dtype), r(n, d).to(dtype)
    eps = 1e-5
    for w, b in ((1 + 0.3 * r(d), r(d)), (None, None), (1 + 0.3 * r(d), None)):
        y, mean, rstd = ops.layer_norm_forward(x, w, b, eps=eps)
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
        e = norm_exact(x, w, b, dy, eps)
        k = 2 * (4 + math.log2(d)) * U
        out = 2.0 ** -8 if dtype == torch.bfloat16 else 2 * U
        top = e["X"].abs().amax(1, keepdim=True)
        dH = 2 * k * top * e["inv"] + 2 * k * e["H"].abs() * (1 + top * e["inv"])            # error of xhat
        aw = 1.0 if w is None else w.double().abs()
        assert ((y.double() - e["y"]).abs() <= dH * aw + 2 * U * (e["H"].abs() * aw) + out * e["y"].abs() + U * e["y"].abs() + 1e-30).all()
        assert ((mean.double() - e["mu"][:, 0]).abs() <= k * top[:, 0]).all()
        assert ((rstd.double() - e["inv"][:, 0]).abs() <= 2 * k * (1 + top * e["inv"])[:, 0] * e["inv"][:, 0]).all()
        A, H = e["A"].abs(), e["H"].abs()
        hmean = (A * H).mean(1, keepdim=True)
        tol = e["inv"] * (4 * k * (A + A.mean(1, keepdim=True) + H * hmean) * (1 + top * e["inv"]) + dH * hmean + H * (A * dH).mean(1, keepdim=True)) + out * e["dx"].abs()
        assert ((dx.double() - e["dx"]).abs() <= tol + 1e-30).all()
        kn = 2 * (40 + math.log2(n + 1)) * U                                               # a thread's rows one after the other, then halvings
        kn += 2 * max(0, n // 1024) * U
        assert ((dw.double() - e["dw"]).abs() <= (kn * (e["D"].abs() * H) + e["D"].abs() * dH).sum(0) + 1e-30).all()
        assert ((db.double() - e["db"]).abs() <= kn * e["D"].abs().sum(0) + 1e-30).all()
        again = ops.layer_norm_backward(dy, x, mean, rstd, w)
        assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))
        if dtype == torch.bfloat16:
            break


def test_layer_norm_views_and_autograd():
    from graphqembed_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(3, 50, 91, device="cuda").to(dtype)
        x = wide[:, :, 1:78]
        w, b = torch.rand(77, device="cuda") + 0.5, torch.randn(77, device="cuda")
        xa = x.detach().clone().requires_grad_()
        wa, ba = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = ops.layer_norm(xa, wa, ba)
        dy = torch.randn(3, 50, 77, device="cuda").to(dtype)
        y.backward(dy)
        e = norm_exact(x.reshape(-1, 77), w, b, dy.reshape(-1, 77), 1e-5)
        rel = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18
        for got, want in ((y, e["y"]), (xa.grad, e["dx"]), (wa.grad, e["dw"]), (ba.grad, e["db"])):
            assert (got.double().reshape(want.shape) - want).norm() <= rel * want.norm()
        rows = x[1]                                           # strided rows, unaligned start
        y2, mean, rstd = ops.layer_norm_forward(rows, w, b)
        assert torch.equal(y2, y.detach()[1])
        got = ops.layer_norm_backward(wide[2, :, :77], rows, mean, rstd, w)
        e = norm_exact(rows, w, b, wide[2, :, :77], 1e-5)
        for a, c in zip(got, (e["dx"], e["dw"], e["db"])):
            assert (a.double() - c).norm() <= rel * c.norm()
    h = 1e-3                                                  # differences of the forward call itself (in float32: 2^-24 / h of its size)
    x = torch.randn(20, 33, device="cuda")
    v, c = torch.randn_like(x), torch.randn_like(x)
    xa = x.clone().requires_grad_()
    (ops.layer_norm(xa) * c).sum().backward()
    f = lambda t: (ops.layer_norm_forward(t)[0].double() * c.double()).sum().item()
    assert abs((f(x + h * v) - f(x - h * v)) / (2 * h) - (xa.grad.double() * v.double()).sum().item()) < 0.02


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_of_rows_without_spread(dtype):
    """Equal elements so large that one less the mean of a column past the row's end would overflow: xhat is 0, so dx = (dy - its
    mean) / sqrt(eps) and the weights' gradients are sums."""
    from graphqembed_amd import ops
    for n, d in ((3, 3), (2100, 13)):
        x = torch.full((n, d), 2.0 ** 122, device="cuda", dtype=dtype)          # (d of them: 2^126, the sums are exact)
        dy = torch.randn(n, d, device="cuda").to(dtype)
        y, mean, rstd = ops.layer_norm_forward(x)
        assert not y.any() and (mean == 2.0 ** 122).all()
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd)
        e = dy.double()
        want = (e - e.mean(1, keepdim=True)) * rstd.double()[:, None]
        half = torch.finfo(dtype).eps / 2
        # the mean: d + 2 roundings of at most the largest partial sum; then one difference, one product and the result's rounding
        bound = rstd.double()[:, None] * ((d + 5) * U * e.abs().sum(1, keepdim=True) + 3 * U * e.abs()) + half * want.abs() * 1.01
        assert ((dx.double() - want).abs() <= bound).all()
        assert not dw.any() and (db.double() - e.sum(0)).abs().max() <= 2 * n * U * e.abs().sum(0).max()


def test_a_run_of_operators_in_two_graphs():
    """Chain rows, layer norm, cross entropy, their backward passes and clipping, captured for two batches whose graphs share a memory
    pool and replayed in turn, eager steps between them: every replay has the eager bits."""
    from graphqembed_amd import ops
    V, d = 700, 96
    table = torch.randn(V, d, device="cuda")
    rels = [torch.randn(d, device="cuda") for _ in range(2)]
    w, b = torch.rand(d, device="cuda") + 0.5, torch.randn(d, device="cuda")

    def step(rows, target):
        grads = [torch.zeros_like(t) for t in [table] + rels + [w, b]]
        q = ops.chain_rows(table, rows, rels)
        y, mean, rstd = ops.layer_norm_forward(q, w, b)
        loss, lse, dy, _ = ops.softmax_xent_grads(y, table, target, normalize=True, grad_table=grads[0])
        dq, _, _ = ops.layer_norm_backward(dy, q, mean, rstd, w, grads[3], grads[4])
        ops.chain_rows_backward(dq, table, rows, rels, grads[0], grads[1:3])
        small = ops.clip_grad_norm_(grads[1:], 0.1)
        return [loss, lse, ops.clip_grad_norm_(grads, 0.5), small] + grads

    def batch(n):
        rows, target = (torch.randint(0, V, (n,), device="cuda", dtype=torch.int32) for _ in range(2))
        target[::5] = -1
        return rows, target

    feeds = [batch(150), batch(40)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in feeds:
            step(*f)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for f in feeds:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(step(*f))
    for _ in range(3):
        table.copy_(torch.randn(V, d, device="cuda"))
        for f, graph, out in zip(feeds, graphs, outs):
            for into, value in zip(f, batch(len(f[0]))):
                into.copy_(value)
            graph.replay()
            want = step(*f)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_autograd_forms_are_not_captured(monkeypatch):
    """What autograd would record raises inside a capture; what it would not is the plain call, and works there."""
    from graphqembed_amd import ops
    q, table, target, _ = xent_inputs(20, 300, 64, torch.float32, seed=5)
    qa, w = q.clone().requires_grad_(), torch.ones(64, device="cuda", requires_grad=True)
    norm = ops.layer_norm(q, w)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: ops.softmax_xent(qa, table, target), lambda: ops.softmax_xent(q, table.clone().requires_grad_(), target),
                 lambda: ops.layer_norm(qa), lambda: ops.layer_norm(q, w), lambda: ops.layer_norm(q, None, w)):
        with pytest.raises(ValueError, match="captured"):
            call()
    with torch.no_grad():
        got, same = ops.softmax_xent(qa, table, target, reduction="none"), ops.layer_norm(q, w)
    assert not got.requires_grad and torch.equal(same, norm)
    loss = ops.softmax_xent_loss(q, table, target)[0]
    assert torch.equal(got, loss)


@pytest.mark.parametrize("n,d,dtype", [(33000, 513, torch.float32), (17000, 1024, torch.float32), (70001, 481, torch.bfloat16)])
def test_layer_norm_of_large_outputs(n, d, dtype):
    """Outputs that are written past the caches: row for row the bits of a small call, the columns' sums by the formula."""
    from graphqembed_amd import ops
    x, dy = torch.randn(n, d, device="cuda").to(dtype), torch.randn(n, d, device="cuda").to(dtype)
    w, b = torch.rand(d, device="cuda") + 0.5, torch.randn(d, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    for i in (0, n // 2, n - 700):
        part = slice(i, i + 700)
        y2, mean2, rstd2 = ops.layer_norm_forward(x[part], w, b)
        dx2, _, _ = ops.layer_norm_backward(dy[part], x[part], mean2, rstd2, w)
        assert torch.equal(y[part], y2) and torch.equal(dx[part], dx2) and torch.equal(mean[part], mean2) and torch.equal(rstd[part], rstd2)
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    kn = (2 * (40 + math.log2(n)) + 2 * (n // 1024)) * U                # as above; xhat itself rounds 3 times more
    assert ((dw.double() - (dy.double() * h).sum(0)).abs() <= (kn + 4 * U) * (dy.double() * h).abs().sum(0)).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= kn * dy.double().abs().sum(0)).all()


def test_layer_norm_edges_and_refusals():
    from graphqembed_amd import ops
    flat = torch.full((4, 50), 3.0, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(flat, eps=1e-5)
    assert not y.any() and (mean == 3.0).all() and torch.isfinite(rstd).all()
    empty = torch.empty(0, 16, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(empty)
    dx, dw, db = ops.layer_norm_backward(empty, empty, mean, rstd)
    assert y.shape == dx.shape == (0, 16) and not dw.any() and not db.any()
    x = torch.randn(6, 40, device="cuda")
    x[2, 3] = float("nan")
    y, mean, rstd = ops.layer_norm_forward(x)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4, 5]]).all()
    far = torch.randn(30, 128, device="cuda") + 3e4           # a mean far above the spread: two passes, no cancellation
    e = norm_exact(far, None, None, far, 1e-5)
    assert ((ops.layer_norm_forward(far)[0].double() - e["y"]).abs() < 0.02).all()
    for call in (lambda: ops.layer_norm_forward(x, weight=torch.ones(39, device="cuda")), lambda: ops.layer_norm_forward(x.half()),
                 lambda: ops.layer_norm_forward(x, bias=torch.ones(40, device="cuda", dtype=torch.bfloat16)), lambda: ops.layer_norm_forward(x[0]),
                 lambda: ops.layer_norm_backward(x[:3], x, mean, rstd), lambda: ops.layer_norm_backward(x, x, mean[:2], rstd)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops.GqeError):
        ops.layer_norm_forward(x, eps=-1.0)
    with pytest.raises(ops.GqeError):
        ops.layer_norm_forward(torch.randn(2, 16385, device="cuda"))
