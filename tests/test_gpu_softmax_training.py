"""The operators of include/gqe_ops.h in the framework's own training: query rows of relation chains, the softmax loss of
QueryEncoderDecoder against every entity, the optimisers' gradient clipping, and all of them in a row.

u = 2^-24.  A chain's q is its row over a length: the squares' sum runs through 4 + 6 additions (5 u on its root), the reciprocal root and
the row's product 2 u, three relations 3 u - 12 u of |q| covers it.  Its gradient carries 16 u of the magnitudes M that its sums run over,
and one u more for each term added in a row (duplicates; n / 32 + 32 queries for the relations).  The model's losses and gradients are
compared with the same formulas in 64 bits; what 32 bits may cost there is taken from torch evaluating them in 32 bits: 8 times its own
largest error of each tensor, as the loss kernel's products round in 8 u + 4 u where a plain one rounds in 2 u, and 64 u of the tensor's
largest value as the floor where torch happens to be exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def chain_exact(table, rows, rels, dq):
    T = table.double().detach().requires_grad_()
    R = [r.double().detach().requires_grad_() for r in rels]
    w = T[rows.long()]
    length = w.norm(dim=1, keepdim=True)
    a = w / torch.where(length > 0, length, torch.ones_like(length)) * (length > 0)      # a zero row stays zero, and has no gradient
    q = a
    for r in R:
        q = q * r
    (q * dq.double()).sum().backward()
    ad = a.detach()
    prod = torch.ones(table.shape[1], dtype=torch.float64, device=table.device)
    for r in rels:
        prod = prod * r.double().abs()
    g = dq.double().abs() * prod
    inv = torch.where(length > 0, 1 / length, torch.zeros_like(length)).detach()
    M = (g + ad.abs() * (g * ad.abs()).sum(1, keepdim=True)) * inv
    mag = torch.zeros_like(T).index_add_(0, rows.long(), M)
    S = (dq.double().abs() * ad.abs()).sum(0)
    mag_r = []
    for j in range(len(rels)):
        m = S.clone()
        for i, r in enumerate(rels):
            if i != j:
                m = m * r.double().abs()
        mag_r.append(m)
    return q.detach(), T.grad, [r.grad for r in R], mag, mag_r


@pytest.mark.parametrize("n,V,d,k", [(1, 1, 1, 0), (1, 5, 16, 1), (7, 3, 33, 2), (512, 1000, 128, 3), (513, 40, 256, 1), (65, 9, 100, 3), (3000, 2000, 255, 2)])
def test_chain_rows(n, V, d, k):
    from graphqembed_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n + V + d)
    wide = torch.randn(V + 1, d + 5, generator=g, device="cuda") / d
    table = wide[1:, 2:2 + d]
    if V > 4:
        table[2] = 0.0
        table[3] *= 1e-30
    rows = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    rels = [torch.rand(d, generator=g, device="cuda") - 0.5 for _ in range(k)]
    dq = torch.randn(n, d, generator=g, device="cuda")
    q, dt, dr, mag, mag_r = chain_exact(table, rows, rels, dq)
    got = ops.chain_rows(table, rows, rels)
    assert (got.double() - q).abs().le(12 * U * q.abs() + 1e-45).all()
    base, rbase = torch.randn(V, d, generator=g, device="cuda"), [torch.randn(d, generator=g, device="cuda") for _ in rels]
    gt, gr = torch.full((V, d + 3), 7.0, device="cuda"), [b.clone() for b in rbase]
    gt[:, :d] = base
    ops.chain_rows_backward(dq, table, rows, rels, gt[:, :d], gr)
    again, gr2 = base.clone(), [b.clone() for b in rbase]
    ops.chain_rows_backward(dq, table, rows, rels, again, gr2)
    assert torch.equal(gt[:, :d], again) and all(torch.equal(a, b) for a, b in zip(gr, gr2)) and (gt[:, d:] == 7.0).all()
    most = int(torch.bincount(rows.long()).max())
    assert ((again.double() - base.double()) - dt).abs().le((16 + most) * U * mag + U * (again.double().abs() + base.double().abs())).all()
    for a, b, want, m in zip(gr, rbase, dr, mag_r):
        assert ((a.double() - b.double()) - want).abs().le((16 + n / 32 + 32) * U * m + U * (a.double().abs() + b.double().abs())).all()
    untouched = torch.ones(V, dtype=torch.bool, device="cuda")
    untouched[rows.long()] = False
    assert torch.equal(again[untouched], base[untouched])


def test_chain_rows_repeats_and_bad_rows():
    """The same relation twice, rows outside the table (NaN embeddings, no gradient, nothing read or written), no queries."""
    from graphqembed_amd import ops
    d, V = 24, 6
    table, r = torch.randn(V, d, device="cuda"), torch.rand(d, device="cuda") + 0.5
    rows = torch.tensor([2, -1, 2, V, 0], dtype=torch.int32, device="cuda")
    q = ops.chain_rows(table, rows, [r, r])
    assert torch.isnan(q[[1, 3]]).all() and torch.isfinite(q[[0, 2, 4]]).all()
    dq = torch.randn(5, d, device="cuda")
    gt, gr = torch.zeros(V, d, device="cuda"), torch.zeros(d, device="cuda")
    ops.chain_rows_backward(dq, table, rows, [r, r], gt, [gr, gr])
    good = [0, 2, 4]
    _, dt, dr, mag, mag_r = chain_exact(table, rows[good], [r, r], dq[good])
    assert (gt.double() - dt).abs().le(24 * U * mag).all()
    assert (gr.double() - (dr[0] + dr[1])).abs().le(64 * U * (mag_r[0] + mag_r[1])).all()
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.chain_rows(table, empty, [r]).shape == (0, d)
    ops.chain_rows_backward(torch.empty(0, d, device="cuda"), table, empty, [r], gt, [gr])


# ---- the model -----------------------------------------------------------------------------------------------------------------
SIZES = {"a": 400, "b": 37, "c": 1}
REL = {"a": [("b", "x"), ("a", "y")], "b": [("a", "x"), ("c", "z")], "c": [("b", "z")]}
CHAINS = [("1-chain", (("a", "x", "b"),)), ("2-chain", (("b", "x", "a"), ("a", "y", "a"))), ("3-chain", (("a", "y", "a"), ("a", "y", "a"), ("a", "x", "b"))),
          ("1-chain", (("c", "z", "b"),))]


def build(d=32, decoder="bilinear-diag", seed=0, **kw):
    from graphqembed_amd import utils
    from graphqembed_amd.graph import Formula, Graph
    from graphqembed_amd.model import QueryEncoderDecoder
    torch.manual_seed(seed)
    maps = {m: {i: i for i in range(n)} for m, n in SIZES.items()}
    dims = {m: d for m in SIZES}
    graph = Graph(None, dims, REL, {})
    features = {m: torch.nn.Embedding(n + 1, d) for m, n in SIZES.items()}
    for f in features.values():
        f.weight.data.normal_(0, 1.0 / d)
    enc = utils.get_encoder(0, graph, dims, features, True, node_maps=maps)
    model = QueryEncoderDecoder(graph, enc, utils.get_metapath_decoder(graph, dims, decoder), utils.get_intersection_decoder(graph, dims, "mean"), **kw)
    if hasattr(model, "query_norm"):
        model.query_norm.weight.data.uniform_(0.5, 1.5)
        model.query_norm.bias.data.uniform_(-0.2, 0.2)
    return model, [Formula(t, rels if t != "1-chain" else rels) for t, rels in CHAINS]


def batches(formulas, rng, n=50):
    out = []
    for i, f in enumerate(formulas):
        k = n + 13 * i
        target = rng.randint(0, SIZES[f.target_mode] + 1, size=k).astype(np.int32)       # 0: the dummy row, ignored
        out.append((f, target, rng.randint(0, SIZES[f.anchor_modes[0]] + 1, size=(1, k)).astype(np.int32), 1.0 - 0.3 * i))
    return out


def plain(model, items, scale, dtype, params=None):
    """losses and gradients by torch's autograd on the CPU"""
    p = {k: v.detach().cpu().to(dtype).requires_grad_() for k, v in (params or dict(model.named_parameters())).items()}
    total, losses = 0.0, []
    for f, target, anchors, weight in items:
        unit = lambda w: w / w.norm(dim=1, keepdim=True)
        q = unit(p["enc.feat-%s.weight" % f.anchor_modes[0]][torch.from_numpy(anchors[0]).long()])
        for r in f.rels:
            q = q * p["path_dec." + "_".join(r)]
        if "query_norm.weight" in p:
            q = torch.nn.functional.layer_norm(q, (q.shape[1],), p["query_norm.weight"], p["query_norm.bias"], model.query_norm.eps)
        z = scale * q @ unit(p["enc.feat-%s.weight" % f.target_mode][1:]).t()
        t = torch.from_numpy(target).long() - 1
        loss = torch.where(t >= 0, torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros((), dtype=dtype))
        losses.append(loss.sum() / max(int((t >= 0).sum()), 1))
        total = total + weight * losses[-1]
    total.backward()
    return torch.stack(losses + [total]).detach(), {k: torch.zeros_like(v) if v.grad is None else v.grad for k, v in p.items()}


def read_grads(model):
    model.engine.materialize()
    return {k: model.layout.view(model.engine.grads, k).cpu() for k in model.layout.entries}


def close(got, exact, single, what):
    got, exact, single = got.double().cpu(), exact.double(), single.double()
    tol = 8 * (single - exact).abs().max().item() + 64 * U * exact.abs().max().item()
    off = (got - exact).abs().max().item()
    assert off <= tol, (what, off, tol)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d", [16, 48, 128])
def test_softmax_step(d, norm):
    """Losses and gradients of four chains in one call; then against differences of the formula in 64 bits."""
    model, formulas = build(d, query_norm=norm)
    scale = 1.5 if norm else 300.0
    items = batches(formulas, np.random.RandomState(d))
    losses = model.softmax_step(items, scale)
    exact, grads = plain(model, items, scale, torch.float64)
    single, grads32 = plain(model, items, scale, torch.float32)
    close(losses, exact, single, "losses")
    got = read_grads(model)
    for k in grads:
        close(got[k], grads[k], grads32[k], k)
    touched = set().union(*[model._softmax_keys(f) for f in formulas])
    assert model._touched == touched and ("query_norm.bias" in touched) == norm
    for i, (f, target, anchors, w) in enumerate(items):
        each = model.softmax_losses(f, target, anchors, scale)
        assert each.shape == (len(target),) and (each[torch.from_numpy(target == 0).cuda()] == 0).all()
        close(each.sum() / max((target > 0).sum(), 1), exact[i], single[i], "softmax_losses")
    # along a random direction v: (L(p + h v) - L(p - h v)) / 2 h, off by h^2 of the third derivative and 1e-16 / h
    g = torch.Generator().manual_seed(1)
    p = {k: v.detach().cpu().double() for k, v in model.named_parameters()}
    v = {k: torch.randn(x.shape, generator=g, dtype=torch.float64) * (x.norm(dim=-1, keepdim=True) / d ** 0.5) for k, x in p.items()}
    h = 1e-5
    up, down = (plain(model, items, scale, torch.float64, {k: p[k] + s * h * v[k] for k in p})[0][-1].item() for s in (1, -1))
    along = sum(float((got[k].double() * v[k]).sum()) for k in p)
    slack = sum(float((v[k].abs()).sum()) * (8 * (grads32[k].double() - grads[k]).abs().max().item() + 64 * U * grads[k].abs().max().item()) for k in p)
    assert abs(along - (up - down) / (2 * h)) <= slack + 1e-6 * abs(along) + 1e-9


def test_softmax_step_next_to_margin_step():
    """Both losses in one iteration: their gradients add up, and the optimiser leaves the gradient arena clean."""
    from graphqembed_amd.model import FusedAdam
    model, formulas = build(48, query_norm=True)
    items = batches(formulas, np.random.RandomState(3))
    margin = [(f, np.maximum(t, 1), np.roll(np.maximum(t, 1), 1), np.maximum(a, 1), w, 1.0) for f, t, a, w in items]
    model.margin_step(margin)
    one = read_grads(model)
    model.engine.zero_grads(list(model.layout.entries))
    model.softmax_step(items, 1.5)
    two = read_grads(model)
    model.engine.zero_grads(list(model.layout.entries))
    for first, second in ((lambda: model.margin_step(margin), lambda: model.softmax_step(items, 1.5)),
                          (lambda: model.softmax_step(items, 1.5), lambda: model.margin_step(margin))):
        first()
        second()
        both = read_grads(model)
        for k in both:
            # (float atomics in the margin launch: its sums come in another order, 64 u of the largest term's reach)
            assert (both[k] - one[k] - two[k]).abs().max().item() <= 256 * U * (one[k].abs().max() + two[k].abs().max()).item(), k
        FusedAdam(model, lr=0.0).step()
        assert all(not g.any() for g in read_grads(model).values())


@pytest.mark.parametrize("lazy", [False, True])
def test_softmax_training_steps_like_torch(lazy):
    """Six iterations of query rows -> layer norm -> softmax loss -> clipping -> Adam against torch's modules and optimiser in
    64 bits on the CPU; margin iterations between them in lazy mode's deferred rows included."""
    from graphqembed_amd.model import FusedAdam
    model, formulas = build(32, query_norm=True, lazy_adam=lazy)
    opt = FusedAdam(model, lr=0.01, max_grad_norm=0.05)
    ref = {k: torch.nn.Parameter(v.detach().cpu().double()) for k, v in model.named_parameters()}
    topt = torch.optim.Adam(list(ref.values()), lr=0.01)
    rng = np.random.RandomState(4)
    for it in range(6):
        items = batches(formulas[:2] if it % 2 else formulas, rng, 40)
        losses = model.softmax_step(items, 1.5)
        exact, grads = plain(model, items, 1.5, torch.float64, ref)
        assert abs(losses[-1].item() - exact[-1].item()) <= 2e-4 * abs(exact[-1].item())
        opt.step()
        touched = set().union(*[model._softmax_keys(item[0]) for item in items])
        for k, p in ref.items():
            p.grad = grads[k] if k in touched else None
        norm = torch.nn.utils.clip_grad_norm_([p for p in ref.values() if p.grad is not None], 0.05)
        assert norm > 0.05 and abs(opt.grad_norm.item() - norm.item()) <= 1e-3 * norm.item()
        topt.step()
    state = {k: v.cpu().double() for k, v in model.state_dict().items()}
    for k, p in ref.items():
        # Adam turns the sign of a gradient that is rounding noise into a move of lr per step: at most that anywhere, and 1e-4 (of
        # lr 0.01: a relative gradient error of about 1e-2 near Adam's first steps' knee) at all but a few of the elements
        off = (state[k] - p.detach()).abs()
        assert off.max().item() <= 2 * 6 * 0.011, k
        assert (off > 1e-4).double().mean().item() <= 0.02, (k, off.max().item())


@pytest.mark.parametrize("norm", [False, True])
def test_softmax_loss_is_differentiable(norm):
    model, formulas = build(32, query_norm=norm)
    f = formulas[1]
    rng = np.random.RandomState(5)
    n = 30
    target, anchors = rng.randint(0, SIZES[f.target_mode], n), rng.randint(0, SIZES[f.anchor_modes[0]], n)

    class Q(object):
        def __init__(self, t, a):
            self.target_node, self.anchor_nodes = t, (a,)
    queries = [Q(t, a) for t, a in zip(target, anchors)]
    items = [(f, (target + 1).astype(np.int32), (anchors + 1).astype(np.int32)[None], 1.0)]
    exact, grads = plain(model, items, 300.0, torch.float64)
    single, grads32 = plain(model, items, 300.0, torch.float32)
    for p in model.parameters():
        p.grad = None
    loss = model.softmax_loss(f, queries, scale=300.0)
    close(loss.detach(), exact[0], single[0], "loss")
    (2.0 * loss).backward()
    for k in model._softmax_keys(f):
        close(model._param(k).grad, 2 * grads[k], 2 * grads32[k], k)
    for p in model.parameters():
        p.grad = None
    model.softmax_loss(f, queries, scale=300.0).backward()          # starts from zero again
    for k in model._softmax_keys(f):
        close(model._param(k).grad, grads[k], grads32[k], k)


def test_softmax_trainer_steps_with_clipping():
    from graphqembed_amd.model import FusedAdam, FusedSGD
    from graphqembed_amd.trainer import TensorizedTrainer

    class Pool(object):
        def __init__(self, f, seed):
            rng = np.random.RandomState(seed)
            self.formula, self.n = f, 300
            self.anchors = rng.randint(1, SIZES[f.anchor_modes[0]] + 1, size=(1, self.n)).astype(np.int32)
            self.target = rng.randint(1, SIZES[f.target_mode] + 1, size=self.n).astype(np.int32)
    for opt_type in (FusedAdam, FusedSGD):
        model, formulas = build(32, query_norm=True)
        pools = {"1-chain": [Pool(formulas[0], 1)], "2-chain": [Pool(formulas[1], 2)], "3-chain": [Pool(formulas[2], 3)]}
        opt = opt_type(model, lr=0.01, max_grad_norm=1.0)
        tr = TensorizedTrainer(model, opt, pools, {}, batch_size=128, loss="softmax")
        seen = [tr.step(it).clone() for it in range(4)]
        assert all(s.shape == (4,) and torch.isfinite(s).all() for s in seen) and tr.queries_seen == 3 * (128 + 128 + 44) + 3 * 128
        assert opt.grad_norm.item() > 0 and not model._touched


def test_clipping_of_the_fused_optimisers():
    """max_grad_norm on the margin loss: the step equals a step on gradients scaled by hand; a norm that nothing reaches changes no
    bit of what a plain step does."""
    from graphqembed_amd.model import FusedSGD
    def run(max_norm, by_hand=None):
        model, formulas = build(32, seed=2)
        items = batches(formulas, np.random.RandomState(6))
        margin = [(f, np.maximum(t, 1), np.roll(np.maximum(t, 1), 1), np.maximum(a, 1), w, 1.0) for f, t, a, w in items]
        before = {k: v.detach().clone() for k, v in model.named_parameters()}
        model.margin_step(margin)
        grads = read_grads(model)
        opt = FusedSGD(model, lr=1.0, max_grad_norm=max_norm)
        opt.step()
        after = model.state_dict()
        return grads, {k: (before[k] - after[k]).cpu() for k in before}, opt.grad_norm, before
    grads, moved, none, before = run(None)
    assert none is None
    norm = sum(float((g.double() ** 2).sum()) for g in grads.values()) ** 0.5
    grads, moved, got, before = run(norm / 4)
    # the norm's sum is in 64 bits, each gradient 32: u; the factor, the product and the step's subtraction 3 u more, atomics' order 64 u
    assert abs(got.item() - norm) <= 64 * U * norm
    for k in grads:
        want = grads[k].double() * (norm / 4) / (norm + 1e-6)
        assert (moved[k].double() - want).abs().max().item() <= 80 * U * (want.abs().max().item() + before[k].abs().max().item()), k
    grads, moved, got, before = run(norm * 4)
    for k in grads:
        assert (moved[k].double() - grads[k].double()).abs().max().item() <= 4 * U * (grads[k].abs().max().item() + before[k].abs().max().item()), k


def test_train_step_with_clipping_is_margin_step_and_step():
    """model.train_step / TensorizedTrainer take the clipped way by themselves (matrices' deferred launch included)."""
    from graphqembed_amd.model import FusedAdam
    out = []
    for way in range(2):
        model, formulas = build(32, decoder="bilinear", seed=3)
        items = batches(formulas, np.random.RandomState(7))
        margin = [(f, np.maximum(t, 1), np.roll(np.maximum(t, 1), 1), np.maximum(a, 1), w, 1.0) for f, t, a, w in items]
        model.engine.set_deferred_gemm(way == 0)
        opt = FusedAdam(model, lr=0.01, max_grad_norm=1e-3)
        if way == 0:
            losses = model.train_step(margin, opt)
        else:
            losses, _, _ = model.margin_step(margin)
            opt.step()
        assert not model._touched and abs(opt.grad_norm.item()) > 1e-3
        out.append((losses.cpu(), opt.grad_norm.cpu()))
    assert torch.allclose(out[0][0], out[1][0], rtol=1e-5) and torch.allclose(out[0][1], out[1][1], rtol=1e-4)


def test_softmax_step_on_empty_and_ignored_batches():
    """A batch without queries and one whose targets are all the dummy row: loss 0, no gradient."""
    model, formulas = build(32, query_norm=True)
    none = np.zeros(0, np.int32)
    items = [(formulas[0], none, none[None], 1.0), (formulas[1], np.zeros(5, np.int32), np.ones((1, 5), np.int32), 2.0)]
    losses = model.softmax_step(items, 1.5)
    assert (losses == 0).all() and all(not g.any() for g in read_grads(model).values())
    assert model.softmax_losses(formulas[0], none, none[None]).shape == (0,)


def test_softmax_step_on_another_stream():
    """The calls follow torch's current stream."""
    from graphqembed_amd.model import FusedSGD
    out = []
    for side in (False, True):
        model, formulas = build(32, query_norm=True, seed=4)
        items = batches(formulas, np.random.RandomState(8))
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
            opt = FusedSGD(model, lr=0.1, max_grad_norm=0.5)
            losses = [model.softmax_step(items, 1.5).clone()]
            opt.step()
            losses.append(model.softmax_step(items, 1.5).clone())
        torch.cuda.synchronize()
        out.append(torch.stack(losses).cpu())
    assert torch.equal(out[0], out[1]) and out[0][1, -1] != out[0][0, -1]


def test_softmax_refusals():
    from graphqembed_amd.graph import Formula
    from graphqembed_amd.model import FusedAdam
    model, formulas = build(16)
    inter = Formula("2-inter", (("a", "x", "b"), ("a", "y", "a")))
    one = np.ones(3, np.int32)
    for call in (lambda: model.softmax_step([(inter, one, np.ones((2, 3), np.int32), 1.0)]),
                 lambda: model.softmax_losses(formulas[0], np.full(3, SIZES["a"] + 1, np.int32), one[None]),
                 lambda: model.softmax_losses(formulas[0], one, -one[None]),
                 lambda: model.softmax_losses(formulas[0], one, np.ones((1, 4), np.int32))):
        with pytest.raises(Exception):
            call()
    for call in (lambda: model.softmax_step([]), lambda: model.softmax_step([(formulas[0], one, one[None], 1.0)], scale=float("inf")),
                 lambda: model.softmax_step([(formulas[0], np.ones(65537, np.int32), np.ones((1, 65537), np.int32), 1.0)])):
        with pytest.raises(Exception):
            call()
    assert not model._touched and all(not g.any() for g in read_grads(model).values())
    with pytest.raises(ValueError):
        FusedAdam(model, max_grad_norm=float("nan"))
    other, f = build(16, decoder="transe")
    with pytest.raises(Exception):
        other.softmax_losses(f[0], one, one[None])
