"""The operators of training against a whole entity table, as cases that can be timed and checked: the softmax cross entropy of
query embeddings over every row of a table with its gradients, the global gradient norm with clipping, and layer normalisation
with its backward pass.

``run`` computes a case in plain torch operations, or (``own`` set) through graphqembed_amd.ops; ``exact`` computes it in 64 bits
from the formulas.  Table sizes are those of the synthetic graphs in graphqembed_amd/data_utils.py and synth.py (10 000 drugs,
27 000 functions, 40 000 proteins, 500 000 users), d = 128 and 256, batches of 512 queries and of 9 x 512 (the full mix)."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
XENT_MAX_LOGITS = 4608 * 131071         # the largest listed case: queries x entities, and the same times d
XENT_MAX_WORK = XENT_MAX_LOGITS * 256


def listed():
    return [
        # one 1-chain batch of a training step against all proteins: unit rows (the encoder normalises), cosine logits at 1 / 0.05
        {"name": "xent step proteins", "op": "xent", "grads": True, "B": 512, "V": 40000, "d": 128, "dtype": "f32", "normalize": True, "scale": 20.0, "ignored": 0.0},
        # the same against the largest table of the Reddit-shaped graph: few queries, many rows, a gradient as large as the table
        {"name": "xent step users", "op": "xent", "grads": True, "B": 512, "V": 500000, "d": 256, "dtype": "f32", "normalize": True, "scale": 20.0, "ignored": 0.0},
        # nine batches at once in bfloat16 on raw rows (an output projection's weight), an odd number of rows, some targets ignored
        {"name": "xent step bf16 odd", "op": "xent", "grads": True, "B": 4608, "V": 131071, "d": 256, "dtype": "bf16", "normalize": False, "scale": 1.0, "ignored": 0.05},
        # the last, short slice of a formula's queries on a small mode: latency, ragged everywhere
        {"name": "xent step ragged", "op": "xent", "grads": True, "B": 37, "V": 1001, "d": 48, "dtype": "f32", "normalize": False, "scale": 1.0, "ignored": 0.1},
        # validation of a whole mix of queries: losses only
        {"name": "xent loss functions", "op": "xent", "grads": False, "B": 4608, "V": 27000, "d": 128, "dtype": "f32", "normalize": True, "scale": 20.0, "ignored": 0.0},
        # a single query answered against all drugs: latency
        {"name": "xent loss one query", "op": "xent", "grads": False, "B": 1, "V": 10000, "d": 128, "dtype": "f32", "normalize": True, "scale": 20.0, "ignored": 0.0},
        # a handful of relation vectors and two matrices, odd sizes
        {"name": "clip few", "op": "clip", "tables": 0, "rows": 0, "d": 63, "vectors": 14, "matrices": 2, "dtype": "f32"},
        # the gradients of the five-mode graph at d = 128: five tables, 14 relation vectors, Pre / Post of five modes
        {"name": "clip five modes", "op": "clip", "tables": 5, "rows": 19402, "d": 128, "vectors": 14, "matrices": 10, "dtype": "f32"},
        # three tables of 300 000 rows at d = 256 kept in bfloat16
        {"name": "clip bf16 tables", "op": "clip", "tables": 3, "rows": 300001, "d": 256, "vectors": 12, "matrices": 6, "dtype": "bf16"},
        # one batch of query embeddings, forward and backward: latency
        {"name": "norm one batch", "op": "norm", "n": 512, "d": 128, "dtype": "f32"},
        # nine batches, an odd number of rows and a width that no vector divides, bfloat16 rows with float32 gain and bias
        {"name": "norm odd bf16", "op": "norm", "n": 4609, "d": 257, "dtype": "bf16"},
        # all users' rows at once, the widest embedding: bandwidth
        {"name": "norm users", "op": "norm", "n": 500000, "d": 256, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "xent", "clip", "norm"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "xent":
        d = rng.randint(8, 256)
        B = _spread(rng, 1, 4608)
        V = _spread(rng, 64, max(65, min(500000, XENT_MAX_LOGITS // B, XENT_MAX_WORK // (B * d))))
        normalize = rng.random() < 0.5
        return {"op": "xent", "grads": rng.random() < 0.7, "B": B, "V": V, "d": d, "dtype": dtype, "normalize": normalize,
                "scale": 20.0 if normalize else 1.0, "ignored": rng.choice([0.0, 0.2])}
    if op == "clip":
        d = rng.randint(8, 256)
        tables = rng.randint(0, 5)
        return {"op": "clip", "tables": tables, "rows": _spread(rng, 16, 150000), "d": d, "vectors": rng.randint(1, 20),
                "matrices": rng.randint(0, 10), "dtype": dtype}
    d = _spread(rng, 8, 4096)
    return {"op": "norm", "n": _spread(rng, 1, min(500000, 500000 * 256 // d)), "d": d, "dtype": dtype}


def _shapes(case):
    d = case["d"]
    return [(case["rows"] + 7 * i, d) for i in range(case["tables"])] + [(d,)] * case["vectors"] + [(d, d)] * case["matrices"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "xent":
        B, V, d = case["B"], case["V"], case["d"]
        target = torch.randint(0, V, (B,), generator=g, device="cuda")
        if case["normalize"]:       # tables start at N(0, 1 / d); a partly trained query points near its target's row
            table = normal(V, d) / d
            near = table[target] / table[target].norm(dim=1, keepdim=True)
            q = 0.6 * near + 0.8 * normal(B, d) / math.sqrt(d)
        else:
            table = normal(V, d) / math.sqrt(d)
            q = 1.5 * normal(B, d) + 4.0 * table[target]
        if case["ignored"]:
            target = torch.where(torch.rand(B, generator=g, device="cuda") < case["ignored"], torch.full_like(target, -1), target)
        weight = (0.5 + torch.rand(B, generator=g, device="cuda")) / B      # loss weight of each query (a batch's mean, weighted)
        return {"case": case, "q": q.to(t), "table": table.to(t), "target": target.to(torch.int32), "weight": weight}
    if case["op"] == "clip":
        # a few heavy entries among small ones, as the rows a batch names; the threshold decays a little from pass to pass, so
        # that gradients which were clipped before are clipped again
        grads = [(normal(*s) * 0.02 * torch.exp(normal(s[0], *([1] * (len(s) - 1))))).to(t) for s in _shapes(case)]
        return {"case": case, "grads": grads, "max_norm": 1.0 if case["tables"] else 0.1}
    n, d = case["n"], case["d"]
    return {"case": case, "x": (normal(n, d) + 0.5).to(t), "dy": normal(n, d).to(t), "weight": 1.0 + 0.1 * normal(d), "bias": 0.1 * normal(d), "eps": 1e-5}


# -- the plain forms ------------------------------------------------------------------------------------------------------

def _plain_xent(s):
    c = s["case"]
    q, table, target = s["q"].float(), s["table"].float(), s["target"].long()
    length = table.square().sum(1, keepdim=True).sqrt() if c["normalize"] else None
    rows = table / length if c["normalize"] else table
    valid = target >= 0
    at = target.clamp(min=0).unsqueeze(1)
    logits = (q @ rows.t()) * c["scale"]
    top = logits.max(1, keepdim=True).values
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    loss = torch.where(valid, lse - logits.gather(1, at).squeeze(1), torch.zeros_like(lse))
    if not c["grads"]:
        return {"loss": loss, "lse": lse}
    w = torch.where(valid, s["weight"], torch.zeros_like(lse)).unsqueeze(1)
    p *= w / total
    p.scatter_add_(1, at, -w)
    p *= c["scale"]
    dq = p @ rows
    drows = p.t() @ q
    if c["normalize"]:
        drows = (drows - rows * (rows * drows).sum(1, keepdim=True)) / length
    return {"loss": loss, "lse": lse, "dq": dq.to(s["q"].dtype), "dtable": drows.to(s["table"].dtype)}


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g in s["grads"]:
        g.copy_(g.float() * coef)
    return {"norm": norm, "grads": s["grads"]}


def _plain_norm(s):
    x, dy, w, b = s["x"].float(), s["dy"].float(), s["weight"], s["bias"]
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + s["eps"])
    xhat = centred * rstd
    y = xhat * w + b
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def run(state):
    c = state["case"]
    if own:
        from graphqembed_amd import ops
        if c["op"] == "xent":
            if c["grads"]:
                loss, lse, dq, dtable = ops.softmax_xent_grads(state["q"], state["table"], state["target"], weight=state["weight"],
                                                               scale=c["scale"], normalize=c["normalize"])
                return {"loss": loss, "lse": lse, "dq": dq, "dtable": dtable}
            loss, lse = ops.softmax_xent_loss(state["q"], state["table"], state["target"], scale=c["scale"], normalize=c["normalize"])
            return {"loss": loss, "lse": lse}
        if c["op"] == "clip":
            norm = ops.clip_grad_norm_(state["grads"], state["max_norm"])
            state["max_norm"] *= 0.9999
            return {"norm": norm, "grads": state["grads"]}
        y, mean, rstd = ops.layer_norm_forward(state["x"], state["weight"], state["bias"], eps=state["eps"])
        dx, dweight, dbias = ops.layer_norm_backward(state["dy"], state["x"], mean, rstd, state["weight"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    if c["op"] == "xent":
        return _plain_xent(state)
    if c["op"] == "clip":
        out = _plain_clip(state)
        state["max_norm"] *= 0.9999
        return out
    return _plain_norm(state)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "xent":
        B, V, d = case["B"], case["V"], case["d"]
        moved = (B + V) * d * size + 12 * B
        if case["grads"]:       # logits, the queries' gradient and the table's: three products
            return {"bytes": 2 * (B + V) * d * size + 16 * B, "flops": 6.0 * B * V * d}
        return {"bytes": moved, "flops": 2.0 * B * V * d}
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": 3 * n * size, "flops": 3.0 * n}      # read for the norm; read and written to scale
    n, d = case["n"], case["d"]
    return {"bytes": 4 * n * d * size + 16 * d, "flops": 16.0 * n * d}      # x and dy read, y and dx written


# -- 64 bits ---------------------------------------------------------------------------------------------------------------

def _exact_xent(s):
    c = s["case"]
    B, V = c["B"], c["V"]
    Q = s["q"].double()
    W = s["table"].double()
    tgt = s["target"].long()
    keep = tgt >= 0
    unit = torch.nn.functional.normalize(W, dim=1, eps=0.0) if c["normalize"] else W
    lse = torch.empty(B, dtype=torch.float64, device="cuda")
    loss = torch.zeros(B, dtype=torch.float64, device="cuda")
    dQ = torch.zeros_like(Q)
    dU = torch.zeros_like(W)
    rows = max(1, min(B, int(2.5e8) // V))
    for b in range(0, B, rows):
        e = min(B, b + rows)
        z = c["scale"] * torch.mm(Q[b:e], unit.t())
        lse[b:e] = torch.logsumexp(z, 1)
        i = torch.nonzero(keep[b:e]).squeeze(1)
        loss[b + i] = lse[b + i] - z[i, tgt[b + i]]
        if c["grads"]:
            a = torch.exp(z - lse[b:e, None])
            a[i, tgt[b + i]] -= 1.0
            a *= (s["weight"][b:e].double() * keep[b:e])[:, None] * c["scale"]
            dQ[b:e] = torch.mm(a, unit)
            dU += torch.mm(a.t().contiguous(), Q[b:e])
        del z
    if not c["grads"]:
        return {"loss": loss, "lse": lse}
    if c["normalize"]:
        radial = torch.einsum("vd,vd->v", unit, dU)
        dU = (dU - unit * radial[:, None]) / torch.linalg.vector_norm(W, dim=1)[:, None]
    return {"loss": loss, "lse": lse, "dq": dQ, "dtable": dU}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "xent":
        return _exact_xent(s)
    if case["op"] == "clip":
        G = [g.double() for g in s["grads"]]
        norm = math.sqrt(math.fsum(float(torch.dot(g.reshape(-1), g.reshape(-1))) for g in G))
        c = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g * c for g in G]}
    X, D, w, b = s["x"].double(), s["dy"].double(), s["weight"].double(), s["bias"].double()
    var, mu = torch.var_mean(X, dim=1, correction=0)
    inv = 1.0 / torch.sqrt(var + s["eps"])
    H = (X - mu[:, None]) * inv[:, None]
    A = D * w
    dX = inv[:, None] * (A - (A.sum(1) / case["d"])[:, None] - H * ((A * H).sum(1) / case["d"])[:, None])
    return {"y": torch.addcmul(b, H, w), "dx": dX, "dweight": (D * H).sum(0), "dbias": D.sum(0)}
