"""The row operators beside the engine, as timed cases: layer norm, routing to the nearest clusters, rows sorted by cluster
(dispatch) and back with weights (combine), forward and backward.

A k-means model routes the rows of a layer of experts: its distances are the scores, its clusters the experts.  Widths and
cluster counts come from the benchmark configurations (784 columns; 8, 100, 1000 clusters) or are generic powers of two and
odd sizes; rows go from one token to a long prompt's.

A case is a dict: ``kind`` (which operator and direction), ``rows``, ``cols``, ``k`` clusters, ``n`` chosen per row, ``dtype``
of the rows or scores, and what the kind needs besides: ``params`` (type of the norm's weight and bias), ``layout`` of the
scores ("rows": one row's scores side by side, as a linear router leaves them; "cols": one cluster's distances side by side,
as ``transform`` leaves them), ``over`` (which scores share the softmax), ``scale`` of the scores, ``align`` of the groups.
"""
import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5
HUGE = torch.finfo(torch.float32).max


def listed():
    return [
        # one new token in front of a router: latency
        dict(name="norm_token", kind="norm", rows=1, cols=4096, dtype="bfloat16", params="bfloat16"),
        # a long prompt, wide hidden states
        dict(name="norm_bulk", kind="norm", rows=16384, cols=4096, dtype="bfloat16", params="bfloat16"),
        # training on rows as wide as the image-like configuration, float32, an odd number of rows
        dict(name="norm_grad_784", kind="norm_grad", rows=30001, cols=784, dtype="float32", params="float32"),
        # a few tokens over eight experts: latency
        dict(name="route_few", kind="route", rows=5, k=8, n=2, dtype="float32", layout="rows", over="chosen", scale=1.0),
        # the distances that transform gives for 100 clusters, four nearest
        dict(name="route_distances", kind="route", rows=300_000, k=100, n=4, dtype="float32", layout="cols",
             over="chosen", scale=-0.05),
        # many clusters, scores of a linear router, softmax over all of them
        dict(name="route_wide", kind="route", rows=32768, k=1000, n=8, dtype="bfloat16", layout="rows", over="all",
             scale=1.0),
        # the router's gradient, softmax over all
        dict(name="route_grad", kind="route_grad", rows=65536, k=256, n=8, dtype="float32", layout="rows", over="all",
             scale=1.0),
        # a decoding batch: latency of sort and gather
        dict(name="dispatch_decode", kind="dispatch", rows=16, cols=1024, k=8, n=2, dtype="bfloat16", align=1),
        # a training batch: the largest
        dict(name="dispatch_bulk", kind="dispatch", rows=32768, cols=2048, k=64, n=4, dtype="bfloat16", align=128),
        # gradient of the sorted rows back to their tokens, rows that are not 16-byte aligned
        dict(name="dispatch_grad_odd", kind="dispatch_grad", rows=20011, cols=1021, k=100, n=2, dtype="float16", align=1),
        # a prompt's experts joined, eight each
        dict(name="combine_bulk", kind="combine", rows=16384, cols=2048, k=256, n=8, dtype="bfloat16", align=1),
        # its gradient in float32, groups on tile boundaries
        dict(name="combine_grad", kind="combine_grad", rows=15013, cols=784, k=100, n=3, dtype="float32", align=16),
    ]


def _spread(rng, lo, hi):
    """Log-uniform whole number of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "route", "route_grad", "dispatch", "dispatch_grad", "combine", "combine_grad"])
    c = dict(kind=kind, rows=_spread(rng, 1, 32768), dtype=rng.choice(sorted(DTYPES)))
    if kind.startswith("norm"):
        c.update(cols=_spread(rng, 16, 8192), params=rng.choice(["float32", c["dtype"]]))
        if rng.random() < 0.6:
            c["cols"] = max(16, c["cols"] // 16 * 16)
    elif kind.startswith("route"):
        c.update(k=_spread(rng, 2, 4096), layout=rng.choice(["rows", "cols"]), over=rng.choice(["chosen", "all"]))
        c.update(n=rng.randint(1, min(8, c["k"])), scale=-0.05 if c["layout"] == "cols" else 1.0)
    else:
        c.update(cols=_spread(rng, 16, 4096), k=_spread(rng, 2, 4096), align=rng.choice([1, 1, 16, 128]))
        c.update(n=rng.randint(1, min(8, c["k"])))
        if rng.random() < 0.6:
            c["cols"] = max(16, c["cols"] // 16 * 16)
        c["rows"] = min(c["rows"], max(1, int(2.5e8 / (c["cols"] * c["n"]))))
        if c["align"] > 1:      # padding of many clusters must not outweigh the rows
            c["k"] = min(c["k"], max(2, 4 * c["rows"] * c["n"] // c["align"]))
            c["n"] = min(c["n"], c["k"])
    largest = max(work(x)["bytes"] for x in listed())
    while work(c)["bytes"] > largest:
        c["rows"] = c["rows"] * 3 // 4
    return c


def _capacity(c):
    s = c["rows"] * c["n"]
    return s + min(c["k"], s) * (c["align"] - 1)


def work(case):
    c = case
    t = c["rows"]
    size = 4 if c["dtype"] == "float32" else 2
    kind = c["kind"]
    if kind.startswith("norm"):
        d = c["cols"]
        psize = 4 if c["params"] == "float32" else 2
        if kind == "norm":
            return {"bytes": 2 * t * d * size + 2 * d * psize + 8 * t, "flops": 8 * t * d}
        return {"bytes": 3 * t * d * size + d * psize + 8 * d + 8 * t, "flops": 14 * t * d}
    if kind.startswith("route"):
        k, n = c["k"], c["n"]
        if kind == "route":
            return {"bytes": t * k * size + 8 * t * n + 8 * t, "flops": (4 if c["over"] == "all" else 1) * t * k}
        reads = t * k * size + 8 * t if c["over"] == "all" else 0
        return {"bytes": reads + t * k * size + 12 * t * n, "flops": (6 if c["over"] == "all" else 1) * t * k}
    d, n = c["cols"], c["n"]
    s, cap = t * n, _capacity(c)
    if kind == "dispatch":
        return {"bytes": 4 * s + t * d * size + cap * d * size + 4 * s + 4 * cap + 8 * c["k"], "flops": s}
    if kind == "dispatch_grad":
        return {"bytes": s * d * size + 4 * s + t * d * size, "flops": s * d}
    if kind == "combine":
        return {"bytes": s * d * size + 8 * s + t * d * size, "flops": 2 * s * d}
    return {"bytes": t * d * size + s * d * size + cap * d * size + 12 * s, "flops": 3 * s * d}


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    t, kind = c["rows"], c["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = dict(case=c)
    if kind.startswith("norm"):
        d, pt = c["cols"], DTYPES[c["params"]]
        # hidden states: an offset, row lengths that differ, a few columns far larger than the rest
        x = normal(t, d) * torch.exp(0.5 * normal(t, 1)) + 0.3
        x[:, :: max(1, d // 7)] *= 8.0
        st["x"] = x.to(dt)
        st["weight"] = (1.0 + 0.1 * normal(d)).to(pt)
        st["bias"] = (0.1 * normal(d)).to(pt)
        if kind == "norm_grad":
            st["dy"] = (0.1 * normal(t, d)).to(dt)
            xd = st["x"].double()
            mean = xd.mean(1)
            st["mean"] = mean.float()
            st["rstd"] = ((xd - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
        return st
    if kind.startswith("route"):
        k, n = c["k"], c["n"]
        shape = (t, k) if c["layout"] == "rows" else (k, t)
        if c["scale"] > 0:
            s = 2.0 * normal(*shape)
        else:      # squared distances
            s = 40.0 + 80.0 * normal(*shape).square()
        # some clusters are closed to some rows, and padding rows have none open
        s[torch.rand(*shape, generator=gen, device="cuda") < 0.03] = float("-inf") if c["scale"] > 0 else float("inf")
        s = s.to(dt)
        s = s if c["layout"] == "rows" else s.t()
        if t > 8:
            s[t - t // 8:: 5] = float("-inf") if c["scale"] > 0 else float("inf")
        st["scores"] = s
        if kind == "route_grad":
            st["ids"], st["weights"], st["best"], st["total"] = _route(s, n, c["scale"], c["over"])
            st["dweights"] = normal(t, n)
        return st
    d, k, n = c["cols"], c["k"], c["n"]
    # uneven clusters; the last rows of the batch are padding and go nowhere
    ids = torch.multinomial(torch.softmax(normal(k), 0), t * n, replacement=True, generator=gen).to(torch.int32).view(t, n)
    ids[t - t // 50:] = -1
    st["ids"] = ids
    if kind == "dispatch":
        st["x"] = normal(t, d).to(dt)
        return st
    offsets, counts, slot, source = _sort(ids, k, c["align"])
    st.update(offsets=offsets, counts=counts, slot=slot, source=source)
    st["rows"] = normal(_capacity(c), d).to(dt)
    if kind != "dispatch_grad":
        st["weights"] = torch.softmax(normal(t, n), 1)
    if kind == "combine_grad":
        st["dy"] = normal(t, d).to(dt)
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _norm(x, weight, bias):
    xf = x.float()
    mean = xf.mean(1)
    xc = xf - mean[:, None]
    rstd = (xc.square().mean(1) + EPS).rsqrt()
    y = xc * rstd[:, None] * weight.float() + bias.float()
    return y.to(x.dtype), mean, rstd


def _norm_grad(dy, x, mean, rstd, weight):
    dyf = dy.float()
    xh = (x.float() - mean[:, None]) * rstd[:, None]
    g = dyf * weight.float()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx.to(x.dtype), (dyf * xh).sum(0), dyf.sum(0)


def _quality(scores, scale):
    """Scores with the better one larger, and -inf where a cluster cannot be chosen."""
    q = scores.float() * (1.0 if scale > 0 else -1.0)
    return torch.where(torch.isnan(q), torch.full_like(q, float("-inf")), q).clamp(max=HUGE)


def _route(scores, n, scale, over):
    q = _quality(scores, scale)
    top, idx = torch.sort(q, dim=1, descending=True, stable=True)
    top, idx = top[:, :n], idx[:, :n]
    open_ = top > float("-inf")
    best = torch.where(open_[:, 0], top[:, 0], torch.zeros_like(top[:, 0]))
    e = torch.where(open_, torch.exp(abs(scale) * (top - best[:, None])), torch.zeros_like(top))
    total = torch.exp(abs(scale) * (q - best[:, None])).sum(1) if over == "all" else e.sum(1)
    weights = torch.where(open_, e / total[:, None], torch.zeros_like(e))
    ids = torch.where(open_, idx, torch.full_like(idx, -1)).to(torch.int32)
    return ids, weights, best * (1.0 if scale > 0 else -1.0), total


def _route_grad(dweights, scores, ids, weights, best, total, scale, over):
    t, k = scores.shape
    at = torch.where(ids >= 0, ids, torch.full_like(ids, k)).long()
    g = torch.where(ids >= 0, dweights, torch.zeros_like(dweights))
    c = (weights * g).sum(1, keepdim=True)
    out = torch.zeros(t, k + 1, device=scores.device)
    if over == "chosen":
        return (scale * out.scatter_add_(1, at, weights * (g - c)))[:, :k].to(scores.dtype)
    q = _quality(scores, scale)
    sign = 1.0 if scale > 0 else -1.0
    p = torch.exp(abs(scale) * (q - sign * best[:, None])) / total[:, None]
    p = torch.where((q > float("-inf")) & (total[:, None] > 0), p, torch.zeros_like(p))
    return (scale * p * (out.scatter_add_(1, at, g)[:, :k] - c)).to(scores.dtype)


def _sort(ids, k, align):
    t, n = ids.shape
    flat = ids.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < k), flat, torch.full_like(flat, k))
    order = torch.argsort(flat, stable=True)
    group = flat[order]
    counts = torch.zeros(k + 1, dtype=torch.long, device=ids.device).index_add_(0, flat, torch.ones_like(flat))
    first = torch.cumsum(counts, 0) - counts
    padded = (counts[:k] + align - 1) // align * align
    offsets = torch.zeros(k + 1, dtype=torch.long, device=ids.device)
    offsets[1:] = torch.cumsum(padded, 0)
    place = offsets[group] + torch.arange(t * n, device=ids.device) - first[group]
    kept = group < k
    cap = t * n + min(k, t * n) * (align - 1)
    slot = torch.empty_like(flat)
    slot[order] = torch.where(kept, place, torch.full_like(place, -1))
    source = torch.full((cap + 1,), -1, dtype=torch.long, device=ids.device)
    source[torch.where(kept, place, torch.full_like(place, cap))] = order
    i32 = torch.int32
    return offsets.to(i32), counts[:k].to(i32), slot.to(i32).view(t, n), source[:cap].to(i32)


def _dispatch(x, source, n):
    rows = x[source.long().clamp(min=0) // n]
    return torch.where(source[:, None] >= 0, rows, torch.zeros_like(rows))


def _gathered(rows, slot):
    g = rows[slot.long().clamp(min=0)].float()
    return torch.where(slot[:, :, None] >= 0, g, torch.zeros_like(g))


def _combine(rows, slot, weights):
    g = _gathered(rows, slot)
    return (g if weights is None else g * weights[:, :, None]).sum(1).to(rows.dtype)


def _combine_grad(dy, rows, slot, weights):
    dyf = dy.float()
    dweights = (_gathered(rows, slot) * dyf[:, None, :]).sum(2)
    cap = rows.shape[0]
    drows = torch.zeros(cap + 1, rows.shape[1], dtype=rows.dtype, device=rows.device)
    at = torch.where(slot >= 0, slot, torch.full_like(slot, cap)).long()
    drows[at.reshape(-1)] = (weights[:, :, None] * dyf[:, None, :]).to(rows.dtype).reshape(-1, rows.shape[1])
    return drows[:cap], dweights


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    return _run_own(s, c, c["kind"]) if own else _run_plain(s, c, c["kind"])


def _run_own(s, c, kind):
    from h2o4gpu_b200 import rows
    if kind == "norm":
        return tuple(rows.layer_norm(s["x"], s["weight"], s["bias"], EPS))
    if kind == "norm_grad":
        return tuple(rows.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"]))
    if kind == "route":
        return tuple(rows.route(s["scores"], c["n"], c["scale"], c["over"]))
    if kind == "route_grad":
        routes = rows.Routes(s["ids"], s["weights"], s["best"], s["total"])
        return rows.route_grad(s["dweights"], s["scores"], routes, c["scale"], c["over"])
    if kind == "dispatch":
        plan = rows.sort_rows(s["ids"], c["k"], c["align"])
        return plan.offsets, plan.counts, plan.slot, plan.source, rows.dispatch(s["x"], plan)
    plan = rows.SortedRows(s["offsets"], s["counts"], s["slot"], s["source"])
    if kind == "dispatch_grad":
        return rows.dispatch_grad(s["rows"], plan)
    if kind == "combine":
        return rows.combine(s["rows"], plan, s["weights"])
    return tuple(rows.combine_grad(s["dy"], s["rows"], plan, s["weights"]))


def _run_plain(s, c, kind):
    if kind == "norm":
        return _norm(s["x"], s["weight"], s["bias"])
    if kind == "norm_grad":
        return _norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if kind == "route":
        return _route(s["scores"], c["n"], c["scale"], c["over"])
    if kind == "route_grad":
        return _route_grad(s["dweights"], s["scores"], s["ids"], s["weights"], s["best"], s["total"], c["scale"], c["over"])
    if kind == "dispatch":
        offsets, counts, slot, source = _sort(s["ids"], c["k"], c["align"])
        return offsets, counts, slot, source, _dispatch(s["x"], source, c["n"])
    if kind == "dispatch_grad":
        return _combine(s["rows"], s["slot"], None)
    if kind == "combine":
        return _combine(s["rows"], s["slot"], s["weights"])
    return _combine_grad(s["dy"], s["rows"], s["slot"], s["weights"])


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    f = {name: v.double() for name, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if kind == "norm":
        var, mean = torch.var_mean(f["x"], 1, correction=0)
        r = 1.0 / torch.sqrt(var + EPS)
        return torch.addcmul(f["bias"], (f["x"] - mean[:, None]) / torch.sqrt(var + EPS)[:, None], f["weight"]), mean, r
    if kind == "norm_grad":
        d = c["cols"]
        mu, r = f["mean"][:, None], f["rstd"][:, None]
        g = f["dy"] * f["weight"]
        along = torch.einsum("td,td->t", g, f["x"] - mu)[:, None]
        dx = r * g - r * (g.sum(1, keepdim=True) / d) - r ** 3 * (f["x"] - mu) * along / d
        return dx, torch.einsum("td,td->d", f["dy"], (f["x"] - mu) * r), torch.einsum("td->d", f["dy"])
    if kind == "route":
        if c["rows"] * c["k"] > 5e7:
            return None      # sorting on the host takes too long
        return _exact_route(f["scores"].cpu().numpy(), c)
    if kind == "route_grad":
        return _exact_route_grad(s, f, c)
    if kind == "dispatch":
        ids = s["ids"].cpu().numpy().reshape(-1)
        cap, k, n = _capacity(c), c["k"], c["n"]
        counts = np.bincount(ids[ids >= 0], minlength=k)
        ends = np.cumsum(-(-counts // c["align"]) * c["align"])
        starts = np.concatenate([[0], ends])
        order = np.argsort(ids, kind="stable")[int((ids < 0).sum()):]
        place = np.concatenate([np.arange(m) + b for m, b in zip(counts, starts)]) if order.size else order
        source, slot = np.full(cap, -1), np.full(ids.size, -1)
        source[place], slot[order] = order, place
        x = torch.cat([f["x"], torch.zeros_like(f["x"][:1])])
        at = torch.from_numpy(np.where(source >= 0, source // n, c["rows"])).cuda()
        return starts.astype(np.int32), counts.astype(np.int32), slot.reshape(-1, n).astype(np.int32), source.astype(np.int32), x[at]
    t, n, d = c["rows"], c["n"], c["cols"]
    full = torch.cat([f["rows"], torch.zeros_like(f["rows"][:1])])
    at = torch.where(s["slot"] < 0, f["rows"].shape[0], s["slot"]).long()
    w = f.get("weights", torch.ones(t, n, dtype=torch.float64, device="cuda"))
    if kind != "combine_grad":
        y = torch.zeros(t, d, dtype=torch.float64, device="cuda")
        for j in range(n):
            y.addcmul_(full[at[:, j]], w[:, j:j + 1])
        return y
    dw = torch.stack([torch.einsum("td,td->t", full[at[:, j]], f["dy"]) for j in range(n)], 1)
    src = s["source"].long()
    drows = f["dy"][src.clamp(min=0) // n] * (w.reshape(-1)[src.clamp(min=0)] * (src >= 0))[:, None]
    return drows, dw


def _exact_route(v, c):
    up = 1.0 if c["scale"] > 0 else -1.0
    v = v * up
    v[np.isnan(v)] = -np.inf
    v = np.minimum(v, float(HUGE))
    t, k, n = c["rows"], c["k"], c["n"]
    ids = np.argsort(-v, axis=1, kind="stable")[:, :n]
    top = np.take_along_axis(v, ids, 1)
    there = np.isfinite(top)
    best = np.where(there[:, 0], top[:, 0], 0.0)
    with np.errstate(invalid="ignore"):
        z = np.where(there, np.exp(abs(c["scale"]) * (top - best[:, None])), 0.0)
        total = np.exp(abs(c["scale"]) * (v - best[:, None])).sum(1) if c["over"] == "all" else z.sum(1)
    weights = np.divide(z, total[:, None], out=np.zeros_like(z), where=there)
    return np.where(there, ids, -1).astype(np.int32), weights, best * up, total


def _exact_route_grad(s, f, c):
    k, scale = c["k"], c["scale"]
    ids, w = s["ids"].long(), f["weights"]
    chosen = torch.nn.functional.one_hot(ids + 1, k + 1)[:, :, 1:].to(torch.float64)     # t x n x k
    g = torch.einsum("tn,tnk->tk", f["dweights"], chosen)
    mean = torch.einsum("tn,tn,tn->t", w, f["dweights"], (ids >= 0).double())[:, None]
    if c["over"] == "chosen":
        return scale * torch.einsum("tn,tnk->tk", w, chosen) * (g - mean)
    z = scale * (f["scores"] - f["best"][:, None])
    p = torch.where(torch.isfinite(z), torch.exp(z) / f["total"][:, None], 0.0)
    return torch.where(f["total"][:, None] > 0, scale * p * (g - mean), 0.0)
