"""The operators around the expert products that are trained or that differ from request to request, as a user's program
calls them: routing by the rules of several model families, low-rank adapters of many requests beside a projection, and
the gradients of both over frozen expert weights.

  route              logits -> expert ids and weights (softmax or sigmoid scores, a bias for balance, expert groups)
  route_backward     the weights' gradient -> the logits'
  combine_backward   the layer output's gradient -> that of the routing weights, the expert rows, the shared expert
  adapters           y = base + scale B (A x), each row with the adapter of its request
  adapters_backward  the gradients of x, A and B

`own` false: plain torch operations, in 32 bits; the order of the experts, which 32 bits cannot always tell, in 64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
FLOOR = 6.103515625e-5  # the least sum that weights are divided by


def _router(name, op, tokens, experts, k, score, dtype="f32", bias=False, groups=1, top_groups=1, group_top=1, norm=True,
            scale=1.0, padded=0, removed=0, counts=False):
    c = dict(op=op, tokens=tokens, experts=experts, k=k, score=score, dtype=dtype, bias=bias, groups=groups,
             top_groups=top_groups, group_top=group_top, norm=norm, scale=scale, padded=padded, removed=removed,
             counts=counts)
    return {"name": name, **c} if name else c


def _combine(name, tokens, n, k, shared, sorted_rows):
    c = dict(op="combine_backward", tokens=tokens, n=n, k=k, shared=shared, sorted=sorted_rows)
    return {"name": name, **c} if name else c


def _adapters(name, op, rows, n_in, n_out, rank, adapters, used, dtype, order="segments", bare=0):
    """used: adapters that rows refer to; order: the rows of a request together, or mixed; bare: rows without an adapter."""
    c = dict(op=op, rows=rows, n_in=n_in, n_out=n_out, rank=rank, adapters=adapters, used=used, dtype=dtype, order=order,
             bare=bare)
    return {"name": name, **c} if name else c


def listed():
    v3 = dict(experts=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5)
    return [
        # one sequence decoding: one token by sigmoid scores, a balance bias and expert groups
        _router("route1_groups", "route", 1, **v3),
        # the ragged last chunk of a prompt on a model of few experts, half-precision logits, weights as they are
        _router("route777_softmax", "route", 777, 60, 4, "softmax", "bf16", norm=False),
        # a training batch with padding at its end, the experts' load counted for the bias
        _router("route16k_groups", "route", 16384, padded=300, counts=True, **v3),
        # the router's gradient on a short chunk: softmax with experts removed from the model
        _router("route_back512", "route_backward", 512, 128, 8, "softmax", removed=5),
        # the router's gradient of a training batch, half-precision logits
        _router("route_back16k", "route_backward", 16384, dtype="bf16", **v3),
        # the combine's gradient of a few tokens, rows in entry order
        _combine("combine_back4", 4, 2048, 8, shared=True, sorted_rows=False),
        # the combine's gradient of a training batch, rows sorted by expert
        _combine("combine_back4096", 4096, 2048, 8, shared=True, sorted_rows=True),
        # one request decoding through the shared expert's down projection
        _adapters("adapters1", "adapters", 1, 512, 2048, 16, 8, 1, "bf16"),
        # a serving batch of 60 requests with adapters of their own and four without, through a gate projection
        _adapters("adapters64_mixed", "adapters", 64, 2048, 512, 16, 64, 60, "f16", "mixed", bare=4),
        # the prompts of six requests in one chunk, a larger rank, through gate and up at once
        _adapters("adapters4096", "adapters", 4096, 2048, 1024, 64, 8, 6, "bf16", bare=100),
        # training on a short ragged batch: three adapters in 32 bits, a gate projection
        _adapters("adapters_back300", "adapters_backward", 300, 2048, 512, 32, 3, 3, "f32"),
        # training eight adapters of a down projection at once
        _adapters("adapters_back4096", "adapters_backward", 4096, 512, 2048, 16, 8, 8, "bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["route", "route", "route_backward", "combine_backward", "adapters", "adapters", "adapters_backward"])
    if op == "combine_backward":
        k, n = rng.choice([1, 2, 4, 6, 8, 10]), rng.choice([512, 1000, 1536, 2048, 2046, 4096])
        return _combine(None, log_int(1, 4096 * 8 * 2048 / (k * n)), n, k, rng.random() < 0.5, rng.random() < 0.5)
    if op in ("route", "route_backward"):
        groups = rng.choice([1, 1, 4, 8])
        experts = rng.choice([8, 16, 32, 64, 64]) * groups if groups > 1 else log_int(4, 512)
        experts = min(experts, 512)
        top_groups = rng.randint(1, groups)
        k = min(rng.choice([1, 2, 4, 6, 8, 8, 16]), top_groups * experts // groups)
        tokens = log_int(1, 16384 * 256 / experts if experts > 256 else 16384)
        # one expert's weight divided by itself has no gradient
        norm = rng.random() < 0.75 and (k > 1 or op == "route")
        return _router(None, op, tokens, experts, k, rng.choice(["softmax", "sigmoid"]), rng.choice(list(TORCH)),
                       rng.random() < 0.5, groups, top_groups, rng.choice([1, 2]), norm, rng.choice([1.0, 2.5]),
                       padded=rng.choice([0, tokens // 8]), removed=rng.choice([0, experts // 16]),
                       counts=op == "route" and rng.random() < 0.25)
    n_in, n_out = (rng.choice([256, 500, 512, 768, 1024, 1111, 2048, 2048]) for _ in range(2))
    rank = rng.choice([4, 8, 16, 16, 24, 32, 64, 100])
    most = 4096 * (2048 + 1024) * 64 / ((n_in + n_out) * rank)
    if op == "adapters_backward":
        most = min(most, 4096 * (512 + 2048) * 2 / (n_in + n_out))
    rows = log_int(1, min(8192, most))
    used = min(rows, log_int(1, 64 if op == "adapters" else 16))
    return _adapters(None, op, rows, n_in, n_out, rank, used + rng.randint(0, 8), used, rng.choice(list(TORCH)),
                     rng.choice(["segments", "segments", "mixed"]), bare=rng.choice([0, (rows - used) // 10]))


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device=DEV).normal_(0.0, std, generator=g)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] in ("route", "route_backward"):
        T, E = c["tokens"], c["experts"]
        # a model's router: a spread of its own per expert, shared by the tokens, and each token's own
        z = _normal(g, T, E) + 0.5 * _normal(g, E)
        if c["removed"]:
            z[:, torch.randperm(E, generator=g, device=DEV)[: c["removed"]]] = -math.inf
        if c["padded"]:
            z[T - c["padded"]:] = -math.inf
        s["logits"] = z.to(TORCH[c["dtype"]])
        s["bias"] = _normal(g, E, std=0.1) if c["bias"] else None
        if own:
            from tinystrata_amd import ops
            s["router"] = ops.Router(E, c["k"], score=c["score"], bias=s["bias"], n_group=c["groups"],
                                     topk_group=c["top_groups"], group_top=c["group_top"], norm=c["norm"],
                                     scale=c["scale"], floor=FLOOR)
        if c["op"] == "route":
            s["ids"] = torch.empty((T, c["k"]), dtype=torch.int32, device=DEV)
            s["wts"] = torch.empty((T, c["k"]), device=DEV)
        else:
            s["ids"] = _choice(c, s["logits"], s["bias"]).to(torch.int32)
            s["dwts"] = _normal(g, T, c["k"])
            s["dlogits"] = torch.empty_like(s["logits"])
    elif c["op"] == "combine_backward":
        T, n, k = c["tokens"], c["n"], c["k"]
        s["dy"], s["parts"] = _normal(g, T, n), _normal(g, T * k, n)
        w = torch.rand((T, k), generator=g, device=DEV)
        s["wts"] = w / w.sum(1, keepdim=True)
        s["prow"] = None
        if c["sorted"]:
            s["prow"] = torch.randperm(T * k, generator=g, device=DEV).to(torch.int32).view(T, k)
        s["shared"] = _normal(g, T, n) if c["shared"] else None
        s["sgate"] = _normal(g, T) if c["shared"] else None
        s["dparts"], s["dwts"] = torch.empty_like(s["parts"]), torch.empty_like(s["wts"])
        s["dshared"] = torch.empty_like(s["dy"]) if c["shared"] else None
        s["dsgate"] = torch.empty(T, device=DEV) if c["shared"] else None
    else:
        R, N, M, r, n = c["rows"], c["n_in"], c["n_out"], c["rank"], c["adapters"]
        t = TORCH[c["dtype"]]
        s["a"] = _normal(g, n, r, N, std=N ** -0.5).to(t)
        s["b"] = _normal(g, n, M, r, std=r ** -0.5).to(t)
        s["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device=DEV)
        # every used adapter once, the other rows' by chance; the rows of a request lie together unless mixed
        pick = torch.randperm(n, generator=g, device=DEV)[: c["used"]]
        ids = torch.cat([pick, pick[torch.randint(c["used"], (R,), generator=g, device=DEV)]])[: R - c["bare"]]
        ids = torch.cat([ids, torch.full((c["bare"],), -1, device=DEV)])
        ids = ids[torch.randperm(R, generator=g, device=DEV)]
        s["ids"] = (ids if c["order"] == "mixed" else torch.sort(ids).values).to(torch.int32)
        s["x"] = _normal(g, R, N)
        if own:
            from tinystrata_amd import ops
            s["ad"] = ops.Adapters(s["a"], s["b"], s["scale"])
        if c["op"] == "adapters":
            s["base"] = _normal(g, R, M)
            s["y"] = torch.empty((R, M), device=DEV)
        else:
            s["dy"] = _normal(g, R, M)
            s["dx"] = torch.empty((R, N), device=DEV)
            s["da"], s["db"] = torch.empty((n, r, N), device=DEV), torch.empty((n, M, r), device=DEV)
            if own:
                s["scratch"] = torch.empty(ops.adapters_scratch_bytes(s["ad"], R), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _scores(c, logits, dtype):
    """The experts' scores; an expert whose logit is -inf or NaN has none (0)."""
    z = logits.to(dtype)
    off = torch.isnan(z) | (z == -math.inf)
    z = torch.where(off, -math.inf, z)
    if c["score"] == "sigmoid":
        return torch.where(off, 0.0, 1.0 / (1.0 + torch.exp(-z))), off
    m = z.amax(1, keepdim=True)
    e = torch.where(off, 0.0, torch.exp(z - torch.where(m == -math.inf, 0.0, m)))
    return e / torch.where(m == -math.inf, 1.0, e.sum(1, keepdim=True)), off


def _choice(c, logits, bias):
    """The picked experts, int64 [tokens, k], -1 where none is left."""
    T, E, k, G = c["tokens"], c["experts"], c["k"], c["groups"]
    s, off = _scores(c, logits, torch.float64)
    sb = s + bias.double() if bias is not None else s
    key = torch.where(off, -math.inf, sb if bias is not None else logits.double())
    if G > 1:
        if c["group_top"] == 2:
            top = torch.sort(torch.where(off, -math.inf, sb).view(T, G, E // G), dim=2, descending=True).values[:, :, :2]
            gv = top[:, :, 0] + torch.where(top[:, :, 1] == -math.inf, 0.0, top[:, :, 1])
        else:
            gv = key.view(T, G, E // G).amax(2)
        best = torch.sort(gv, dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        keep = torch.zeros((T, G), dtype=torch.bool, device=logits.device).scatter_(1, best, True)
        key = torch.where(keep.repeat_interleave(E // G, dim=1), key, -math.inf)
    v, i = torch.sort(key, dim=1, descending=True, stable=True)
    return torch.where(v[:, :k] == -math.inf, -1, i[:, :k])


def _route(s):
    c = s["case"]
    ids = _choice(c, s["logits"], s["bias"])
    p, _ = _scores(c, s["logits"], torch.float32)
    w = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp(min=0)))
    if c["norm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=FLOOR)
    out = [ids.to(torch.int32), w * c["scale"]]
    if c["counts"]:
        one = torch.zeros(c["experts"], dtype=torch.int32, device=DEV)
        out.append(one.index_add(0, ids.clamp(min=0).view(-1), (ids >= 0).to(torch.int32).view(-1)))
    return out


def _route_backward(s):
    c = s["case"]
    ids = s["ids"].long()
    p, _ = _scores(c, s["logits"], torch.float32)
    at = ids.clamp(min=0)
    sel = torch.where(ids < 0, 0.0, p.gather(1, at))
    dw = torch.where(ids < 0, 0.0, s["dwts"])
    if c["norm"]:
        S = sel.sum(1, keepdim=True)
        mean = (dw * sel).sum(1, keepdim=True) / S.clamp(min=FLOOR)
        ds = c["scale"] / S.clamp(min=FLOOR) * torch.where(S > FLOOR, dw - mean, dw)
    else:
        ds = c["scale"] * dw
    ds = torch.where(ids < 0, 0.0, ds)
    dp = torch.zeros_like(p).scatter_add(1, at, ds)
    if c["score"] == "sigmoid":
        d = dp * p * (1.0 - p)
    else:
        d = p * (dp - (dp * p).sum(1, keepdim=True))
    return [d.to(s["logits"].dtype)]


def _combine_backward(s):
    c = s["case"]
    T, n, k = c["tokens"], c["n"], c["k"]
    rows = s["prow"].long().view(-1) if c["sorted"] else None
    parts = s["parts"][rows] if c["sorted"] else s["parts"]
    dw = (parts.view(T, k, n) * s["dy"][:, None]).sum(2)
    d = (s["wts"][:, :, None] * s["dy"][:, None]).view(T * k, n)
    out = [dw, torch.empty_like(d).index_copy_(0, rows, d) if c["sorted"] else d]
    if c["shared"]:
        g = 1.0 / (1.0 + torch.exp(-s["sgate"]))
        out += [g[:, None] * s["dy"], g * (1.0 - g) * (s["dy"] * s["shared"]).sum(1)]
    return out


def _low_rank(s):
    """Each row's A x, in the columns of its adapter among the columns of all adapters; the other columns are 0."""
    c = s["case"]
    n, r = c["adapters"], c["rank"]
    mine = (s["ids"][:, None] == torch.arange(n, device=DEV)).repeat_interleave(r, dim=1)
    a = s["a"].float().view(n * r, -1)
    return mine, a, torch.where(mine, s["x"] @ a.t(), 0.0)


def _all_b(s):
    """Every adapter's scaled B, [n_out, adapters * rank]."""
    n, r = s["case"]["adapters"], s["case"]["rank"]
    return (s["b"].float() * s["scale"][:, None, None]).permute(1, 0, 2).reshape(-1, n * r)


def _adapters_backward(s):
    c = s["case"]
    n, r = c["adapters"], c["rank"]
    mine, a, u = _low_rank(s)
    v = torch.where(mine, s["dy"] @ _all_b(s), 0.0)
    db = (s["dy"].t() @ u).view(-1, n, r).permute(1, 0, 2) * s["scale"][:, None, None]
    return [v @ a, (v.t() @ s["x"]).view(n, r, -1), db.contiguous()]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from tinystrata_amd import ops
        c = s["case"]
        if op == "route":
            counts = torch.zeros(c["experts"], dtype=torch.int32, device=DEV) if c["counts"] else None
            ops.route(s["router"], s["logits"], ids=s["ids"], wts=s["wts"], counts=counts)
            return [s["ids"], s["wts"]] + ([counts] if c["counts"] else [])
        if op == "route_backward":
            return [ops.route_backward(s["router"], s["logits"], s["ids"], s["dwts"], dlogits=s["dlogits"])]
        if op == "combine_backward":
            ops.moe_combine_backward(s["dy"], s["parts"], s["wts"], c["k"], prow=s["prow"], shared=s["shared"],
                                     sgate=s["sgate"], dwts=s["dwts"], dparts=s["dparts"], dshared=s["dshared"],
                                     dsgate=s["dsgate"])
            return [s["dwts"], s["dparts"]] + ([s["dshared"], s["dsgate"]] if c["shared"] else [])
        if op == "adapters":
            return [ops.adapters(s["ad"], s["ids"], s["x"], s["y"], base=s["base"])]
        ops.adapters_backward(s["ad"], s["ids"], s["x"], s["dy"], dx=s["dx"], da=s["da"], db=s["db"],
                              scratch=s["scratch"])
        return [s["dx"], s["da"], s["db"]]
    if op == "route":
        return _route(s)
    if op == "route_backward":
        return _route_backward(s)
    if op == "combine_backward":
        return _combine_backward(s)
    if op == "adapters":
        return [s["base"] + _low_rank(s)[2] @ _all_b(s).t()]
    return _adapters_backward(s)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] in ("route", "route_backward"):
        T, E, k, z = c["tokens"], c["experts"], c["k"], SIZE[c["dtype"]]
        if c["op"] == "route":
            return {"bytes": T * (E * z + 8 * k) + (4 * E if c["bias"] else 0) + (8 * E if c["counts"] else 0),
                    "flops": T * (4 * E + 4 * k)}
        # a sigmoid's gradient needs the picks' logits alone
        return {"bytes": T * ((k if c["score"] == "sigmoid" else E) * z + E * z + 8 * k), "flops": T * (4 * E + 8 * k)}
    if c["op"] == "combine_backward":
        T, n, k = c["tokens"], c["n"], c["k"]
        rows = 1 + 2 * k + (2 if c["shared"] else 0)
        return {"bytes": 4 * T * (n * rows + (3 if c["sorted"] else 2) * k + (2 if c["shared"] else 0)),
                "flops": 3 * T * n * (k + (1 if c["shared"] else 0))}
    R, N, M, r, n = c["rows"] - c["bare"], c["n_in"], c["n_out"], c["rank"], c["adapters"]
    weights = c["used"] * (N + M) * r * SIZE[c["dtype"]]
    if c["op"] == "adapters":
        return {"bytes": 4 * (R * N + 2 * c["rows"] * M + c["rows"]) + weights, "flops": 2 * R * r * (N + M)}
    return {"bytes": 4 * (R * (N + M) + c["rows"] * (N + 1) + n * (N + M) * r) + weights,
            "flops": 2 * R * r * (3 * N + 2 * M)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _np64(t):
    return None if t is None else t.detach().to("cpu", torch.float64).numpy()


def _exact_scores(c, z):
    with np.errstate(invalid="ignore", over="ignore"):
        live = ~(np.isnan(z) | np.isneginf(z))
        if c["score"] == "sigmoid":
            return np.where(live, 1.0 / (1.0 + np.exp(-z)), 0.0), live
        z = np.where(live, z, -np.inf)
        top = z.max(axis=1)
        e = np.exp(z - np.where(np.isneginf(top), 0.0, top)[:, None]) * live
        total = e.sum(axis=1)
        return e / np.where(total == 0.0, 1.0, total)[:, None], live


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "route":
        z, bias, k, G = _np64(s["logits"]), _np64(s["bias"]), c["k"], c["groups"]
        p, live = _exact_scores(c, z)
        T, E = z.shape
        pb = p if bias is None else p + bias
        order = z if bias is None else pb
        ok = live.copy()
        if G > 1:
            lists = np.where(live, pb if c["group_top"] == 2 else order, -np.inf).reshape(T, G, E // G)
            two = -np.sort(-lists, axis=2)[:, :, : c["group_top"]]
            value = np.where(np.isneginf(two[:, :, 0]), -np.inf, np.where(np.isneginf(two), 0.0, two).sum(axis=2))
            rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1, kind="stable")
            ok &= np.repeat(rank < c["top_groups"], E // G, axis=1)
        ids = np.lexsort((np.broadcast_to(np.arange(E), (T, E)), -np.where(ok, order, -np.inf)), axis=1)[:, :k]
        ids = np.where(np.take_along_axis(ok, ids, 1), ids, -1)
        w = np.where(ids < 0, 0.0, np.take_along_axis(p, np.maximum(ids, 0), 1))
        if c["norm"]:
            w = w / np.maximum(w.sum(axis=1, keepdims=True), FLOOR)
        out = [torch.from_numpy(ids.astype(np.int32)), torch.from_numpy(w * c["scale"])]
        if c["counts"]:
            out.append(torch.from_numpy(np.bincount(ids[ids >= 0], minlength=E).astype(np.int32)))
        return out
    if c["op"] == "route_backward":
        p, live = _exact_scores(c, _np64(s["logits"]))
        ids, dw = s["ids"].cpu().numpy().astype(np.int64), _np64(s["dwts"])
        T, k = ids.shape
        on = ids >= 0
        t = np.broadcast_to(np.arange(T)[:, None], (T, k))
        sel, dw = np.where(on, p[t, np.maximum(ids, 0)], 0.0), np.where(on, dw, 0.0)
        S = sel.sum(axis=1, keepdims=True)
        if c["norm"]:
            full = (dw * S - (dw * sel).sum(axis=1, keepdims=True)) / np.where(S > FLOOR, S, 1.0) ** 2
            ds = c["scale"] * np.where(S > FLOOR, full, dw / FLOOR)
        else:
            ds = c["scale"] * dw
        grad = np.zeros_like(p)
        np.add.at(grad, (t[on], ids[on]), ds[on])
        if c["score"] == "sigmoid":
            return [torch.from_numpy(grad * p * (1.0 - p))]
        return [torch.from_numpy(p * grad - p * (p * grad).sum(axis=1, keepdims=True))]
    d = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if c["op"] == "combine_backward":
        T, k, dy = c["tokens"], c["k"], d["dy"]
        row = (s["prow"].long() if c["sorted"] else torch.arange(T * k, device=DEV).view(T, k))
        dw, dparts = torch.empty_like(d["wts"]), torch.empty_like(d["parts"])
        for j in range(k):
            dw[:, j] = (d["parts"][row[:, j]] * dy).sum(1)
            dparts[row[:, j]] = d["wts"][:, j, None] * dy
        out = [dw, dparts]
        if c["shared"]:
            g = torch.sigmoid(d["sgate"])
            out += [dy * g[:, None], (dy * d["shared"]).sum(1) * g * torch.sigmoid(-d["sgate"])]
        return out
    ids = s["ids"].long()
    if c["op"] == "adapters":
        y = d["base"].clone()
        for a in range(c["adapters"]):
            j = torch.nonzero(ids == a).view(-1)
            y[j] += d["scale"][a] * ((d["x"][j] @ d["a"][a].t()) @ d["b"][a].t())
        return [y]
    dx, da, db = (torch.zeros(s[key].shape, dtype=torch.float64, device=DEV) for key in ("dx", "da", "db"))
    for a in range(c["adapters"]):
        j = torch.nonzero(ids == a).view(-1)
        x, dy = d["x"][j], d["dy"][j]
        v = d["scale"][a] * (dy @ d["b"][a])
        dx[j] = v @ d["a"][a]
        da[a] = v.t() @ x
        db[a] = d["scale"][a] * (dy.t() @ (x @ d["a"][a].t()))
    return [dx, da, db]
