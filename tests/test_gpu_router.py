"""tsx_moe_route, tsx_moe_route_backward and tsx_moe_combine_backward against 64-bit restatements (router_ref.py)."""
import numpy as np
import pytest
import torch

from tinystrata_amd import ops

import router_ref as R
from gpu_util import dev, host

pytestmark = pytest.mark.gpu

INF = np.inf
NP = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}  # bits of the significand


def rows64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def check_route(logits, k, bias=None, counts=False, prow=False, router=None, **rule):
    """ids, weights (and counts, prow) of a device call against the restatement."""
    pickrule = {n: rule[n] for n in ("score", "n_group", "topk_group", "group_top") if n in rule}
    wrule = {n: rule[n] for n in ("score", "norm", "scale", "floor") if n in rule}
    T, E = logits.shape
    b = None if bias is None else dev(np.asarray(bias, np.float32))
    r = ops.Router(E, k, bias=b, **rule)
    ids = torch.full((T, k), 77, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), float("nan"), device="cuda")
    c = torch.full((E,), 5, dtype=torch.int32, device="cuda") if counts else None
    p = torch.full((T, k), 9, dtype=torch.int32, device="cuda") if prow else None
    ops.route(r, logits, ids=ids, wts=w, prow=p, counts=c)
    z = rows64(logits)
    got, gw = host(ids), host(w)
    b64 = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    for t in range(T):
        want = R.pick(z[t], k, bias=b64, **pickrule)
        assert (got[t] == want).all(), (t, got[t], want)
        ref = R.weights(z[t], want, **wrule)
        tol = R.rel_tolerance(z[t]) * np.abs(ref) + 1e-37
        assert (np.abs(gw[t] - ref) <= tol).all(), (t, gw[t], ref)
    if counts:
        assert (host(c) == 5 + np.bincount(got[got >= 0], minlength=E)).all()
    if prow:
        assert (host(p).ravel() == np.where(got.ravel() < 0, -1, np.arange(T * k))).all()
    return got, gw


# experts, k, groups, kept, by: one expert, as many picks as experts, odd sizes, groups of odd size and number, every lane
# layout (one group to 64), the largest
SHAPES = [(1, 1, 1, 1, 1), (5, 5, 1, 1, 1), (16, 16, 1, 1, 1), (60, 4, 1, 1, 1), (64, 6, 1, 1, 1), (127, 7, 1, 1, 1),
          (256, 8, 8, 4, 2), (256, 8, 8, 3, 1), (160, 6, 8, 3, 1), (257, 16, 1, 1, 1), (512, 16, 1, 1, 1),
          (512, 10, 4, 2, 2), (51, 9, 3, 1, 2), (500, 8, 5, 2, 2), (504, 12, 9, 4, 2), (510, 3, 17, 2, 1),
          (495, 16, 33, 20, 2), (512, 8, 64, 8, 2), (128, 2, 64, 64, 2), (64, 8, 64, 8, 1), (24, 8, 2, 2, 2)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_shapes(shape, score, bias):
    E, k, G, kept, by = shape
    rng = np.random.default_rng(E * 31 + k)
    logits = dev(rng.normal(0, 1.5, (21, E)).astype(np.float32))
    b = rng.normal(0, 0.1, E) if bias else None
    check_route(logits, k, b, score=score, n_group=G, topk_group=kept, group_top=by, counts=True, prow=True, scale=2.5)


@pytest.mark.parametrize("dtype", list(NP))
@pytest.mark.parametrize("T", [1, 2, 65, 1500])
def test_route_types_and_lengths(dtype, T):
    rng = np.random.default_rng(T)
    logits = dev(rng.normal(0, 1, (T, 96)).astype(np.float32)).to(dtype)
    check_route(logits, 6, np.zeros(96), score="sigmoid", norm=False, counts=True)   # zero biases: equal values are common
    check_route(logits, 6, score="softmax", n_group=4, topk_group=2, group_top=2)


@pytest.mark.parametrize("dtype", list(NP))
@pytest.mark.parametrize("pad,shift", [(3, 0), (4, 1), (4, 4), (0, 0)])
def test_route_rows_apart(dtype, pad, shift):
    """Rows further apart than the experts, and not on a 16-byte boundary."""
    rng = np.random.default_rng(pad + shift)
    T, E = 11, 64
    buf = dev(rng.normal(0, 1, (T, E + pad + 4)).astype(np.float32)).to(dtype)
    view = buf.as_strided((T, E), (E + pad, 1), shift)
    check_route(view, 8, rng.normal(0, 0.1, E), score="sigmoid", n_group=8, topk_group=4, group_top=2)
    r = ops.Router(E, 8, score="softmax")
    ids = dev(np.stack([rng.permutation(E)[:8] for _ in range(T)]).astype(np.int32))
    dw = dev(rng.normal(0, 1, (T, 8)).astype(np.float32))
    out = torch.full((T, E + pad + 4), 7.0, dtype=dtype, device="cuda")
    d = out.as_strided((T, E), (E + pad, 1), shift)
    ops.route_backward(r, view, ids, dw, dlogits=d)
    check_gradient(view, ids, dw, d, score="softmax")
    flat = torch.full_like(out, 7.0).view(-1)
    flat.as_strided((T, E), (E + pad, 1), shift).copy_(d)
    assert torch.equal(out.view(-1), flat)                        # what lies between the rows stays


def test_route_order_beyond_32_bits():
    """Choice values within 6e-8 of each other: their order is the 64-bit one (the smallest gap is over 3e-13)."""
    rng = np.random.default_rng(3)
    E, k = 64, 16
    z = rng.normal(0, 1, E).astype(np.float32)
    for score in ("sigmoid", "softmax"):
        s, _ = R.scores(z.astype(np.float64), score)
        bias = (1.25 - s).astype(np.float32)
        c = np.sort(s + bias.astype(np.float64))
        assert c[-1] - c[0] < 2e-7 and np.diff(c).min() > 3e-13
        got, _ = check_route(dev(z[None]), k, bias, score=score)
        by32 = np.argsort(-(s.astype(np.float32) + bias), kind="stable")[:k]
        assert (got[0] != by32).any()                              # 32 bits would pick otherwise
        check_route(dev(z[None]), 8, bias, score=score, n_group=8, topk_group=3, group_top=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 2, 2), (8, 2, 1)])
def test_route_masked(score, bias, groups):
    """Rows of nothing, of fewer experts than picks, NaN, the types' lowest values, infinities; biases of -inf and NaN."""
    rng = np.random.default_rng(9)
    E, k = 64, 8
    z = rng.normal(0, 1, (12, E)).astype(np.float32)
    z[0] = -INF
    z[1] = np.nan
    z[2, 3:] = -INF
    z[3, ::2] = np.nan
    z[4] = np.finfo(np.float32).min
    z[5, 8:] = np.finfo(np.float32).min
    z[6, [5, 40]] = INF
    z[7, :] = -INF
    z[7, 63] = 0.5
    z[8, 10:30] = -INF
    z[9] = 0.0
    z[10, 1::2] = -0.0
    z[10, ::2] = 0.0
    z[11] = -200.0 - np.arange(E)
    b = None
    if bias:
        b = rng.normal(0, 0.1, E)
        b[7], b[20] = -INF, np.nan
    G, kept, by = groups
    got, w = check_route(dev(z), k, b, score=score, n_group=G, topk_group=kept, group_top=by, counts=True, prow=True)
    assert (got[0] == -1).all() and (got[1] == -1).all() and (w[:2] == 0).all() and np.isfinite(w).all()
    for dtype in (torch.float16, torch.bfloat16):
        lows = torch.full((2, E), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        lows[1, 33] = -INF
        check_route(lows, k, b, score=score, n_group=G, topk_group=kept, group_top=by)


def check_gradient(logits, ids, dw, got, **rule):
    z, i, d, g = rows64(logits), host(ids).astype(np.int64), rows64(dw), rows64(got)
    bits = NP[got.dtype]
    tiny = {24: 1e-37, 11: 2.0 ** -25, 8: 1e-37}[bits]              # half of fp16's smallest step
    for t in range(len(z)):
        ref, mag = R.gradient(z[t], i[t].copy(), d[t], **rule)
        tol = R.rel_tolerance(z[t]) * mag + (2.0 ** -bits * np.abs(ref) if bits < 24 else 0.0) * (1 + 1e-3) + tiny
        assert (np.abs(g[t] - ref) <= tol).all(), (t, np.abs(g[t] - ref).max(), tol.min())


@pytest.mark.parametrize("E,k", [(1, 1), (5, 5), (60, 4), (64, 16), (127, 7), (256, 8), (512, 16), (300, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm,dtype", [(True, torch.float32), (False, torch.float32), (True, torch.float16),
                                        (True, torch.bfloat16)])
def test_route_backward(E, k, score, norm, dtype):
    rng = np.random.default_rng(E + k)
    for T in (1, 37):
        logits = dev(rng.normal(0, 1.5, (T, E)).astype(np.float32)).to(dtype)
        r = ops.Router(E, k, score=score, norm=norm, scale=1.5)
        ids, w = ops.route(r, logits)
        dw = dev(rng.normal(0, 1, (T, k)).astype(np.float32))
        d = torch.full_like(logits, float("nan"))
        ops.route_backward(r, logits, ids, dw, dlogits=d)
        check_gradient(logits, ids, dw, d, score=score, norm=norm, scale=1.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_route_backward_masked(score, norm):
    """Empty and thin rows, sums below the floor, NaN and infinities, ids out of range, an id named twice."""
    rng = np.random.default_rng(4)
    E, k = 48, 6
    z = rng.normal(0, 1, (9, E)).astype(np.float32)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(9)]).astype(np.int32)
    z[0] = -INF
    z[1, ids[1, 1:]] = -INF
    z[2, ids[2, 0]] = np.nan
    z[3] = -30.0 - rng.random(E)                                   # sigmoids near 1e-13: their sum is below the floor
    z[4, ids[4, 2]] = INF
    ids[5, 2] = -1
    ids[5, 3] = E
    ids[6] = 11
    ids[7, 1] = ids[7, 0]
    z[8, ids[8, :3]] = [90.0, 60.0, -90.0]
    logits, i, dw = dev(z), dev(ids), dev(rng.normal(0, 1, (9, k)).astype(np.float32))
    r = ops.Router(E, k, score=score, norm=norm)
    d = ops.route_backward(r, logits, i, dw, dlogits=torch.full_like(logits, float("nan")))
    g = host(d)
    assert np.isfinite(g).all() and (g[0] == 0).all()
    check_gradient(logits, i, dw, d, score=score, norm=norm)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_backward_is_the_difference(score):
    """The restatement's gradient (which the kernel is held to) against central differences of the weights."""
    rng = np.random.default_rng(8)
    E, k, h = 24, 4, 1e-5
    z, dw = rng.normal(0, 1, E), rng.normal(0, 1, k)
    for norm in (True, False):
        ids = R.pick(z, k, score)
        g, _ = R.gradient(z, ids, dw, score, norm, 1.7)
        for e in range(E):
            up, down = z.copy(), z.copy()
            up[e] += h
            down[e] -= h
            diff = (R.weights(up, ids, score, norm, 1.7) - R.weights(down, ids, score, norm, 1.7)) @ dw / (2 * h)
            assert abs(diff - g[e]) < 1e-8                          # h^2 times a third derivative of a few
        r = ops.Router(E, k, score=score, norm=norm, scale=1.7)
        d = ops.route_backward(r, dev(z[None].astype(np.float32)), dev(ids[None].astype(np.int32)),
                               dev(dw[None].astype(np.float32)))
        assert np.abs(host(d)[0] - g).max() < 1e-5                  # fp32 inputs: 2^-24 times sums of magnitude below 40


def combine_case(T, n, k, rows, seed):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.normal(0, 1, s).astype(np.float32)
    prow = rng.permutation(rows)[:T * k].astype(np.int32).reshape(T, k)
    return dict(dy=f(T, n), parts=f(rows, n), wts=f(T, k), prow=prow, shared=f(T, n), sgate=3 * f(T))


@pytest.mark.parametrize("T,n,k", [(1, 1, 1), (1, 2048, 8), (3, 77, 2), (5, 2046, 10), (130, 256, 17), (2, 4096, 1)])
@pytest.mark.parametrize("with_prow", [False, True])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_combine_backward(T, n, k, with_prow, shared, shift):
    rows = T * k + 3
    c = combine_case(T, n, k, rows, T * 100 + k)
    if with_prow and T * k > 2:
        c["prow"][0, 0] = -1
    def at(x):  # a copy `shift` floats off a 16-byte boundary
        buf = torch.empty(x.size + shift, device="cuda")
        buf[shift:].copy_(torch.from_numpy(x.ravel()))
        return buf[shift:].view(x.shape)
    dy, parts, sh = at(c["dy"]), at(c["parts"]), at(c["shared"])
    w, prow, sg = dev(c["wts"]), dev(c["prow"]), dev(c["sgate"])
    fill = lambda *s: torch.full(s, 3.0, device="cuda")
    dw, dp, ds, dg = fill(T, k), fill(rows, n), fill(T, n), fill(T)
    kw = dict(shared=sh, sgate=sg, dshared=ds, dsgate=dg) if shared else {}
    ops.moe_combine_backward(dy, parts, w, k, prow=prow if with_prow else None, dwts=dw, dparts=dp, **kw)
    row = c["prow"].astype(np.int64) if with_prow else np.arange(T * k).reshape(T, k)
    d64 = {key: v.astype(np.float64) for key, v in c.items()}
    # a lane sums n / 64 products in a chain, 64 lanes in a tree of six: each product and sum rounds to half a step
    tol = lambda mag: (n / 64 + 12) * 2.0 ** -24 * mag + 1e-37
    want_p = np.full((rows, n), 3.0)
    for t in range(T):
        for j in range(k):
            if row[t, j] < 0:
                assert host(dw)[t, j] == 0
                continue
            q = d64["parts"][row[t, j]]
            assert abs(host(dw)[t, j] - d64["dy"][t] @ q) <= tol(np.abs(d64["dy"][t]) @ np.abs(q))
            want_p[row[t, j]] = d64["wts"][t, j] * d64["dy"][t]
    assert (np.abs(host(dp) - want_p) <= 2.0 ** -24 * np.abs(want_p)).all()     # rows without an entry: as they were
    if shared:
        g = 1.0 / (1.0 + np.exp(-d64["sgate"]))
        assert (np.abs(host(ds) - g[:, None] * d64["dy"]) <= 8 * 2.0 ** -24 * np.abs(g[:, None] * d64["dy"])).all()
        dot, mag = (d64["dy"] * d64["shared"]).sum(1), np.abs(d64["dy"] * d64["shared"]).sum(1)
        ref = g * (1 - g) * dot
        assert (np.abs(host(dg) - ref) <= g * (1 - g) * tol(mag) + 8 * 2.0 ** -24 * np.abs(ref)).all()


def test_combine_backward_some_outputs():
    """Any subset of the outputs, the same bits as all of them; gates a stride apart."""
    T, n, k = 6, 512, 4
    c = {key: dev(v) for key, v in combine_case(T, n, k, T * k, 2).items()}
    gates = torch.randn((T, 3), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    gates[:, 1] = c["sgate"]
    outs = dict(dwts=(T, k), dparts=(T * k, n), dshared=(T, n), dsgate=(T,))
    full = {o: torch.zeros(s, device="cuda") for o, s in outs.items()}
    kw = dict(prow=c["prow"], shared=c["shared"], sgate=gates[:, 1], sg_stride=3)
    ops.moe_combine_backward(c["dy"], c["parts"], c["wts"], k, **kw, **full)
    for mask in range(16):
        some = {o: torch.zeros(s, device="cuda") for b, (o, s) in enumerate(outs.items()) if mask >> b & 1}
        ops.moe_combine_backward(c["dy"], c["parts"], c["wts"], k, **kw, **some)
        for o, v in some.items():
            assert torch.equal(v, full[o]), (mask, o)


@pytest.mark.parametrize("shift", [0, 1])   # four columns per thread, and the one-column forms
@pytest.mark.parametrize("norm", [False, True])
def test_combine_skips_entries_without_a_row(shift, norm):
    """A prow below 0 adds nothing, whatever row 0 holds; route_sort marks ids out of range so."""
    n = 256
    rng = np.random.default_rng(shift)
    T, k, E = 5, 4, 16
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[0, 1] = ids[2, 0] = ids[4, 3] = -1
    ids[3] = -1
    _, _, _, rinv, _ = ops.route_sort(dev(ids), k, E)
    prow = host(rinv).reshape(T, k)
    assert ((prow < 0) == (ids < 0)).all()
    parts = rng.normal(0, 1, (T * k, n)).astype(np.float32)
    prow = np.where(prow < 0, -1, prow + 1)                         # row 0 belongs to no entry
    parts[0] = INF
    w = rng.random((T, k)).astype(np.float32)
    x = rng.normal(0, 1, (T, n)).astype(np.float32)
    ref = x.astype(np.float64)
    for t in range(T):
        for j in range(k):
            if prow[t, j] >= 0:
                ref[t] += w[t, j].astype(np.float64) * parts[prow[t, j]]
    y = torch.empty(T * n + shift, device="cuda")[shift:].view(T, n)
    y.copy_(dev(x))
    pr = dev(prow.astype(np.int32))
    if norm:
        h = torch.empty((T, n), device="cuda")
        ops.moe_combine_norm(y, dev(parts), dev(w), k, torch.ones(n, device="cuda"), 1e-6, h, prow=pr)
        assert np.isfinite(host(h)).all()
    else:
        ops.moe_combine(y, dev(parts), dev(w), k, prow=pr)
    assert np.abs(host(y) - ref).max() <= (k + 2) * 2.0 ** -24 * 40  # sums of magnitude below 40


def test_no_tokens():
    r = ops.Router(32, 4)
    z = torch.empty((0, 32), device="cuda")
    ids, w = ops.route(r, z)
    assert ids.shape == (0, 4) and w.shape == (0, 4)
    assert ops.route_backward(r, z, ids, w).shape == (0, 32)
    ops.moe_combine_backward(z, z, w, 4, dwts=w)


def test_route_graph_and_stream():
    """Captured once and replayed on other logits beside eager work; counts add up; another stream than the current one."""
    rng = np.random.default_rng(1)
    T, E, k = 33, 96, 6
    bias = dev(rng.normal(0, 0.1, E).astype(np.float32))
    r = ops.Router(E, k, score="sigmoid", bias=bias, n_group=6, topk_group=3, group_top=2)
    z = [dev(rng.normal(0, 1, (T, E)).astype(np.float32)) for _ in range(4)]
    logits, dw = z[0].clone(), dev(rng.normal(0, 1, (T, k)).astype(np.float32))
    ids, w = ops.route(r, logits)
    counts, d = torch.zeros(E, dtype=torch.int32, device="cuda"), torch.empty_like(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.route(r, logits, ids=ids, wts=w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.route(r, logits, ids=ids, wts=w, counts=counts)
        ops.route_backward(r, logits, ids, dw, dlogits=d)
    total = np.zeros(E, np.int64)
    for x in z + z[:2]:
        logits.copy_(x)
        bias.add_(0.01 * torch.sign(x.mean(0)))                      # a balance step between the replays
        graph.replay()
        eids, ew = ops.route(r, x)
        ed = ops.route_backward(r, x, eids, dw)
        assert torch.equal(ids, eids) and torch.equal(w, ew) and torch.equal(d, ed)
        total += np.bincount(host(eids).ravel(), minlength=E)
        assert (host(counts) == total).all()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        a = ops.route(r, z[3], stream=torch.cuda.current_stream())
    side.synchronize()
    b = ops.route(r, z[3])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("E,k,seed", [(96, 6, 0), (256, 8, 0), (320, 16, 1)])
@pytest.mark.parametrize("T", [1, 2050])
@pytest.mark.parametrize("groups", [1, 8])
def test_route_many_values_beyond_32_bits(E, k, seed, T, groups):
    """Two thirds of the experts within 6e-8 of each other (the smallest gap is over 4e-13), among ordinary rows or alone; with
    groups, those of a group, the groups well apart."""
    rng = np.random.default_rng(seed)
    z = rng.normal(0, 1, E).astype(np.float32)
    s, _ = R.scores(z.astype(np.float64), "sigmoid")
    bias = (1.25 - s).astype(np.float32)
    bias[::3] -= np.float32(0.5)
    c = np.sort((s + bias.astype(np.float64))[np.arange(E) % 3 > 0])
    assert c[-1] - c[0] < 2e-7 and np.diff(c).min() > 4e-13
    rows = rng.normal(0, 1, (T, E)).astype(np.float32)
    rows[0] = rows[T // 2] = rows[T - 1] = z
    rule = dict(score="sigmoid")
    if groups > 1:
        # a step of 2^-3 between groups: exact in the bias, so the gaps within a group stay
        step = (np.float32(2) ** -3 * (np.arange(E) // (E // groups))).astype(np.float32)
        shifted = (bias + step).astype(np.float32)
        c = s + shifted.astype(np.float64)
        for g in range(groups):
            own = np.sort(c[g * E // groups:(g + 1) * E // groups])
            assert np.diff(own).min() > 3e-13
        bias, rule = shifted, dict(score="sigmoid", n_group=groups, topk_group=4, group_top=2)
    check_route(dev(rows), k, bias, counts=True, prow=True, **rule)
