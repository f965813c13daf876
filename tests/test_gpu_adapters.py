"""tsx_moe_adapters and its gradients against a 64-bit restatement, one adapter at a time."""
import numpy as np
import pytest
import torch

from tinystrata_amd import ops

from gpu_util import dev, host

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24  # half a step of fp32
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(n, rank, n_in, n_out, rows, order, dtype, seed=0, scaled=True):
    rng = np.random.default_rng(seed)
    f = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).cuda()
    a, b = f(n, rank, n_in).to(dtype), f(n, n_out, rank).to(dtype)
    scale = torch.from_numpy(rng.uniform(0.5, 2, n).astype(np.float32)).cuda() if scaled else None
    ids = rng.integers(0, max(n, 1), rows)
    if order == "segments":
        ids = np.sort(ids)
    elif order == "none":
        ids[:] = -1
    if order in ("some", "segments") and rows > 2:
        ids[::5] = [-1, n, -7, 1 << 30, -(1 << 31)][rows % 5]
    return dict(a=a, b=b, scale=scale, ids=torch.from_numpy(ids.astype(np.int32)).cuda(), x=f(rows, n_in),
                base=f(rows, n_out), dy=f(rows, n_out), dbase=f(rows, n_in))


def cpu64(c):
    d = {key: None if v is None else v.detach().cpu().double().numpy() for key, v in c.items()}
    d["ids"] = c["ids"].cpu().numpy().astype(np.int64)
    d["scale"] = d["scale"] if d["scale"] is not None else np.ones(len(d["a"]))
    return d


def forward_ref(c, with_base=True):
    d = cpu64(c)
    y = d["base"].copy() if with_base else np.zeros_like(d["base"])
    mag = np.abs(y)
    for a in range(len(d["a"])):
        j = np.flatnonzero(d["ids"] == a)
        y[j] += d["scale"][a] * (d["x"][j] @ d["a"][a].T) @ d["b"][a].T
        mag[j] += d["scale"][a] * (np.abs(d["x"][j]) @ np.abs(d["a"][a]).T) @ np.abs(d["b"][a]).T
    return y, mag


def backward_ref(c, with_base=True):
    d = cpu64(c)
    dx = d["dbase"].copy() if with_base else np.zeros_like(d["dbase"])
    da, db = np.zeros(d["a"].shape), np.zeros(d["b"].shape)
    m = [np.abs(dx), np.zeros_like(da), np.zeros_like(db)]
    for a in range(len(d["a"])):
        j = np.flatnonzero(d["ids"] == a)
        s, A, B, x, dy = d["scale"][a], d["a"][a], d["b"][a], d["x"][j], d["dy"][j]
        v, u, vm, um = s * dy @ B, s * x @ A.T, s * np.abs(dy) @ np.abs(B), s * np.abs(x) @ np.abs(A).T
        dx[j] += v @ A
        da[a], db[a] = v.T @ x, dy.T @ u
        m[0][j] += vm @ np.abs(A)
        m[1][a], m[2][a] = vm.T @ np.abs(x), np.abs(dy).T @ um
    return [dx, da, db], m


def tolerance(c):
    """A first product sums its columns in at least four waves' chains and adds those; the second sums ranks, or rows in
    eight waves' chains: each step of a chain rounds once, relative to the sum of magnitudes."""
    rank, n_in, n_out, rows = c["a"].shape[1], c["a"].shape[2], c["b"].shape[1], len(c["ids"])
    return (max(n_in, n_out) / 4 + max(rank, rows / 8) + 40) * STEP


def close(got, want, mag, tol):
    got = host(got).astype(np.float64)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol * mag + 1e-37).all(), (np.abs(got - want) / np.maximum(mag, 1e-37)).max()


def check(c, ad=None):
    ad = ad or ops.Adapters(c["a"], c["b"], c["scale"])
    tol = tolerance(c)
    y = torch.full_like(c["base"], float("nan"))
    ops.adapters(ad, c["ids"], c["x"], y, base=c["base"])
    close(y, *forward_ref(c), tol)
    same = c["base"].clone()
    ops.adapters(ad, c["ids"], c["x"], same, base=same)                  # in place
    assert torch.equal(same, y)
    n, rank = c["a"].shape[:2]
    nan = lambda *s: torch.full(s, float("nan"), device="cuda")
    dx, da, db = nan(*c["x"].shape), nan(*c["a"].shape), nan(*c["b"].shape)
    ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], dx=dx, da=da, db=db, dbase=c["dbase"])
    want, mag = backward_ref(c)
    for got, w, m in zip((dx, da, db), want, mag):
        close(got, w, m, tol)
    return y, dx, da, db


SIZES = [(1, 1, 1, 1), (3, 4, 4, 4), (2, 16, 64, 64), (3, 5, 100, 36), (5, 16, 256, 512), (2, 32, 512, 200), (4, 17, 333, 77),
         (2, 64, 2048, 128), (2, 100, 96, 1000), (2, 130, 128, 96), (2, 256, 64, 48), (2, 250, 70, 33), (40, 8, 128, 132)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,order", [(1, "some"), (17, "segments"), (131, "some")])
def test_adapters_sizes(size, dtype, rows, order):
    n, rank, n_in, n_out = size
    check(make(n, rank, n_in, n_out, rows, order, dtype, seed=rows + n_in))


@pytest.mark.parametrize("rows", [2, 15, 16, 33, 64, 257, 1025])
@pytest.mark.parametrize("order", ["some", "segments", "none"])
def test_adapters_rows(rows, order):
    check(make(6, 16, 128, 192, rows, order, torch.bfloat16, seed=rows, scaled=rows % 2 == 0))


def test_adapters_many_rows():
    """More rows than blocks that fill the card, one adapter with most of them."""
    c = make(3, 8, 64, 68, 9001, "segments", torch.float16, seed=5)
    c["ids"][:8000] = 1
    check(c)


@pytest.mark.parametrize("n,rows", [(4096, 70), (700, 5000), (300, 40), (2, 4097), (1, 4113)])
def test_adapters_regrouped(n, rows):
    """Mixed rows with many adapters, over the edges of the chunks that rows are regrouped in; a last chunk of one row."""
    check(make(n, 4, 16, 20, rows, "some", torch.bfloat16, seed=rows, scaled=n != 300))
    c = make(n, 4, 16, 20, rows, "segments", torch.float16, seed=n)
    c["ids"][rows // 2:] = c["ids"][rows // 2:].flip(0)
    check(c)


def test_no_rows_and_no_adapters():
    c = make(2, 8, 32, 16, 0, "some", torch.float32)
    ad = ops.Adapters(c["a"], c["b"], c["scale"])
    assert ops.adapters(ad, c["ids"], c["x"], torch.empty_like(c["base"]), base=c["base"]).shape == (0, 16)
    da, db = torch.full_like(c["a"], 3.0), torch.full_like(c["b"], 3.0)
    ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], da=da, db=db)
    assert (da == 0).all() and (db == 0).all()
    c = make(1, 8, 32, 16, 9, "some", torch.float32)
    none = ops.Adapters(c["a"][:0], c["b"][:0])
    y, dx = torch.full_like(c["base"], 3.0), torch.full_like(c["x"], 3.0)
    ops.adapters(none, c["ids"], c["x"], y, base=c["base"])
    assert torch.equal(y, c["base"])
    ops.adapters(none, c["ids"], c["x"], y)
    assert (y == 0).all()
    ops.adapters_backward(none, c["ids"], c["x"], c["dy"], dx=dx, dbase=c["dbase"])
    assert torch.equal(dx, c["dbase"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,shift", [(4, 0), (3, 0), (4, 1), (0, 2)])
def test_adapters_apart(dtype, pad, shift):
    """Rows and adapters further apart than their lengths and off the 16-byte boundary; what lies between is left alone."""
    n, rank, n_in, n_out, rows = 3, 12, 96, 40, 37
    c = make(n, rank, n_in, n_out, rows, "some", dtype, seed=pad + shift)

    def apart(t, fill=float("nan")):
        r, cols = t.shape[0], t[0].numel()
        buf = torch.full((r * (cols + pad) + shift + 4,), fill, dtype=t.dtype, device="cuda")
        view = buf.as_strided(tuple(t.shape), (cols + pad,) + tuple(t[0].stride()), shift)
        view.copy_(t)
        return buf, view

    ref = check(c)
    e = dict(c)
    for key in ("a", "b", "x", "base", "dy", "dbase"):
        e[key] = apart(c[key])[1]
    ad = ops.Adapters(e["a"], e["b"], e["scale"])
    ybuf, y = apart(torch.zeros_like(c["base"]), 7.0)
    xbuf, dx = apart(torch.zeros_like(c["x"]), 7.0)
    da, db = torch.empty_like(c["a"], dtype=torch.float32), torch.empty_like(c["b"], dtype=torch.float32)
    ops.adapters(ad, c["ids"], e["x"], y, base=e["base"])
    ops.adapters_backward(ad, c["ids"], e["x"], e["dy"], dx=dx, da=da, db=db, dbase=e["dbase"])
    tol = tolerance(c)
    close(y, *forward_ref(c), tol)
    for got, w, m in zip((dx, da, db), *backward_ref(c)):
        close(got, w, m, tol)
    for buf, view, t in ((ybuf, y, ref[0]), (xbuf, dx, ref[1])):
        between = torch.full_like(buf, 7.0)
        between.as_strided(tuple(view.shape), view.stride(), shift).copy_(view)
        assert torch.equal(buf, between)


def test_without_base_and_some_gradients():
    c = make(4, 24, 160, 96, 50, "some", torch.bfloat16, seed=2)
    ad, tol = ops.Adapters(c["a"], c["b"], c["scale"]), tolerance(c)
    y = torch.full_like(c["base"], float("nan"))
    ops.adapters(ad, c["ids"], c["x"], y)
    close(y, *forward_ref(c, False), tol)
    want, mag = backward_ref(c, False)
    scratch = torch.empty(ops.adapters_scratch_bytes(ad, 50), dtype=torch.uint8, device="cuda")
    full = None
    for mask in (7, 1, 2, 3, 4, 5, 6, 0):
        outs = [torch.full(s, float("nan"), device="cuda") if mask >> i & 1 else None
                for i, s in enumerate((c["x"].shape, c["a"].shape, c["b"].shape))]
        scratch.fill_(0xFF)                                              # nothing is taken from an earlier call
        ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], *outs, scratch=scratch)
        full = full or outs
        for got, f, w, m in zip(outs, full, want, mag):
            if got is not None:
                close(got, w, m, tol)
                assert torch.equal(got, f)


def test_values_stay_with_their_rows():
    """Infinities and NaN in an adapter no row names, and in the rows of others, reach no other row or adapter."""
    c = make(4, 16, 128, 64, 40, "mixed", torch.float32, seed=7)
    ids = c["ids"]
    ids[ids == 3] = 0
    c["a"][3], c["b"][3] = float("nan"), float("inf")
    bad = (ids == 1) | (torch.arange(40, device="cuda") == 5)
    ids[5] = -1
    ad = ops.Adapters(c["a"], c["b"], c["scale"])
    y0, (dx0, da0, db0) = torch.empty_like(c["base"]), [torch.empty_like(t, dtype=torch.float32) for t in (c["x"], c["a"], c["b"])]
    ops.adapters(ad, ids, c["x"], y0, base=c["base"])
    ops.adapters_backward(ad, ids, c["x"], c["dy"], dx0, da0, db0)
    x, dy = c["x"].clone(), c["dy"].clone()
    x[bad], dy[bad] = float("nan"), float("-inf")
    y, (dx, da, db) = torch.empty_like(y0), [torch.empty_like(t) for t in (dx0, da0, db0)]
    ops.adapters(ad, ids, x, y, base=c["base"])
    ops.adapters_backward(ad, ids, x, dy, dx, da, db)
    good = ~bad
    assert torch.isfinite(y0).all() and torch.isfinite(da0).all() and torch.isfinite(db0).all()
    assert torch.equal(y[good], y0[good]) and torch.equal(y[5], c["base"][5]) and torch.equal(dx[good], dx0[good])
    for i in (0, 2, 3):
        assert torch.equal(da[i], da0[i]) and torch.equal(db[i], db0[i])
    assert (da[3] == 0).all() and not torch.isfinite(y[ids == 1]).any()


def test_gradients_are_the_differences():
    """The restatement's gradients against central differences of sum(y * dy): y is linear in each of x, A and B."""
    c = make(2, 3, 6, 5, 4, "mixed", torch.float32, seed=1)
    (dx, da, db), _ = backward_ref(c, False)
    h = 2.0 ** -8
    for key, grad in (("x", dx), ("a", da), ("b", db)):
        flat = c[key].view(-1)
        for i in range(flat.numel()):
            kept = flat[i].item()
            vals = []
            for s in (h, -h):
                flat[i] = kept + s
                vals.append((forward_ref(c, False)[0] * c["dy"].cpu().double().numpy()).sum())
                step = flat[i].item()
                vals.append(step)
            flat[i] = kept
            diff = (vals[0] - vals[2]) / (vals[1] - vals[3])
            assert abs(diff - grad.ravel()[i]) < 1e-9 * max(1.0, abs(diff)) * 100
    check(c)


def test_adapters_graph_and_repeat():
    """Captured with the backward, replayed on other rows and ids beside eager work; the same bits every time."""
    cs = [make(5, 16, 256, 128, 70, o, torch.bfloat16, seed=9) for o in ("some", "segments", "mixed")]
    c = {key: None if v is None else v.clone() for key, v in cs[0].items()}
    ad = ops.Adapters(c["a"], c["b"], c["scale"])
    scratch = torch.empty(ops.adapters_scratch_bytes(ad, 70), dtype=torch.uint8, device="cuda")
    y, dx, da, db = (torch.empty_like(t, dtype=torch.float32) for t in (c["base"], c["x"], c["a"], c["b"]))

    def both(c, y, dx, da, db, scratch=None):
        ops.adapters(ad, c["ids"], c["x"], y, base=c["base"])
        ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], dx, da, db, dbase=c["dbase"], scratch=scratch)

    both(c, y, dx, da, db, scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(c, y, dx, da, db, scratch)
    for k in (0, 1, 2, 1, 0):
        for key in ("ids", "x", "base", "dy", "dbase"):
            c[key].copy_(cs[k][key])
        c["a"].mul_(0.5)                                                 # a training step between the replays
        graph.replay()
        out = [torch.empty_like(t) for t in (y, dx, da, db)]
        both(c, *out)
        assert all(torch.equal(p, q) for p, q in zip((y, dx, da, db), out)), k


@pytest.mark.parametrize("n,rank,rows", [(1, 5, 600), (1, 24, 4600), (2, 60, 1500), (1, 130, 1100), (3, 16, 1700)])
@pytest.mark.parametrize("vec", [True, False])
def test_adapters_shared_sums(n, rank, rows, vec):
    """Few adapters of many rows: blocks share an adapter's rows, for one gradient or both, with the same bits every time."""
    c = make(n, rank, 72 if vec else 70, 132 if vec else 131, rows, "some", torch.float32, seed=rows)
    ad = ops.Adapters(c["a"], c["b"], c["scale"])
    pad = next(q for q in (16, 32, 64, 128, 256) if q >= rank)
    assert ops.adapters_scratch_bytes(ad, rows) > 2 * (rows * pad * 4 + 256)  # more than u and v: the parts' sums
    (_, da, db), (_, ma, mb) = backward_ref(c)
    tol, seen = tolerance(c), {}
    for want_a, want_b in [(True, True), (True, False), (False, True), (True, True)]:
        ga = torch.full(ad.a.shape, 7.0, device="cuda") if want_a else None
        gb = torch.full(ad.b.shape, 7.0, device="cuda") if want_b else None
        ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], da=ga, db=gb)
        for name, g, want, mag in [("a", ga, da, ma), ("b", gb, db, mb)]:
            if g is not None:
                close(g, want, mag, tol)
                assert torch.equal(seen.setdefault(name, g.clone()), g)


@pytest.mark.parametrize("rows", [2, 3, 15, 17, 31, 48, 63, 64, 65])
@pytest.mark.parametrize("n", [1, 2, 17, 4096])
def test_adapters_decode_steps(rows, n):
    """Mixed rows of a decode step, few and many to an adapter, more than 16 of one among them."""
    c = make(n, 8, 40, 24, rows, "some", torch.bfloat16, seed=rows * 31 + n)
    check(c)
    c["ids"] = torch.where(torch.arange(rows, device="cuda") % 3 > 0, 0, c["ids"]).to(torch.int32)
    check(c)


def test_adapters_on_two_streams():
    """Two calls at once on streams of their own, their scratch from the allocator."""
    cs = [make(3, 16, 256, 320, 900, "some", torch.bfloat16, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for c, st in zip(cs, streams):
            ad = ops.Adapters(c["a"], c["b"], c["scale"])
            y, dx = torch.empty_like(c["base"]), torch.empty_like(c["x"])
            da, db = (torch.empty(t.shape, device="cuda") for t in (ad.a, ad.b))
            torch.cuda.synchronize()
            ops.adapters(ad, c["ids"], c["x"], y, base=c["base"], stream=st)
            ops.adapters_backward(ad, c["ids"], c["x"], c["dy"], dx=dx, da=da, db=db, dbase=c["dbase"], stream=st)
            outs.append((c, y, dx, da, db))
    torch.cuda.synchronize()
    for c, y, *grads in outs:
        want, mag = forward_ref(c)
        close(y, want, mag, tolerance(c))
        for got, want, mag in zip(grads, *backward_ref(c)):
            close(got, want, mag, tolerance(c))
