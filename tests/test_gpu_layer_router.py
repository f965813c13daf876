"""A MoE layer with another routing rule, its requests' adapters on the shared expert, and the gradients behind the last
quantized product: routing, grouped experts, adapters and combine as they are used together (marked gpu).

The forward is held against the oracle's products in Q8_1 mode at the 1e-3 of the other layer tests: a code of h that two
sums of fp32 round apart (a few in 1e5 of them) moves a token's expert by about 1e-3 of it, the whole batch by a small part
of that.  The gradients are held against 64-bit ones of what the layer's own products left.
"""
import numpy as np
import pytest
import torch

import oracle as O
import router_ref as R
from tinystrata_amd import moe, ops
from tinystrata_amd._lib import Q4_K, Q8_0

from gpu_util import dev, experts, host, rel_l2

pytestmark = pytest.mark.gpu

N, FF, E, K, NAD, RANK = 512, 256, 16, 4, 3, 12
RULE = dict(score="sigmoid", n_group=4, topk_group=2, group_top=2)
WEIGHT = dict(score="sigmoid", scale=2.5)
STEP = 2.0 ** -24


def product(type_, w, n_in, n_out, row):
    return O.mmvq_q8_1(type_, w, n_in, n_out, O.quantize_q8_1(row[None].astype(np.float32)), 1)[0].astype(np.float64)


def expert(L, blob, row, adapt=lambda name, x, y: y):
    """down(silu(gate x) * up x) of one row with Q8_1 activations; adapt(name, x, y): y with its adapter."""
    g = adapt("gate", row, product(L.gu_type, blob[: L.up_off], N, FF, row))
    u = adapt("up", row, product(L.gu_type, blob[L.up_off: L.down_off], N, FF, row))
    h = g / (1.0 + np.exp(-g)) * u
    return adapt("down", h.astype(np.float32), product(L.d_type, blob[L.down_off: L.bytes], FF, N, h))


class Case:
    def __init__(self, gu, d, T, fused, dtype, adapted=True, seed=0):
        self.rng = rng = np.random.default_rng(100 * T + seed)
        self.T = T
        self.L, self.blobs, p = experts(gu, d, N, FF, E)
        order = (np.arange(E) * 5 + 3) % len(p)
        self.shared = p[-1]
        self.W = moe.weights_from_pool(self.L, dev(p), E, order, len(p) - 1)
        self.bias = rng.normal(0, 0.1, E).astype(np.float32)
        self.router = ops.Router(E, K, bias=dev(self.bias), scale=2.5, **RULE)
        self.ads = None
        if adapted:
            def mk(n_in, n_out):
                a = torch.from_numpy(rng.normal(0, n_in ** -0.5, (NAD, RANK, n_in)).astype(np.float32)).to("cuda", dtype)
                b = torch.from_numpy(rng.normal(0, 0.3, (NAD, n_out, RANK)).astype(np.float32)).to("cuda", dtype)
                return ops.Adapters(a, b, dev(rng.uniform(0.5, 2, NAD).astype(np.float32)))
            self.ads = moe.SharedAdapters(gate=mk(N, FF), up=mk(N, FF), down=mk(FF, N))
        self.layer = moe.MoELayer(self.W, K, T, torch.device("cuda"), fused=fused, router=self.router, adapters=self.ads,
                                  train=True)
        self.x, self.z, self.sg, self.y, self.dy = (torch.empty(s, device="cuda") for s in
                                                    ((T, N), (T, E), (T,), (T, N), (T, N)))
        self.ids = torch.empty(T, dtype=torch.int32, device="cuda") if adapted else None
        self.out = dict(dlogits=torch.empty(T, E, device="cuda"), dsgate=torch.empty(T, device="cuda"))
        if adapted:
            self.out.update(da=torch.empty(NAD, RANK, FF, device="cuda"), db=torch.empty(NAD, N, RANK, device="cuda"))
        self.fill()

    def fill(self):
        rng, T = self.rng, self.T
        z = rng.normal(0, 1, (T, E)).astype(np.float32)
        if T > 2:
            z[1, : E - 2] = -np.inf                                 # two experts left of four picks
            z[T - 1] = -np.inf                                      # none
        self.x.copy_(dev(rng.normal(0, 1, (T, N)).astype(np.float32)))
        self.z.copy_(dev(z))
        self.sg.copy_(dev(rng.normal(0, 1, T).astype(np.float32)))
        self.dy.copy_(dev(rng.normal(0, 1, (T, N)).astype(np.float32)))
        if self.ids is not None:
            self.ids.copy_(dev(rng.integers(-1, NAD + 1, T).astype(np.int32)))   # -1 and NAD: none
        for t in (self.layer.parts, self.layer.sh, self.layer.wts):
            t.fill_(float("nan"))                                   # nothing stale may be read

    def run(self):
        self.y.zero_()
        self.layer(self.x, self.z, self.sg, self.y, adapter_ids=self.ids)
        self.layer.backward(self.dy, self.z, self.sg, adapter_ids=self.ids, **self.out)

    def results(self):
        return {"y": host(self.y).copy(), **{n: host(t).copy() for n, t in self.out.items()}}


def matrices(ad, i):
    return (t[i].detach().to("cpu", torch.float64).numpy() for t in (ad.a, ad.b))


def check_forward(c):
    x, z, sg = host(c.x), host(c.z), host(c.sg).astype(np.float64)
    got, w = host(c.layer.ids), host(c.layer.wts)
    ids = None if c.ids is None else host(c.ids)
    want = np.zeros((c.T, N))
    for t in range(c.T):
        picks = R.pick(z[t].astype(np.float64), K, bias=c.bias.astype(np.float64), **RULE)
        assert (got[t] == picks).all()
        wt = R.weights(z[t].astype(np.float64), picks, **WEIGHT)
        assert np.allclose(w[t], wt, rtol=1e-5, atol=0)
        for e, we in zip(picks, wt):
            if e >= 0:
                want[t] += we * expert(c.L, c.blobs[e], x[t])

        def adapt(name, row, y):
            ad = None if ids is None or not 0 <= ids[t] < NAD else getattr(c.ads, name)
            if ad is None:
                return y
            a, b = matrices(ad, ids[t])
            return y + float(ad.scale[ids[t]]) * (b @ (a @ row.astype(np.float64)))
        want[t] += expert(c.L, c.shared, x[t], adapt) / (1.0 + np.exp(-sg[t]))
    assert rel_l2(host(c.y), want) < 1e-3
    if c.T > 2:
        assert (got[1] >= 0).sum() <= 2 and (got[c.T - 1] < 0).all()


def check_backward(c):
    """Against 64-bit sums over the layer's own products.  A sum of n terms in fp32 is within n 2^-24 of the terms' sizes."""
    dy, sg, z, ids = host(c.dy).astype(np.float64), host(c.sg).astype(np.float64), host(c.z), host(c.layer.ids)
    parts, sh, prow = (host(t).astype(np.float64) for t in (c.layer.parts, c.layer.sh, c.layer.prow.view(c.T, K)))
    prow = prow.astype(np.int64)
    got = c.results()
    s = 1.0 / (1.0 + np.exp(-sg))
    slope = s * (1.0 - s)
    size = (np.abs(dy) * np.abs(sh)).sum(1) * slope
    assert (np.abs(got["dsgate"] - (dy * sh).sum(1) * slope) <= (N + 80) * STEP * size).all()
    for t in range(c.T):
        rows = np.where(prow[t, :, None] >= 0, parts[np.maximum(prow[t], 0)], 0.0)
        assert ((prow[t] >= 0) == (ids[t] >= 0)).all()
        dw, dw_size = rows @ dy[t], np.abs(rows) @ np.abs(dy[t])
        want, size = R.gradient(z[t].astype(np.float64), ids[t], dw, **WEIGHT)
        _, moved = R.gradient(z[t].astype(np.float64), ids[t], (N + 8) * STEP * dw_size, **WEIGHT)
        assert (np.abs(got["dlogits"][t] - want) <= moved + R.rel_tolerance(z[t]) * size + 1e-37).all()
    if c.ads is None:
        return
    h, of = host(c.layer.sh_h).astype(np.float64), host(c.ids)
    for i in range(NAD):
        a, b = matrices(c.ads.down, i)
        scale, own = float(c.ads.down.scale[i]), of == i
        dsh = s[own, None] * dy[own]
        tol = (N + c.T + 40) * STEP
        da = scale * (dsh @ b).T @ h[own]
        assert (np.abs(got["da"][i] - da) <= tol * scale * (np.abs(dsh) @ np.abs(b)).T @ np.abs(h[own]) + 1e-37).all()
        db = scale * dsh.T @ (h[own] @ a.T)
        assert (np.abs(got["db"][i] - db) <= tol * scale * np.abs(dsh).T @ (np.abs(h[own]) @ np.abs(a).T) + 1e-37).all()


# tokens: one, a decode step, prompts short and longer (both prompt paths)
CASES = [(Q8_0, Q8_0, 1, True, torch.bfloat16), (Q4_K, Q8_0, 5, True, torch.float32), (Q8_0, Q8_0, 8, True, torch.float16),
         (Q4_K, Q4_K, 12, True, torch.bfloat16), (Q4_K, Q4_K, 12, False, torch.float16), (Q8_0, Q8_0, 130, True, torch.float32),
         (Q8_0, Q8_0, 130, False, torch.bfloat16)]


@pytest.mark.parametrize("gu,d,T,fused,dtype", CASES)
@pytest.mark.parametrize("adapted", [True, False])
def test_layer_with_router_and_adapters(gu, d, T, fused, dtype, adapted):
    c = Case(gu, d, T, fused, dtype, adapted)
    c.run()
    check_forward(c)
    check_backward(c)


@pytest.mark.parametrize("T", [5, 40])
def test_layer_forward_and_backward_in_a_graph(T):
    """Captured once, replayed for other inputs with eager work in between: the eager results, bit by bit."""
    c = Case(Q8_0, Q8_0, T, True, torch.bfloat16)
    c.run()                                                          # makes the second stream and loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for _ in range(3):
        c.fill()
        g.replay()
        replayed = c.results()
        for t in c.out.values():
            t.fill_(7.0)
        c.run()
        eager = c.results()
        for n in eager:
            assert (replayed[n] == eager[n]).all(), n
    check_forward(c)
    check_backward(c)


def test_plain_rule_is_the_layer_without_a_router():
    """Softmax, no bias, one group: the picks, weights and output of the layer's own routing (which takes experts by 64)."""
    c, n = Case(Q8_0, Q8_0, 6, True, torch.float32, adapted=False), 64
    _, _, p = experts(Q8_0, Q8_0, N, FF, n)
    W = moe.weights_from_pool(c.L, dev(p), n, (np.arange(n) * 5 + 3) % len(p), len(p) - 1)
    z = dev(np.random.default_rng(9).normal(0, 1, (6, n)).astype(np.float32))
    a = moe.MoELayer(W, K, 6, torch.device("cuda"), fused=False)
    b = moe.MoELayer(W, K, 6, torch.device("cuda"), router=ops.Router(n, K))
    ya, yb = torch.zeros(6, N, device="cuda"), torch.zeros(6, N, device="cuda")
    a(c.x, z, c.sg, ya)
    b(c.x, z, c.sg, yb)
    assert (host(a.ids) == host(b.ids)).all()
    assert np.allclose(host(a.wts), host(b.wts), rtol=1e-5, atol=0)
    assert rel_l2(host(yb), host(ya)) < 1e-5
