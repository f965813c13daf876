"""tsx_moe_route, its gradient and the combine's: refusals, without a GPU."""
import ctypes as C

import pytest
import torch

from tinystrata_amd import _lib, ops


def router(**kw):
    a = dict(type=_lib.F32, score=1, n_expert=64, k=4, n_group=1, topk_group=1, group_top=1, norm=1, scale=1.0, floor=1e-5)
    a.update(kw)
    return _lib.RouterArgs(**a)


UNSUPPORTED = [dict(type=_lib.Q8_0), dict(n_expert=0), dict(n_expert=513), dict(k=0), dict(k=17), dict(n_expert=3, k=4),
               dict(n_group=0), dict(n_group=65, n_expert=130), dict(n_group=3), dict(n_group=4, topk_group=5),
               dict(n_group=4, topk_group=0), dict(n_group=4, group_top=3), dict(n_group=4, group_top=0),
               dict(n_group=64, topk_group=64, group_top=2), dict(n_group=16, topk_group=1, k=5)]
WRONG = [dict(score=2), dict(score=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(floor=0.0),
         dict(floor=-1.0), dict(floor=float("nan")), dict(bias=2)]


@pytest.mark.parametrize("kw,rc", [(a, _lib.TSX_ERR_UNSUPPORTED) for a in UNSUPPORTED] + [(a, _lib.TSX_ERR_ARG) for a in WRONG])
def test_router_refusals(kw, rc):
    lib, a = _lib.lib(), router(**kw)
    assert lib.tsx_moe_route(C.byref(a), 256, 512, 256, 256, None, None, 1, None) == rc
    assert b"tsx_moe_route" in lib.tsx_moe_last_error()
    assert lib.tsx_moe_route_backward(C.byref(a), 256, 512, 256, 256, 256, 512, 1, None) == rc


def test_route_buffers_refused():
    lib, a, e = _lib.lib(), router(), _lib.TSX_ERR_ARG
    good = [256, 64, 256, 256, None, None, 1, None]

    def call(i, v):
        args = list(good)
        args[i] = v
        return lib.tsx_moe_route(C.byref(a), *args)

    for i, v in [(0, None), (0, 258), (1, 63), (2, None), (2, 258), (3, None), (4, 258), (5, 258), (6, -1)]:
        assert call(i, v) == e, (i, v)
    assert lib.tsx_moe_route(None, *good) == e
    assert call(6, 0) == _lib.TSX_OK              # no tokens: nothing to do
    assert call(6, (1 << 29) + 1) == e            # entry numbers past 31 bits
    back = [256, 64, 256, 256, 256, 64, 1, None]
    for i, v in [(0, None), (1, 63), (2, None), (3, None), (4, None), (4, 257), (5, 63), (6, -1)]:
        args = list(back)
        args[i] = v
        assert lib.tsx_moe_route_backward(C.byref(a), *args) == e, (i, v)


def test_combine_backward_refused():
    lib, e = _lib.lib(), _lib.TSX_ERR_ARG
    good = [256, 256, None, 256, 8, 256, 256, 1, 64, 1, 256, 256, 256, 256, None]

    def call(**kw):
        args = list(good)
        for i, v in kw.items():
            args[int(i[1:])] = v
        return lib.tsx_moe_combine_backward(*args)

    for kw in [dict(a0=None), dict(a1=None), dict(a3=None), dict(a4=0), dict(a6=None), dict(a5=None), dict(a8=0), dict(a8=-1),
               dict(a9=-1), dict(a0=257), dict(a11=258), dict(a9=(1 << 31) - 1, a4=1 << 20)]:
        assert call(**kw) == e, kw
    assert call(a9=0) == _lib.TSX_OK


def test_python_refusals():
    f32, i32 = torch.float32, torch.int32
    with pytest.raises(ValueError, match="score"):
        ops.Router(64, 4, score="tanh")
    with pytest.raises(ValueError, match="bias"):
        ops.Router(64, 4, bias=torch.zeros(63))
    with pytest.raises(ValueError, match="bias"):
        ops.Router(64, 4, bias=torch.zeros(64, dtype=torch.float64))
    r, x = ops.Router(64, 4), torch.zeros(3, 64)
    for bad in (torch.zeros(64), torch.zeros(3, 63), torch.zeros(3, 64, dtype=torch.float64), torch.zeros(64, 3).t(),
                torch.zeros(1, 64).expand(3, 64)):
        with pytest.raises(ValueError):
            ops.route(r, bad)
    with pytest.raises(ValueError, match="ids"):
        ops.route(r, x, ids=torch.zeros(3, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="wts"):
        ops.route(r, x, wts=torch.zeros(3, 5))
    with pytest.raises(ValueError, match="counts"):
        ops.route(r, x, counts=torch.zeros(3, dtype=i32))
    with pytest.raises(ValueError, match="device"):
        ops.route(r, x)
    ids = torch.zeros(3, 4, dtype=i32)
    with pytest.raises(ValueError, match="dwts"):
        ops.route_backward(r, x, ids, torch.zeros(3, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="dlogits"):
        ops.route_backward(r, x, ids, torch.zeros(3, 4), dlogits=torch.zeros(3, 64, dtype=torch.float16))
    dy, parts, w = torch.zeros(3, 32), torch.zeros(12, 32), torch.zeros(3, 4)
    for kw, name in [(dict(parts=torch.zeros(11, 32)), "part rows"), (dict(parts=torch.zeros(12, 31)), "parts"),
                     (dict(wts=torch.zeros(3, 5)), "wts"), (dict(dparts=torch.zeros(11, 32)), "dparts"),
                     (dict(prow=torch.zeros(11, dtype=i32)), "prow"), (dict(shared=torch.zeros(2, 32)), "shared"),
                     (dict(shared=torch.zeros(3, 32), sgate=torch.zeros(2)), "sgate"),
                     (dict(dsgate=torch.zeros(4)), "dsgate"), (dict(dwts=torch.zeros(3, 4, dtype=torch.float16)), "dwts")]:
        args = dict(parts=parts, wts=w)
        args.update(kw)
        with pytest.raises(ValueError, match=name):
            ops.moe_combine_backward(dy, k=4, **args)


def test_overlaps_and_grids_refused():
    """The combine's gradient over its dy, and more threads than a launch counts."""
    lib, a, e = _lib.lib(), router(k=1), _lib.TSX_ERR_ARG
    for i, want in [(11, b"not overwritten"), (12, b"not overwritten")]:
        args = [256, 512, None, 256, 8, 1024, 256, 1, 64, 1, 256, 2048, 4096, 256, None]
        args[i] = 256
        assert lib.tsx_moe_combine_backward(*args) == e and want in lib.tsx_moe_last_error()
    args = [256, 512, None, 256, 8, 1024, 256, 1, 64, 1 << 30, 256, 2048, 4096, 256, None]
    assert lib.tsx_moe_combine_backward(*args) == e and b"too many rows" in lib.tsx_moe_last_error()
    assert lib.tsx_moe_route(C.byref(a), 256, 64, 256, 256, None, None, 1 << 26, None) == e
    assert b"2^26" in lib.tsx_moe_last_error()
    assert lib.tsx_moe_route_backward(C.byref(a), 256, 64, 256, 256, 256, 64, 1 << 28, None) == e
    assert b"2^28" in lib.tsx_moe_last_error()
