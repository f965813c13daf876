"""tsx_moe_adapters and its gradients: refusals, without a GPU."""
import ctypes as C

import pytest
import torch

from tinystrata_amd import _lib, ops


def args(**kw):
    a = dict(type=_lib.BF16, n=4, rank=16, n_in=64, n_out=32, a=256, b=256, a_stride=1024, b_stride=512, scale=256)
    a.update(kw)
    return _lib.AdapterArgs(**a)


FORWARD = [256, 256, 64, 256, 32, 1024, 32, 3, None]
BACKWARD = [256, 256, 64, 256, 32, 256, 64, 1024, 64, 256, 256, 3, 256, None]


@pytest.mark.parametrize("kw,rc", [(dict(type=_lib.Q8_0), -1), (dict(rank=0), -1), (dict(rank=257), -1), (dict(n_in=0), -1),
                                   (dict(n_out=0), -1), (dict(n_in=(1 << 24) + 1), -1), (dict(n=4097), -1), (dict(n=-1), -2), (dict(a=None), -2),
                                   (dict(b=None), -2), (dict(a=257), -2), (dict(b=257), -2), (dict(a_stride=1023), -2),
                                   (dict(b_stride=511), -2), (dict(scale=258), -2), (dict(type=_lib.F32, a=258), -2)])
def test_adapters_refused(kw, rc):
    lib, a = _lib.lib(), args(**kw)
    assert lib.tsx_moe_adapters(C.byref(a), *FORWARD) == rc
    assert b"tsx_moe_adapters" in lib.tsx_moe_last_error()
    assert lib.tsx_moe_adapters_backward(C.byref(a), *BACKWARD) == rc


def test_adapters_buffers_refused():
    lib, a = _lib.lib(), args()
    for i, v in [(0, None), (1, None), (5, None), (0, 258), (1, 258), (3, 258), (5, 258), (2, 63), (4, 31), (6, 31), (7, -1),
                 (7, 1 << 31)]:
        b = list(FORWARD)
        b[i] = v
        assert lib.tsx_moe_adapters(C.byref(a), *b) == _lib.TSX_ERR_ARG, (i, v)
    inplace = list(FORWARD)
    inplace[3], inplace[5], inplace[6] = 256, 256, 36
    assert lib.tsx_moe_adapters(C.byref(a), *inplace) == _lib.TSX_ERR_ARG     # base is y, at another distance
    empty = list(FORWARD)
    empty[7] = 0
    assert lib.tsx_moe_adapters(C.byref(a), *empty) == _lib.TSX_OK
    assert lib.tsx_moe_adapters(None, *FORWARD) == _lib.TSX_ERR_ARG
    for i, v in [(0, None), (1, None), (3, None), (12, None), (12, 128), (1, 258), (3, 258), (5, 258), (7, 258), (9, 258),
                 (10, 258), (2, 63), (4, 31), (6, 63), (8, 63), (11, -1)]:
        b = list(BACKWARD)
        b[i] = v
        assert lib.tsx_moe_adapters_backward(C.byref(a), *b) == _lib.TSX_ERR_ARG, (i, v)


def test_scratch_bytes():
    lib = _lib.lib()
    up = lambda v: (v + 255) // 256 * 256
    for rows, rank, pad in [(0, 16, 16), (5, 3, 16), (100, 33, 64), (4096, 100, 128), (7, 200, 256)]:
        a = args(rank=rank)
        uv, sums = 2 * up(rows * pad * 4), a.n * rank * (a.n_in + a.n_out) * 4     # and the sums of up to 16 parts of the rows
        need = lib.tsx_moe_adapters_scratch_bytes(C.byref(a), rows)
        assert need == uv or (need - uv) % sums == 0 and 2 <= (need - uv) // sums <= 16
    assert lib.tsx_moe_adapters_scratch_bytes(None, 5) == 0
    assert lib.tsx_moe_adapters_scratch_bytes(C.byref(args()), -1) == 0


def test_python_refusals():
    a, b = torch.zeros(2, 8, 32), torch.zeros(2, 16, 8)
    for bad in [(a[0], b), (a, b[:1]), (a, b.half()), (a.double(), b.double()), (a.transpose(1, 2), b), (a, torch.zeros(2, 16, 9)),
                (a, b, torch.zeros(3)), (a, b, torch.zeros(2).half())]:
        with pytest.raises(ValueError):
            ops.Adapters(*bad)
    ad = ops.Adapters(a, b)
    ids, x, y = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 32), torch.zeros(3, 16)
    for bad in [(ids.long(), x, y), (ids, x[:2], y), (ids, x.half(), y), (ids, x, y[:, :15]), (ids, torch.zeros(32, 3).t(), y),
                (ids, x, torch.zeros(1, 16).expand(3, 16))]:
        with pytest.raises(ValueError):
            ops.adapters(ad, *bad)
    with pytest.raises(ValueError, match="base"):
        ops.adapters(ad, ids, x, y, base=torch.zeros(3, 15))
    with pytest.raises(ValueError, match="device"):
        ops.adapters(ad, ids, x, y)
    for kw in [dict(dx=torch.zeros(3, 31)), dict(da=torch.zeros(2, 8, 32).half()), dict(db=torch.zeros(2, 8, 16)),
               dict(dbase=torch.zeros(2, 32)), dict(scratch=torch.zeros(8, dtype=torch.uint8))]:
        with pytest.raises(ValueError, match=next(iter(kw))):
            ops.adapters_backward(ad, ids, x, y, **kw)


def test_overlaps_and_grids_refused():
    """Outputs in place of what other blocks read, and more threads than a launch counts."""
    lib, a = _lib.lib(), args(n_in=32, n_out=32, a_stride=512)
    for fn, good, changes in [(lib.tsx_moe_adapters, FORWARD, dict(x=(1, 1024), rows=(7, (1 << 31) - 1))),
                              (lib.tsx_moe_adapters_backward, BACKWARD, dict(x=(1, 1024), dy=(3, 1024), rows=(11, 1 << 30)))]:
        for name, (i, v) in changes.items():
            b = list(good)
            b[i] = v
            assert fn(C.byref(a), *b) == _lib.TSX_ERR_ARG, name
            said = lib.tsx_moe_last_error()
            assert (b"too many rows" if name == "rows" else b"other blocks") in said, (name, said)
