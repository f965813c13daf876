"""What MoELayer refuses of a router and of adapters, without a GPU (its buffers are plain tensors)."""
import numpy as np
import pytest
import torch

from tinystrata_amd import moe, ops
from tinystrata_amd._lib import Q8_0

N, FF, E, K = 256, 128, 8, 2


def weights(shared=True):
    L = ops.native_expert_layout(Q8_0, Q8_0, N, FF)
    stride = moe.blob_stride(L)
    return moe.MoEWeights(L=L, n_expert=E, stride=stride, blobs=torch.zeros(E * stride, dtype=torch.uint8),
                          shared=torch.zeros(stride, dtype=torch.uint8) if shared else None)


def layer(n_tok=4, shared=True, **kw):
    return moe.MoELayer(weights(shared), K, n_tok, torch.device("cpu"), **kw)


def adapters(n_in, n_out, n=2, rank=4):
    return ops.Adapters(torch.zeros(n, rank, n_in), torch.zeros(n, n_out, rank))


def test_router_and_adapters_fit_the_layer():
    good = moe.SharedAdapters(gate=adapters(N, FF), up=adapters(N, FF), down=adapters(FF, N))
    for n_tok in (4, 40):
        assert not layer(n_tok, router=ops.Router(E, K), adapters=good, train=True).fused
    assert layer().fused                                              # neither: the two-launch layer as before
    for router in (ops.Router(E + 1, K), ops.Router(E, K + 1)):
        with pytest.raises(ValueError, match="router of"):
            layer(router=router)
    for bad in (dict(gate=adapters(FF, N)), dict(up=adapters(N, N)), dict(down=adapters(N, FF))):
        with pytest.raises(ValueError, match="adapters of " + next(iter(bad))):
            layer(adapters=moe.SharedAdapters(**bad))
    with pytest.raises(ValueError, match="without a shared expert"):
        layer(shared=False, adapters=good)
    with pytest.raises(ValueError, match="train with a router"):
        layer(train=True)


def test_calls_that_do_not_fit():
    x, z = torch.zeros(4, N), torch.zeros(4, E)
    ids = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="adapter_ids with adapters"):
        layer(router=ops.Router(E, K))(x, z, torch.zeros(4), x, adapter_ids=ids)
    with_down = moe.SharedAdapters(down=adapters(FF, N))
    with pytest.raises(ValueError, match="adapter_ids with adapters"):
        layer(adapters=with_down)(x, z, torch.zeros(4), x)
    with pytest.raises(ValueError, match="without train"):
        layer(router=ops.Router(E, K)).backward(x, z)
    train = layer(router=ops.Router(E, K), train=True)
    with pytest.raises(ValueError, match="da, db without"):
        train.backward(x, z, torch.zeros(4), da=torch.zeros(2, 4, FF))
    with pytest.raises(ValueError, match="da, db without"):
        layer(router=ops.Router(E, K), adapters=moe.SharedAdapters(gate=adapters(N, FF)), train=True).backward(
            x, z, torch.zeros(4), adapter_ids=ids, db=torch.zeros(2, N, 4))
    with pytest.raises(ValueError, match="dsgate without"):
        layer(shared=False, router=ops.Router(E, K), train=True).backward(x, z, dsgate=torch.zeros(4))
