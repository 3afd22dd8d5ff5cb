"""KVCache.add: tokens of a step that do not stay leave no weight and no position behind."""
import pytest
import torch

import kv_cache_oracle as K
from sigma0_b200.ops.kv_cache import KVCache

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _step(c, T, g, dev):
    """One step of T tokens in every layer; returns the weights that its rows add, [layers, B, heads, slots]."""
    layers, B, nkv, S, hd = c.k.shape
    added = []
    for layer in range(layers):
        q, kn, vn = (torch.randn(B, T, nkv, hd, generator=g).to(dev) for _ in range(3))
        _, w = K.attention(q, kn, vn, c.k[layer], c.v[layer], c.lengths.tolist(), None, hd ** -0.5)
        c.attend(layer, q, kn, vn)
        added.append(w)
    return torch.stack(added)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("S", [40, 11])
def test_dropped_tokens_leave_nothing_behind(dev, S):
    """Steps of several lengths of which some tokens stay (an int, one number per sequence, none), at last past the end."""
    g = torch.Generator().manual_seed(S)
    B, layers, nkv, hd = 3, 2, 2, 8
    c = KVCache(layers, B, nkv, S, hd, torch.float32, dev, budget=S)
    want = torch.zeros(layers, B, nkv, S, dtype=torch.float64, device=dev)
    n = torch.zeros(B, dtype=torch.int32, device=dev)
    for T, keep in ((5, 2), (3, 0), (4, [0, 4, 1]), (1, 1), (7, [3, 0, 5]), (2, 2)):
        want += _step(c, T, g, dev)
        keep = torch.tensor(keep, dtype=torch.int32, device=dev) if isinstance(keep, list) else keep
        c.add(keep)
        n = (n + keep).clamp(max=S)
        free = torch.arange(S, device=dev) >= n[:, None, None]
        want = want.masked_fill(free, 0.0)
        assert torch.equal(c.lengths, n)
        assert K.rel(c.weight, want) < K.WEIGHT_TOL and (c.weight.masked_select(free.expand_as(c.weight)) == 0).all()
        assert (c.positions.masked_select(free.expand_as(c.positions)) == -1).all()
        live = torch.arange(S, device=dev).expand_as(c.positions).masked_fill(free, -1)
        assert torch.equal(c.positions.long(), live)          # nothing was dropped before the end, so slot = position


@pytest.mark.parametrize("dev", DEVICES)
def test_add_without_a_budget(dev):
    c = KVCache(1, 2, 1, 6, 8, torch.float32, dev)
    q = torch.randn(2, 4, 1, 8).to(dev)
    c.attend(0, q, q, q)
    c.add(3)
    c.attend(0, q, q, q)
    c.add(torch.tensor([4, 1], dtype=torch.int32, device=dev))
    assert c.lengths.tolist() == [6, 4] and c.seen.tolist() == [7, 4]
