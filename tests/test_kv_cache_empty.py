"""Eviction where there is no layer, head, sequence or slot."""
import pytest
import torch

from sigma0_b200.ops.kv_cache import cache_evict


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("shape", [(0, 3, 2, 9), (2, 3, 0, 9), (2, 0, 2, 9), (2, 3, 2, 0)])
def test_nothing_to_evict(dev, shape):
    kc, w = torch.zeros(*shape, 4, device=dev), torch.zeros(shape, device=dev)
    B, S = shape[1], shape[3]
    ls = torch.tensor([9, 2, -1][:B], dtype=torch.int32, device=dev)
    want = [min(max(n, 0), S, 5) for n in ls.tolist()]
    for out in (None, (w, w.int(), ls.clone())):
        filler = torch.full((64,), -77, dtype=torch.int32, device=dev)   # what the next allocation finds
        del filler
        got = cache_evict(kc, kc.clone(), w, w.int(), ls, ls, 5, out=out)
        assert got[2].tolist() == want and got[0].shape == shape
