"""Eviction of cached tokens without a position (-1): neither first nor recent, they stay by their weight alone."""
import pytest
import torch

from sigma0_b200.ops.kv_cache import cache_evict


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("recent,sinks,seen", [(0, 2, 8), (3, 0, 2), (2, 2, 8)])
def test_tokens_without_a_position(dev, recent, sinks, seen):
    S, keep = 8, 4
    pos = torch.tensor([-1, 0, 1, 2, -1, 5, 6, 7], dtype=torch.int32).expand(1, 2, S).contiguous().to(dev)
    w = torch.tensor([1.0, 2.0, 3.0, 9.0, 0.0, 8.0, 5.0, 4.0]).expand(1, 2, S).contiguous().to(dev)
    kc = torch.arange(8.0, device=dev)[:, None].expand(1, 2, S, 4).contiguous()
    ls, sn = (torch.tensor([n], dtype=torch.int32, device=dev) for n in (S, seen))
    _, p2, _ = cache_evict(kc, kc.clone(), w, pos, ls, sn, keep, recent, sinks)
    first = [p for p in (0, 1, 2, 5, 6, 7) if p < sinks or p >= seen - recent]
    weight = dict(zip((0, 1, 2, 5, 6, 7), (2.0, 3.0, 9.0, 8.0, 5.0, 4.0)))
    # of the equally held the lower slot: slots are in the order of the positions here
    want = (first + sorted((p for p in weight if p not in first), key=lambda p: -weight[p]))[:keep]
    for h in range(2):
        assert sorted(p2[0, h, :keep].tolist()) == sorted(want)
