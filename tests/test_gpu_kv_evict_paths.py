"""Every launch of the eviction (blocks per unit, keys in shared memory or formed again, who moves the rows, lengths in place)
gives bit for bit what the CPU form does."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(layers, B, nkv, S, hd, dtype, weights, lengths):
    g = torch.Generator().manual_seed(S + layers)
    kc, vc = (torch.randn(layers, B, nkv, S, hd, generator=g).to(dtype) for _ in range(2))
    if weights == "equal":
        w = torch.full((layers, B, nkv, S), 0.5)
    elif weights == "few":                       # many ties in every bin
        w = torch.randint(0, 3, (layers, B, nkv, S), generator=g).float()
    else:
        w = torch.randn(layers, B, nkv, S, generator=g).mul_(2).exp_()
        w[:, 0, 0, ::97], w[:, -1, -1, 5], w[0, 0, 0, 1::101] = float("nan"), float("inf"), -0.0
    pos = torch.rand(layers, B, nkv, S, generator=g).argsort(-1).int()
    ls = torch.tensor([lengths[b % len(lengths)] for b in range(B)], dtype=torch.int32)
    return kc, vc, w, pos, ls, torch.full((B,), S, dtype=torch.int32)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layers,B,nkv,S,hd,dtype,keep,recent,sinks,weights,lengths", [
    (5, 4, 16, 300, 40, torch.bfloat16, 200, 30, 4, "spread", [300, 201, 150, 299]),       # 320 units, 256 threads
    (5, 4, 16, 300, 3, torch.float16, 290, 0, 0, "equal", [300, 0, 291, 299]),
    (5, 4, 16, 3000, 8, torch.bfloat16, 1024, 256, 4, "few", [3000, 1025, 2222, 17]),
    (5, 4, 16, 7000, 2, torch.float32, 4096, 1000, 2, "spread", [7000, 4097, 6999, 5000]),  # 512 threads
    (2, 5, 16, 40000, 2, torch.float32, 9000, 700, 4, "spread", [40000, 39999, 9001, 20000, 1]),   # 79 slots of a thread
    (2, 5, 16, 40000, 2, torch.float32, 39000, 0, 0, "few", [40000, 39990, 39001, 39500, 40000]),
    (1, 1, 2, 8000, 40, torch.bfloat16, 3000, 100, 4, "spread", [8000]),                   # two units, 1,024 threads
    (1, 1, 1, 60000, 8, torch.bfloat16, 20000, 600, 4, "spread", [60000]),                 # keys formed again on every pass
    (2, 5, 16, 60000, 2, torch.float32, 20000, 600, 4, "few", [60000, 59999, 20001, 0, 40000]),
])
def test_every_launch(in_place, layers, B, nkv, S, hd, dtype, keep, recent, sinks, weights, lengths):
    from sigma0_b200.ops.kv_cache import cache_evict
    host = _inputs(layers, B, nkv, S, hd, dtype, weights, lengths)
    dev = [x.cuda() for x in host]
    saved = [x.clone() for x in dev[2:5]]
    got = cache_evict(*dev, keep, recent, sinks, out=(dev[2], dev[3], dev[4]) if in_place else None)
    want = cache_evict(*host, keep, recent, sinks)
    assert torch.equal(got[0].cpu().view(torch.int32), want[0].view(torch.int32))
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    for a, b in zip(dev[:2], host[:2]):
        assert torch.equal(a.cpu(), b)
    if not in_place:                             # the inputs stay
        for a, b in zip(dev[2:5], saved):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32))
