"""Both devices take and refuse the same arguments."""
import pytest
import torch

from sigma0_b200.ops.kv_cache import cache_attention, cache_evict, tree_commit, tree_mask

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
REFUSED = (RuntimeError, ValueError)


def _args(dev, B=2, T=3, nkv=2, S=9, hd=8, group=1, dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    q, kn, vn = (torch.randn(B, T, n, hd, generator=g).to(dev, dtype) for n in (nkv * group, nkv, nkv))
    kc, vc = (torch.randn(B, nkv, S, hd, generator=g).to(dev, dtype) for _ in range(2))
    return dict(q=q, k_new=kn, v_new=vn, k_cache=kc, v_cache=vc, lengths=torch.full((B,), 4, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("dev", DEVICES)
def test_attention(dev):
    a = _args(dev)
    m = torch.ones(3, 3, dtype=torch.bool, device=dev).tril()
    w, pos = torch.zeros(2, 2, 9, device=dev), torch.zeros(2, 2, 9, dtype=torch.int32, device=dev)
    kc = a["k_cache"].clone()
    bad = [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(mask=m.float()),
           dict(mask=m[:2]), dict(mask=m.t()), dict(mask=m.expand(3, 3, 3)), dict(lengths=a["lengths"].long()), dict(lengths=a["lengths"][:1]),
           dict(weight=w.half()), dict(weight=w[..., :8]), dict(positions=pos), dict(positions=pos, seen=a["lengths"].long()),
           dict(positions=pos.long(), seen=a["lengths"]), dict(q=a["q"].half()), dict(q=a["q"][:1]), dict(v_cache=a["v_cache"].half()),
           dict(v_cache=a["v_cache"][:, :, :8]), {k: v.double() if v.is_floating_point() else v for k, v in a.items()}]
    for b in bad:
        with pytest.raises(REFUSED):
            cache_attention(**{**a, **b})
    for wide in (dict(T=1025, S=1), dict(hd=513), dict(group=1025, nkv=1, T=1)):
        with pytest.raises(REFUSED):
            cache_attention(**_args(dev, **wide))
    assert torch.equal(a["k_cache"], kc)
    cache_attention(**_args(dev, T=1024, S=1, B=1, nkv=1))
    cache_attention(**_args(dev, hd=512))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,T", [(1, 1), (2, 3), (3, 20), (2, 1)])
def test_masks_may_be_expanded(dev, B, T):
    """One mask for all sequences: [T, T], [1, T, T], expanded, every other of a batch -- the same outputs."""
    a = _args(dev, B=B, T=T, S=40, dtype=torch.bfloat16)
    par = torch.tensor([-1] + [i // 2 for i in range(T - 1)], dtype=torch.int32)
    m = tree_mask(par).to(dev)
    want = cache_attention(**a, mask=m.expand(B, T, T).contiguous())
    for mask in (m, m[None], m.expand(B, T, T), m[None].expand(B, T, T), m.expand(2 * B, T, T).contiguous()[::2]):
        assert torch.equal(cache_attention(**a, mask=mask), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_eviction_and_commit(dev):
    a = _args(dev)
    kc, vc, ls = a["k_cache"], a["v_cache"], a["lengths"]
    w, pos = torch.zeros(2, 2, 9, device=dev), torch.zeros(2, 2, 9, dtype=torch.int32, device=dev)
    for x in [(kc, vc.half(), w, pos, ls, ls), (kc, vc[:, :, :8], w, pos, ls, ls), (kc, vc, w.double(), pos, ls, ls), (kc, vc, w, pos.long(), ls, ls),
              (kc, vc, w[..., :8], pos, ls, ls), (kc, vc, w, pos, ls.long(), ls), (kc, vc, w, pos, ls, ls[:1])]:
        with pytest.raises(REFUSED):
            cache_evict(*x, 2)
    par, t = torch.tensor([-1, 0, 1], dtype=torch.int32, device=dev), torch.zeros(2, 3, dtype=torch.long, device=dev)
    for x in [(par.long(), t, t, kc, vc, ls), (par[:2], t, t, kc, vc, ls), (par, t.int(), t, kc, vc, ls), (par, t, t[:, :2], kc, vc, ls),
              (par, t[:1], t[:1], kc, vc, ls), (par, t, t, kc, vc.half(), ls), (par, t, t, kc, vc, ls.long()), (par[:0], t[:, :0], t[:, :0], kc, vc, ls)]:
        with pytest.raises(REFUSED):
            tree_commit(*x)
