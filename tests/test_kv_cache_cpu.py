"""The cache operators' torch expressions (CPU) against 64-bit loops, and the helpers of drafted trees."""
import pytest
import torch

import kv_cache_oracle as K
from sigma0_b200.ops.kv_cache import cache_attention, cache_evict, tree_commit, tree_depth, tree_mask


def test_tree_mask_and_depth():
    par = torch.tensor([[-1, 0, 0, 1, 3], [-1, 0, 1, 2, 3]], dtype=torch.int32)
    m = tree_mask(par)
    want = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 1, 0, 1, 1]]).bool()
    assert torch.equal(m[0], want) and torch.equal(m[1], torch.ones(5, 5).tril().bool())
    assert torch.equal(tree_mask(par[0]), want)
    assert tree_depth(m).tolist() == [[0, 1, 1, 2, 3], [0, 1, 2, 3, 4]]


@pytest.mark.parametrize("B,T,nh,nkv,hd,S,lengths,tree", [
    (1, 1, 2, 2, 8, 9, [5], False),
    (3, 4, 6, 2, 5, 12, [0, 3, 10], True),
    (2, 3, 2, 1, 7, 0, [0, 0], False),
])
def test_attention_cpu(B, T, nh, nkv, hd, S, lengths, tree):
    g = torch.Generator().manual_seed(B * 10 + T)
    q, kn, vn = (torch.randn(B, T, n, hd, generator=g) for n in (nh, nkv, nkv))
    kc, vc = torch.randn(B, nkv, S, hd, generator=g), torch.randn(B, nkv, S, hd, generator=g)
    ls = torch.tensor(lengths, dtype=torch.int32)
    mask = torch.stack([tree_mask(K.random_tree(T, g)) for _ in range(B)]) if tree else None
    if tree:
        mask[0, 1] = False                       # sequence 0 has nothing cached: this row sees nothing
    w, pos, seen = torch.rand(B, nkv, S, generator=g), torch.full((B, nkv, S), -1, dtype=torch.int32), ls + 7
    o64, w64 = K.attention(q, kn, vn, kc, vc, lengths, mask, hd ** -0.5)
    w0 = w.clone()
    o = cache_attention(q, kn, vn, kc, vc, ls, mask=mask, weight=w, positions=pos, seen=seen)
    assert K.rel(o, o64) < K.tolerance(torch.float32)
    if S:
        assert K.rel(w, w0 + w64) < K.WEIGHT_TOL
    if tree:
        assert (o[0, 1] == 0).all()
    for b, n in enumerate(lengths):
        fit = min(T, S - n)
        assert torch.equal(kc[b, :, n:n + fit], kn[b, :fit].transpose(0, 1))
        assert torch.equal(vc[b, :, n:n + fit], vn[b, :fit].transpose(0, 1))
        assert (pos[b, :, n:n + fit] == torch.arange(fit) + n + 7).all()


@pytest.mark.parametrize("keep,recent,sinks", [(4, 0, 0), (5, 2, 1), (6, 6, 0), (1, 0, 0), (30, 3, 2)])
def test_evict_cpu(keep, recent, sinks):
    g = torch.Generator().manual_seed(keep)
    N, B, nkv, S, hd = 2, 3, 2, 14, 3
    kc, vc = torch.randn(N, B, nkv, S, hd, generator=g), torch.randn(N, B, nkv, S, hd, generator=g)
    ls = torch.tensor([14, 9, 0], dtype=torch.int32)
    seen = ls + 20
    w = torch.randint(0, 4, (N, B, nkv, S), generator=g).float()
    w[0, 0, 0, 3] = float("nan")
    pos = torch.rand(N, B, nkv, S, generator=g).argsort(-1).int() + 20
    k0, v0 = kc.clone(), vc.clone()
    w2, p2, l2 = cache_evict(kc, vc, w, pos, ls, seen, keep, recent, sinks)
    assert l2.tolist() == [min(n, keep) for n in ls.tolist()]
    for n in range(N):
        for b in range(B):
            for h in range(nkv):
                src = K.evict(w[n, b, h].tolist(), pos[n, b, h].tolist(), int(ls[b]), int(seen[b]), keep, recent, sinks)
                m = len(src)
                assert torch.equal(kc[n, b, h, :m], k0[n, b, h, src]) and torch.equal(vc[n, b, h, :m], v0[n, b, h, src])
                assert torch.equal(kc[n, b, h, m:], k0[n, b, h, m:])
                assert torch.equal(w2[n, b, h, :m].nan_to_num(99.0), w[n, b, h, src].nan_to_num(99.0)) and (w2[n, b, h, m:] == 0).all()
                assert torch.equal(p2[n, b, h, :m], pos[n, b, h, src]) and (p2[n, b, h, m:] == -1).all()


def test_evict_cpu_in_place_and_one_layer():
    g = torch.Generator().manual_seed(3)
    kc, vc = torch.randn(1, 2, 6, 4, generator=g), torch.randn(1, 2, 6, 4, generator=g)
    w, pos = torch.rand(1, 2, 6, generator=g), torch.arange(6, dtype=torch.int32).expand(1, 2, 6).contiguous()
    ls, seen = torch.tensor([6], dtype=torch.int32), torch.tensor([6], dtype=torch.int32)
    want = cache_evict(kc.clone(), vc.clone(), w, pos, ls, seen, 3, 1, 1)
    got = cache_evict(kc, vc, w, pos, ls, seen, 3, 1, 1, out=(w, pos, ls))
    assert got[0] is w and all(torch.equal(a, b) for a, b in zip(want, got)) and want[0].shape == (1, 2, 6)


def test_commit_cpu():
    par = torch.tensor([-1, 0, 0, 2, 2, 4], dtype=torch.int32)
    tgt = torch.tensor([[7, 1, 5, 2, 9, 3], [7, 1, 5, 2, 9, 3]])
    tok = torch.tensor([[0, 6, 7, 5, 5, 9], [0, 8, 8, 5, 5, 9]])     # row 0: 0 -> 2 -> 3 (the lower twin); row 1: root only
    g = torch.Generator().manual_seed(1)
    kc, vc = torch.randn(2, 2, 3, 10, 4, generator=g), torch.randn(2, 2, 3, 10, 4, generator=g)
    k0, v0 = kc.clone(), vc.clone()
    ls, seen = torch.tensor([2, 4], dtype=torch.int32), torch.tensor([30, 40], dtype=torch.int32)
    w, pos = torch.rand(2, 2, 3, 10, generator=g), torch.zeros(2, 2, 3, 10, dtype=torch.int32)
    w0 = w.clone()
    path, count, token = tree_commit(par, tok, tgt, kc, vc, ls, weight=w, positions=pos, seen=seen)
    assert path.tolist() == [[0, 2, 3, -1, -1, -1], [0, -1, -1, -1, -1, -1]]
    assert count.tolist() == [3, 1] and token.tolist() == [2, 7]
    assert torch.equal(kc[:, 0, :, 2:5], k0[:, 0][:, :, [2, 4, 5]]) and torch.equal(vc[:, 0, :, 2:5], v0[:, 0][:, :, [2, 4, 5]])
    assert torch.equal(kc[:, 1], k0[:, 1])
    assert torch.equal(w[:, 0, :, 2:5], w0[:, 0][:, :, [2, 4, 5]]) and (w[:, 0, :, 5:8] == 0).all() and torch.equal(w[:, 0, :, 8:], w0[:, 0, :, 8:])
    assert pos[0, 0, 0].tolist() == [0, 0, 30, 31, 32, -1, -1, -1, 0, 0] and pos[1, 1, 2].tolist() == [0, 0, 0, 0, 40, -1, -1, -1, -1, -1]


def test_refusals_cpu():
    q, kn = torch.randn(1, 1, 3, 4), torch.randn(1, 1, 2, 4)
    kc = torch.zeros(1, 2, 5, 4)
    ls = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        cache_attention(q, kn, kn, kc, kc.clone(), ls)                    # 3 heads over 2
    with pytest.raises(RuntimeError):
        cache_attention(torch.randn(1, 1, 2, 4, requires_grad=True), kn, kn, kc, kc.clone(), ls)
    w = torch.zeros(1, 2, 5)
    with pytest.raises(ValueError):
        cache_evict(kc, kc.clone(), w, w.int(), ls, ls, keep=3, recent=3, sinks=1)
    with pytest.raises(ValueError):
        tree_commit(torch.tensor([-1], dtype=torch.int32), ls[None].long(), ls[None].long(), kc, kc.clone(), ls, positions=w.int())
