"""The ends of a cache: acceptance where the drafted tree passes the last slot."""
import pytest
import torch

import kv_cache_oracle as K
from sigma0_b200.ops.kv_cache import KVCache, tree_commit, tree_mask

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _walk(par, tok, tgt, fit):
    path = [0] if fit else []
    while path:
        nxt = [i for i in range(path[-1] + 1, fit) if par[i] == path[-1] and tok[i] == tgt[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


@pytest.mark.parametrize("dev", DEVICES)
def test_only_stored_nodes_are_accepted(dev):
    """Six slots, four cached: nodes 0 and 1 are stored, the path 0, 2, 3 is not."""
    par = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device=dev)
    tok = torch.tensor([[3, 8, 7, 9]], device=dev)
    tgt = torch.tensor([[7, 5, 9, 1]], device=dev)
    kc = torch.arange(6.0, device=dev)[:, None].expand(1, 2, 6, 8).contiguous()
    vc = kc + 10
    ls, seen = (torch.tensor([n], dtype=torch.int32, device=dev) for n in (4, 20))
    w, pos = torch.rand(1, 2, 6, device=dev), torch.full((1, 2, 6), 7, dtype=torch.int32, device=dev)
    k0, w0 = kc.clone(), w.clone()
    path, count, token = tree_commit(par, tok, tgt, kc, vc, ls, weight=w, positions=pos, seen=seen)
    assert path.tolist() == [[0, -1, -1, -1]] and count.tolist() == [1] and token.tolist() == [7]
    assert torch.equal(kc, k0) and torch.equal(w[..., :5], w0[..., :5]) and (w[..., 5] == 0).all()
    assert (pos[..., 4] == 20).all() and (pos[..., 5] == -1).all()
    # one slot more: node 2 is stored, node 3 is not
    k7 = torch.arange(7.0, device=dev)[:, None].expand(1, 2, 7, 8).contiguous()
    v7 = k7 + 10
    path, count, token = tree_commit(par, tok, tgt, k7, v7, ls)
    assert path.tolist() == [[0, 2, -1, -1]] and count.tolist() == [2] and token.tolist() == [9]
    assert (k7[..., 5, :] == 6).all() and (v7[..., 5, :] == 16).all()
    # a full cache: not even the root has a row, it stays the token to come
    path, count, token = tree_commit(par, tok, tgt, kc, vc, torch.tensor([6], dtype=torch.int32, device=dev))
    assert path.tolist() == [[-1] * 4] and count.tolist() == [0] and token.tolist() == [3] and torch.equal(kc, k0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,room", [(7, 3), (40, 33), (40, 0), (64, 1), (200, 64)])
def test_a_cache_holds_the_accepted_tokens_and_no_others(dev, T, room):
    """After a step whose tree passes the end: the live slots are the walk over the stored nodes, by their rows and positions."""
    g = torch.Generator().manual_seed(T + room)
    B, layers, nkv, hd, n0 = 3, 2, 2, 16, 5
    S = n0 + room
    c = KVCache(layers, B, nkv, S, hd, torch.float32, dev, budget=S)
    c.lengths.fill_(n0)
    c.seen.fill_(50)
    c.positions[..., :n0] = torch.arange(45, 50, dtype=torch.int32, device=dev)
    par = torch.stack([K.random_tree(T, g, 0.9) for _ in range(B)])
    tgt = torch.randint(0, 2, (B, T), generator=g)
    tok = tgt.gather(1, par.long().clamp_min(0))                       # every child fits: paths reach far down
    new = torch.randn(layers, B, T, nkv, hd, generator=g).to(dev)
    for layer in range(layers):
        c.attend(layer, new[layer], new[layer], -new[layer], tree_mask(par).to(dev))
    path, count, token = c.commit(par.to(dev), tok.to(dev), tgt.to(dev))
    for b in range(B):
        want = _walk(par[b].tolist(), tok[b].tolist(), tgt[b].tolist(), min(T, room))
        n = len(want)
        assert path[b, :n].tolist() == want and (path[b, n:] == -1).all() and int(count[b]) == n
        assert int(token[b]) == (int(tgt[b, want[-1]]) if n else int(tok[b, 0]))
        assert int(c.lengths[b]) == n0 + n <= S and int(c.seen[b]) == 50 + n
        rows = new[:, b, want].transpose(1, 2)
        assert torch.equal(c.k[:, b, :, n0:n0 + n], rows) and torch.equal(c.v[:, b, :, n0:n0 + n], -rows)
        assert (c.positions[:, b, :, :n0 + n] == torch.arange(45, 50 + n, device=dev)).all()
        assert (c.positions[:, b, :, n0 + n:] == -1).all() and (c.weight[:, b, :, n0 + n:] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_one_tensor_for_keys_and_values(dev):
    """Rows that follow one another move down a path whose nodes are others' destinations: each moves once."""
    T, S = 300, 310
    live = [i for i in range(T) if i % 3 != 2]                         # every third node is a draft that does not fit
    par, tok = [0] * T, [5] * T
    for k, i in enumerate(live):
        par[i], tok[i] = live[k - 1] if k else -1, 0
    par, tok = torch.tensor(par, dtype=torch.int32, device=dev), torch.tensor([tok], device=dev)
    kc = torch.arange(float(S), device=dev)[:, None].expand(2, 1, 3, S, 8).contiguous()
    path, count, _ = tree_commit(par, tok, torch.zeros_like(tok), kc, kc, torch.tensor([4], dtype=torch.int32, device=dev))
    n = len(live)
    assert path[0, :n].tolist() == live and int(count) == n
    assert torch.equal(kc[..., 4:4 + n, 0], (torch.tensor(live, device=dev) + 4.0).expand(2, 1, 3, n))
