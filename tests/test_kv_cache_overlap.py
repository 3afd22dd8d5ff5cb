"""Tensors that are written and hold an element at several indexes, and outputs that lie across their inputs, are refused."""
import pytest
import torch

from sigma0_b200.ops.kv_cache import cache_attention, cache_evict, tree_commit

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _case(dev, B=2, nkv=3, S=12, hd=8):
    kc, vc = torch.randn(B, nkv, S, hd, device=dev), torch.randn(B, nkv, S, hd, device=dev)
    w, pos = torch.rand(B, nkv, S, device=dev), torch.arange(S, dtype=torch.int32, device=dev).expand(B, nkv, S).contiguous()
    ls, seen = (torch.full((B,), n, dtype=torch.int32, device=dev) for n in (10, 10))
    return kc, vc, w, pos, ls, seen


def _shared(t):
    """Over books, over heads, over both, and slots that run into the next head's."""
    B, nkv, S = t.shape
    yield t[:1].expand(B, nkv, S)
    yield t[:, :1].expand(B, nkv, S)
    yield t[:1, :1].expand(B, nkv, S)
    yield t.flatten()[:B * nkv + S].as_strided((B, nkv, S), (nkv, 1, 1))


@pytest.mark.parametrize("dev", DEVICES)
def test_shared_elements(dev):
    kc, vc, w, pos, ls, seen = _case(dev)
    q = torch.randn(2, 2, 3, 8, device=dev)
    par, tok = torch.tensor([-1, 0], dtype=torch.int32, device=dev), torch.zeros(2, 2, dtype=torch.long, device=dev)
    before = [x.clone() for x in (kc, vc, w, pos)]
    for bad in _shared(w):
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            cache_attention(q, q, q, kc, vc, ls, weight=bad)
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            tree_commit(par, tok, tok, kc, vc, ls, weight=bad)
    for bad in _shared(pos):
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            cache_attention(q, q, q, kc, vc, ls, positions=bad, seen=seen)
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            tree_commit(par, tok, tok, kc, vc, ls, positions=bad, seen=seen)
    for bad in (kc[:1].expand_as(kc), kc[:, :1].expand_as(kc)):
        for k, v in ((bad, vc), (vc, bad)):
            with pytest.raises((RuntimeError, ValueError), match="expanded"):
                tree_commit(par, tok, tok, k, v, ls)
            with pytest.raises((RuntimeError, ValueError), match="expanded"):
                cache_evict(k, v, w, pos, ls, seen, 4)
    assert all(torch.equal(a, b) for a, b in zip((kc, vc, w, pos), before))


@pytest.mark.parametrize("dev", DEVICES)
def test_eviction_outputs(dev):
    kc, vc, w, pos, ls, seen = _case(dev)
    for o in _shared(w):
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            cache_evict(kc, vc, w, pos, ls, seen, 4, out=(o, pos, ls))
    for o in _shared(pos):
        with pytest.raises((RuntimeError, ValueError), match="expanded"):
            cache_evict(kc, vc, w, pos, ls, seen, 4, out=(w, o, ls))
    # what is only read may be shared: the tokens' numbers are the same in every head
    shared = pos[:1, :1].expand_as(pos)
    k2, v2 = kc.clone(), vc.clone()
    got, want = cache_evict(kc, vc, w, shared, ls, seen, 4, 2, 1), cache_evict(k2, v2, w, pos, ls, seen, 4, 2, 1)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kc, k2) and torch.equal(vc, v2)
    # books interleaved with others' are apart
    wide = torch.empty(2, 2, *w.shape[1:], device=dev)
    wide[:, 0] = w
    cache_evict(kc.clone(), vc.clone(), wide[:, 0], pos, ls, seen, 4, out=(wide[:, 0], pos.clone(), ls.clone()))


@pytest.mark.gpu
def test_outputs_across_their_inputs():
    kc, vc, w, pos, ls, seen = _case("cuda")
    flat = torch.rand(w.numel() + 5, device="cuda")
    a, b = flat[:-5].view_as(w), flat[5:].view_as(w)
    with pytest.raises(RuntimeError, match="overlaps"):
        cache_evict(kc, vc, a, pos, ls, seen, 4, out=(b, pos, ls))
    with pytest.raises(RuntimeError, match="must not be seen"):
        cache_evict(kc, vc, w, pos, ls, seen, 4, out=(w, pos, seen))
    both = torch.full((3,), 10, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        cache_evict(kc, vc, w, pos, both[:2], seen, 4, out=(w, pos, both[1:]))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nkv", [3, 300])
def test_lengths_that_are_also_what_was_seen(dev, nkv):
    """A first cut may be given one tensor for both, in place as well."""
    kc, vc, w, pos, ls, _ = _case(dev, nkv=nkv)
    k2, v2 = kc.clone(), vc.clone()
    want = cache_evict(k2, v2, w, pos, ls.clone(), ls.clone(), 4, 2, 1)
    got = cache_evict(kc, vc, w, pos, ls, ls, 4, 2, 1, out=(w, pos, ls))
    assert got[2].tolist() == [4, 4] and all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kc, k2) and torch.equal(vc, v2)
