"""Decoding over a key / value cache: attention of new tokens, eviction, acceptance of drafts.

A cache is a pair of tensors ``[B, kv_heads, slots, head_dim]`` (one layer; the eviction and the
acceptance also take ``[layers, B, kv_heads, slots, head_dim]``) of which the first ``lengths[b]``
slots of sequence ``b`` hold tokens.  Lengths are int32 on the device and nothing here reads them
on the host, so sequences of different lengths share a batch and a step can be captured in a CUDA
graph.  The order of the cached rows means nothing to the attention; ``positions`` (int32, the
cache's shape without the head dimension, -1 in free slots) says which token a slot holds and
``weight`` (float32, 0 in free slots) how much softmax weight it has received.

* :func:`cache_attention` stores the keys and values of T new tokens in slots ``[len, len + T)``
  and attends from them; ``lengths`` stays as it is until the caller adds the tokens that it keeps.
* :func:`cache_evict` cuts every layer and head to ``keep`` tokens by accumulated weight.
* :func:`tree_commit` accepts the path of a drafted tree that agrees with the model.
* :class:`KVCache` holds the tensors of several layers and calls the three.

CUDA tensors run the kernels of ``csrc/kv_attention.cu``, ``csrc/kv_attention_tc.cu`` and
``csrc/kv_evict.cu``; CPU tensors the torch expressions below.  Inference only: none of them has
a gradient.  The reference decodes one token at a time over a static cache that only grows
(``src/base_model/models/transformer.py:285-392``).
"""
from __future__ import annotations

import torch

from ._ext import ext


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """bool [..., T, T] of int parents [..., T] (-1: no parent): row i sees its ancestors and itself.

    A parent has a lower index than its children."""
    T = parents.shape[-1]
    m = torch.eye(T, dtype=torch.bool, device=parents.device).expand(*parents.shape, T).clone()
    for i in range(1, T):
        p = parents[..., i].long()
        up = m.gather(-2, p.clamp_min(0)[..., None, None].expand(*p.shape, 1, T))[..., 0, :]
        m[..., i, :] |= up & (p >= 0)[..., None]
    return m


def tree_depth(mask: torch.Tensor) -> torch.Tensor:
    """int64 [..., T] depth of every node (0 at the root) from its ancestor mask."""
    return mask.sum(-1) - 1


def _inference_only(*ts):
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError("decoding over a cache has no gradient: call it under torch.no_grad()")


def cache_attention(q, k_new, v_new, k_cache, v_cache, lengths, mask=None, scale=None, weight=None, positions=None,
                    seen=None):
    """Attention of T new tokens over the cached tokens and one another -> [B, T, heads, hd].

    q [B, T, heads, hd], k_new / v_new [B, T, kv_heads, hd], caches [B, kv_heads, slots, hd], all of one
    dtype (float32, float16, bfloat16; hd <= 512, T <= 1024) and ``heads`` a multiple of ``kv_heads``.
    Every new token sees the ``lengths[b]`` cached ones and those new ones that its row of ``mask``
    (bool [T, T] or [B, T, T], which may be expanded over the sequences; None: causal) names; a row that sees nothing gives zeros, and a NaN or an
    infinity in a token shows in no row that does not see it.  The new rows are stored in slots ``lengths[b] ...``; rows past the last slot are attended to but not stored.

    ``weight`` [B, kv_heads, slots] gets the probabilities of all T rows and of the group's query heads
    added (through a scratch of 4 bytes per row and slot), ``positions`` the value ``seen[b] + i`` for new
    token i; both in place, so neither may be expanded.  ``scale`` must be positive; k_new and v_new must not overlap the caches."""
    _inference_only(q, k_new, v_new, k_cache, v_cache)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if k_cache.is_cuda:
        return ext().kv_attn(q, k_new, v_new, k_cache, v_cache, lengths, mask, scale, weight, positions, seen)
    return _attention_torch(q, k_new, v_new, k_cache, v_cache, lengths, mask, scale, weight, positions, seen)


def cache_evict(k_cache, v_cache, weight, positions, lengths, seen, keep, recent=0, sinks=0, out=None):
    """Cut every sequence, layer and head to ``keep`` tokens -> (weight, positions, lengths).

    The tokens at positions below ``sinks`` and the ``recent`` last ones (positions from
    ``seen[b] - recent``; ``seen[b]`` tokens have been through the sequence; a token at -1 is neither) stay, then those with the most
    ``weight`` (the lower slot among equals; NaN counts as the most).  Rows of survivors behind the new
    end move into free slots before it, in place.  A sequence of at most ``keep`` tokens stays as it is.
    Slots from the new length on get weight 0 and position -1.  ``out``: three tensors for the results,
    which may be the inputs themselves but not a part of them."""
    if k_cache.is_cuda:
        ow, op, ol = out if out is not None else (None, None, None)
        return tuple(ext().kv_evict(k_cache, v_cache, weight, positions, lengths, seen, keep, recent, sinks, ow, op, ol))
    layers = k_cache.dim() > 4
    args = (k_cache, v_cache, weight, positions) if layers else (x.unsqueeze(0) for x in (k_cache, v_cache, weight, positions))
    w, p, n = _evict_torch(*args, lengths, seen, keep, recent, sinks)
    res = (w, p, n) if layers else (w[0], p[0], n)
    if out is None:
        return res
    _apart(*zip(("weight output", "positions output", "lengths output"), out))
    for o, r in zip(out, res):
        o.copy_(r)
    return tuple(out)


def tree_commit(parents, tokens, targets, k_cache, v_cache, lengths, weight=None, positions=None, seen=None):
    """Accept the root path of a drafted tree that the model agrees with -> (path, count, token).

    Node 0 of the T nodes is the last accepted token; node i hangs below node ``parents[i] < i`` (int32 [T]
    or [B, T]), drafts ``tokens[b, i]`` (int64) and the model continues it with ``targets[b, i]``.  From the
    root the walk goes to the lowest child whose token is the model's, until there is none (where siblings carry
    the same token, a longer path below the higher one is not seen: merge them): ``path``
    int32 [B, T] holds its nodes (-1 behind them), ``count`` int32 [B] how many, ``token`` int64 [B] the
    model's token after the last.  Nodes past the last slot have no rows and are not accepted; where not even
    the root has one, ``count`` is 0 and ``token`` the root's own.  The path's rows, which :func:`cache_attention` left in slots
    ``lengths[b] + node``, move up to ``lengths[b] + 0, 1, ...`` in all layers; ``weight`` follows and is 0
    for the dropped ones, ``positions`` become ``seen[b] + 0, 1, ...`` and -1.  One tensor may be both caches.  ``lengths`` and ``seen``
    stay as they are: add ``count`` to them."""
    if k_cache.is_cuda:
        return tuple(ext().kv_commit(parents, tokens, targets, k_cache, v_cache, lengths, weight, positions, seen))
    if k_cache.dim() == 4:
        k_cache, v_cache = k_cache.unsqueeze(0), v_cache.unsqueeze(0)
        weight, positions = (None if x is None else x.unsqueeze(0) for x in (weight, positions))
    return _commit_torch(parents, tokens, targets, k_cache, v_cache, lengths, weight, positions, seen)


class KVCache:
    """The caches of several layers of one shape, with the lengths that they share.

    ``k`` / ``v`` [layers, B, kv_heads, slots, head_dim]; with a ``budget`` every layer and head keeps at most
    that many tokens (:meth:`trim`): the ``sinks`` first and ``recent`` last ones and those that received the most
    attention.  All state changes in place, so a step over it can be captured in a CUDA graph."""

    def __init__(self, layers, batch, kv_heads, slots, head_dim, dtype=torch.bfloat16, device=None, budget=None,
                 recent=0, sinks=0):
        if budget is not None and not 1 <= budget <= slots:
            raise ValueError(f"a budget of 1 to {slots} tokens, got {budget}")
        shape = (layers, batch, kv_heads, slots)
        # zeros: a slot is read only once it holds a token, but a fresh cache should not look like data
        self.k = torch.zeros(*shape, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.seen = torch.zeros_like(self.lengths)
        self.budget, self.recent, self.sinks = budget, recent, sinks
        self.weight = self.positions = None
        self._new = 0                                         # the most tokens of a step so far
        if budget is not None:
            self.weight = torch.zeros(shape, dtype=torch.float32, device=device)
            self.positions = torch.full(shape, -1, dtype=torch.int32, device=device)

    @property
    def slots(self):
        return self.k.shape[3]

    def attend(self, layer, q, k_new, v_new, mask=None, scale=None):
        """:func:`cache_attention` of one layer; :meth:`add` or :meth:`commit` makes the tokens stay."""
        w, p = (None, None) if self.weight is None else (self.weight[layer], self.positions[layer])
        self._new = max(self._new, q.shape[1])
        return cache_attention(q, k_new, v_new, self.k[layer], self.v[layer], self.lengths, mask=mask, scale=scale,
                               weight=w, positions=p, seen=None if p is None else self.seen)

    def add(self, n):
        """The first ``n`` (an int, or int32 [B]) new tokens of the last step stay; 0 takes the step back.

        The others' slots are free again: their ``weight`` is 0 and their position -1.  What is past the last slot
        was not stored and does not count in ``lengths``."""
        self._keep(n)
        if self.weight is not None and self._new and self.slots:
            # the slots behind the new end that a step may have used; past the last one they name it again
            at = (self.lengths.long()[:, None] + torch.arange(self._new, device=self.lengths.device))
            free = at.clamp_max(self.slots - 1) >= self.lengths[:, None]
            at = at.clamp_max(self.slots - 1)[:, None].expand(*self.weight.shape[:3], self._new)
            free = free[:, None].expand_as(at)
            self.weight.scatter_(-1, at, self.weight.gather(-1, at).masked_fill(free, 0.0))
            self.positions.scatter_(-1, at, self.positions.gather(-1, at).masked_fill(free, -1))

    def _keep(self, n):
        self.lengths.add_(n).clamp_(max=self.slots)
        self.seen += n

    def commit(self, parents, tokens, targets):
        """:func:`tree_commit` over all layers; the accepted tokens stay."""
        path, count, token = tree_commit(parents, tokens, targets, self.k, self.v, self.lengths, weight=self.weight,
                                         positions=self.positions, seen=self.seen if self.weight is not None else None)
        self._keep(count)
        return path, count, token

    def trim(self):
        """:func:`cache_evict` to the budget, if there is one."""
        if self.budget is not None:
            cache_evict(self.k, self.v, self.weight, self.positions, self.lengths, self.seen, self.budget, self.recent,
                        self.sinks, out=(self.weight, self.positions, self.lengths))


def status(like: torch.Tensor) -> int:
    """1 once a bounded wait of the tcgen05 attention gave up on this device (reads the device word)."""
    return int(ext().kv_status(like).item())


def check(like: torch.Tensor) -> None:
    """RuntimeError if :func:`status` is set, which is cleared then; reads the device word, so it waits for the stream.

    The call whose wait gave up has NaN in the rows concerned and may not have stored its new tokens."""
    if like.is_cuda and status(like):
        ext().kv_status(like).zero_()
        raise RuntimeError("cached attention: a wait inside a kernel took longer than its limit; the outputs since are not valid")


def wait_limit(seconds: float = 2.0) -> None:
    """How long a wait inside the tcgen05 attention may take (calls from now on; a captured call keeps its own).

    At 0 every wait gives up at once, which shows what a caller does then."""
    ext().kv_wait_limit(float(seconds))


# ---- torch expressions (CPU tensors) ------------------------------------------------------------
def _apart(*named):
    for name, t in named:
        if t is not None and t.numel():
            span = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            if span < t.numel() or any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
                raise ValueError(f"{name} is written: it must not be expanded")


def _ints(*named, shape=None):
    for name, t in named:
        if t.dtype != torch.int32 or not t.is_contiguous() or t.shape != shape:
            raise ValueError(f"{name}: contiguous int32 {list(shape)}")


def _caches(kc, vc, layers, weight=None, positions=None):
    """What the CUDA entry points ask of the caches and of the tensors of their slots."""
    if kc.dim() not in ((4, 5) if layers else (4,)) or kc.shape != vc.shape or kc.dtype != vc.dtype:
        raise ValueError("the caches must have one shape and one dtype")
    if kc.dtype not in (torch.float32, torch.float16, torch.bfloat16) or not kc.shape[-1]:
        raise ValueError("caches of float32, float16 or bfloat16")
    if kc.stride(-1) != 1 or vc.stride(-1) != 1:
        raise ValueError("the caches' head dimension must be contiguous")
    for name, t, dt in (("weight", weight, torch.float32), ("positions", positions, torch.int32)):
        if t is not None and (t.dtype != dt or t.shape != kc.shape[:-1] or (t.shape[-1] > 1 and t.stride(-1) != 1)):
            raise ValueError(f"{name}: {dt} of the cache's shape without the head dimension, slots contiguous")


def _attention_torch(q, k_new, v_new, kc, vc, lengths, mask, scale, weight, positions, seen):
    _caches(kc, vc, False, weight, positions)
    if q.dim() != 4 or q.shape[0] != kc.shape[0] or q.shape[3] != kc.shape[3]:
        raise ValueError("q, k_new and v_new must match the caches' batch, kv heads and head dim")
    B, T, nh, hd = q.shape
    nkv, S = kc.shape[1], kc.shape[2]
    if any(t.dtype != kc.dtype or t.stride(-1) != 1 for t in (q, k_new, v_new)):
        raise ValueError("q, k_new and v_new: the caches' dtype, contiguous head dimension")
    if hd > 512 or T > 1024 or B > 8192 or not nkv or nh > 1024 * nkv:
        raise ValueError("head dim up to 512, 1024 new tokens, 1024 heads over one kv head, 8192 sequences")
    if not 0 < scale < 1e30:
        raise ValueError("scale must be positive")
    _ints(("lengths", lengths), shape=(B,))
    if mask is not None and (mask.dtype != torch.bool or mask.shape not in ((T, T), (B, T, T), (1, T, T))
                             or (T > 1 and mask.stride()[-2:] != (T, 1))):
        raise ValueError("mask: bool [T, T] or [B, T, T], a sequence's part contiguous")
    if nh % nkv or k_new.shape != (B, T, nkv, hd) or v_new.shape != k_new.shape or kc.shape != vc.shape:
        raise ValueError("q, k_new and v_new must match the caches' batch, kv heads and head dim")
    if positions is not None and seen is None:
        raise ValueError("positions need seen")
    if positions is not None:
        _ints(("seen", seen), shape=(B,))
    _apart(("weight", weight), ("positions", positions))
    new = torch.ones(T, T, dtype=torch.bool).tril() if mask is None else mask
    new = new.expand(B, T, T)
    o = torch.zeros(B, T, nh, hd, dtype=q.dtype)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        k = torch.cat([kc[b, :, :n], k_new[b].transpose(0, 1)], 1).float()
        v = torch.cat([vc[b, :, :n], v_new[b].transpose(0, 1)], 1).float()
        qf = q[b].float().reshape(T, nkv, nh // nkv, hd).permute(1, 2, 0, 3)
        s = qf @ k[:, None].transpose(-1, -2) * scale
        hide = torch.cat([torch.zeros(T, n, dtype=torch.bool), ~new[b]], 1)
        p = torch.softmax(s.masked_fill(hide, float("-inf")), -1).masked_fill(hide.all(-1, keepdim=True), 0.0)
        if torch.isfinite(v_new[b]).all():
            x = p @ v[:, None]
        else:                                    # 0 times an infinity: what a row does not see adds nothing
            x = (p[..., None] * v[:, None, None]).masked_fill(hide[..., None], 0.0).sum(-2)
        o[b] = x.permute(2, 0, 1, 3).reshape(T, nh, hd).to(q.dtype)
        fit = min(T, S - n)
        if weight is not None:
            weight[b, :, :n + fit] += p.sum((1, 2))[:, :n + fit]
        kc[b, :, n:n + fit] = k_new[b, :fit].transpose(0, 1)
        vc[b, :, n:n + fit] = v_new[b, :fit].transpose(0, 1)
        if positions is not None:
            positions[b, :, n:n + fit] = seen[b] + torch.arange(fit, dtype=torch.int32)
    return o


def _evict_torch(kc, vc, w, pos, lengths, seen, keep, recent, sinks):
    if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError("keep >= 1 and recent + sinks <= keep")
    _caches(kc, vc, True, w, pos)
    _ints(("lengths", lengths), ("seen", seen), shape=(kc.shape[1],))
    _apart(("k_cache", kc), ("v_cache", vc))
    S = w.shape[-1]
    slot = torch.arange(S)
    ls = lengths.long().clamp(0, S)[:, None, None]
    new = ls.clamp_max(keep)
    # float64 leaves room above every float32 weight for NaN and the held positions
    key = w.double().clamp(-1e300, 1e300)
    key = key.masked_fill(w.isnan(), 1e301)
    key = key.masked_fill((pos >= 0) & ((pos >= seen[:, None, None] - recent) | (pos < sinks)), 1e302)
    order = key.masked_fill(slot >= ls, float("-inf")).sort(dim=-1, descending=True, stable=True).indices
    stays = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order)) < new
    hole, mover = (slot < new) & ~stays, (slot >= new) & stays
    frm = torch.where(mover, slot, S).sort(-1).values
    src = torch.where(hole, frm.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slot).clamp_max(max(S - 1, 0))
    rows = src[..., None].expand(kc.shape)
    kc.copy_(torch.where(hole[..., None], kc.gather(-2, rows), kc))
    vc.copy_(torch.where(hole[..., None], vc.gather(-2, rows), vc))
    gone = slot >= new
    return (w.gather(-1, src).masked_fill(gone, 0.0), pos.gather(-1, src).masked_fill(gone, -1),
            lengths.clamp(0, S).clamp_max(keep))


def _commit_torch(parents, tokens, targets, kc, vc, lengths, weight, positions, seen):
    if positions is not None and seen is None:
        raise ValueError("positions need seen")
    _apart(("k_cache", kc), ("v_cache", vc), ("weight", weight), ("positions", positions))
    _caches(kc, vc, True, weight, positions)
    if tokens.dim() != 2 or tokens.shape[0] != kc.shape[1] or targets.shape != tokens.shape:
        raise ValueError("tokens and targets: int64 [B, T]")
    B, T = tokens.shape
    S = kc.shape[3]
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in (tokens, targets)) or not 1 <= T <= 1024 or not kc.shape[0]:
        raise ValueError("tokens and targets: contiguous int64 [B, T], 1 to 1024 nodes, at least one layer")
    _ints(("parents", parents), shape=(T,) if parents.dim() == 1 else (B, T))
    _ints(("lengths", lengths), shape=(B,))
    if positions is not None:
        _ints(("seen", seen), shape=(B,))
    par = parents.expand(B, T).tolist()
    path = torch.full((B, T), -1, dtype=torch.int32)
    count = torch.empty(B, dtype=torch.int32)
    token = torch.empty(B, dtype=torch.int64)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        fit = min(T, S - n)                                   # nodes whose rows are in the cache
        walk = [0][:fit]
        while walk:
            cur = walk[-1]
            nxt = next((i for i in range(cur + 1, fit) if par[b][i] == cur and tokens[b, i] == targets[b, cur]), None)
            if nxt is None:
                break
            walk.append(nxt)
        rows = torch.tensor([n + i for i in walk], dtype=torch.long)
        for cache in (kc,) if kc.data_ptr() == vc.data_ptr() else (kc, vc):   # one tensor for both moves once
            cache[:, b, :, n:n + len(walk)] = cache[:, b].index_select(2, rows)
        if weight is not None:
            was = weight[:, b].index_select(2, rows)
            weight[:, b, :, n:n + fit] = 0.0
            weight[:, b, :, n:n + len(walk)] = was
        if positions is not None:
            positions[:, b, :, n:n + fit] = -1
            positions[:, b, :, n:n + len(walk)] = seen[b] + torch.arange(len(walk), dtype=torch.int32)
        path[b, :len(walk)] = torch.tensor(walk, dtype=torch.int32)
        count[b], token[b] = len(walk), targets[b, walk[-1]] if walk else tokens[b, 0]
    return path, count, token
