"""Decoding over a key / value cache: the cases that time its operators, with their plain forms.

Three operators serve a transformer (or hybrid) model that generates from a cache:

* ``attention`` -- a few new tokens of every sequence (one token, a causal run of them, or a tree of
  drafted tokens under an ancestor mask) are stored behind the ``lengths[b]`` cached ones and attend
  to those and to the new tokens that their mask row lets them see; optionally the softmax weight
  that every cached position received is added up for the eviction;
* ``evict`` -- every sequence, layer and head keeps its first and most recent tokens and those that
  received the most weight; survivors behind the new end move into the holes before it;
* ``commit`` -- the longest root path of drafted tokens that the model itself would have produced is
  accepted, its cache rows move up behind the cached ones, and the others are dropped.

``run`` computes an operator in its plain form (32-bit torch expressions) or, with ``own`` set,
through the package.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


def listed():
    att = dict(op="attention", batch=1, heads=16, kv_heads=16, head_dim=64, dtype="bfloat16", length=440,
               ragged=False, nodes=1, tree=False, weights=False)
    ev = dict(op="evict", layers=1, batch=1, kv_heads=16, head_dim=64, dtype="bfloat16", length=534, ragged=False,
              keep=512, recent=128, sinks=4)
    co = dict(op="commit", layers=1, batch=1, kv_heads=16, head_dim=64, dtype="bfloat16", capacity=512, nodes=8,
              accepted=3)
    return [
        # one book, a short context of 20 messages of 22 tokens, the next token: pure latency
        dict(att, name="one_token_short"),
        # a generation batch: 64 books of up to 500 messages, the next token, weights kept for the eviction
        dict(att, name="one_token_64_books", batch=64, length=11000, ragged=True, weights=True),
        # one book with the longest context of the presets (3,000 messages): work split over the keys
        dict(att, name="one_token_long", head_dim=128, length=66000),
        # grouped heads: four query heads read one key head
        dict(att, name="one_token_grouped", batch=16, kv_heads=4, head_dim=128, dtype="float16", length=26000,
             ragged=True, weights=True),
        # a drafted tree over long contexts of many books: the largest, tensor-core work counts
        dict(att, name="tree_64_many_books", batch=16, head_dim=128, length=22000, ragged=True, nodes=64, tree=True),
        # an odd tree under grouped heads, contexts from none to medium
        dict(att, name="tree_61_grouped", batch=8, kv_heads=4, head_dim=128, dtype="float16", length=3001, ragged=True,
             nodes=61, tree=True),
        # a whole known message (22 tokens, causal) in float32, the package's default compute type
        dict(att, name="message_float32", batch=8, dtype="float32", length=2200, ragged=True, nodes=22, weights=True),
        # after one message over a full budget: 22 tokens go
        dict(ev, name="evict_one_message"),
        # cutting prompts of 500 messages to a budget, four layers at once
        dict(ev, name="evict_prompts", layers=4, batch=16, length=11000, ragged=True, keep=2048, recent=512),
        # the steady state of a 24-layer model: a message over the budget in each of 16 books
        dict(ev, name="evict_24_layers", layers=24, batch=16, length=4118, keep=4096, recent=1024),
        # one book, one layer, eight drafted tokens
        dict(co, name="commit_small"),
        # 24 layers, 32 books, 64 drafted tokens
        dict(co, name="commit_24_layers", layers=24, batch=32, capacity=1001, nodes=64, accepted=9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention"] * 4 + ["evict"] * 2 + ["commit"])
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["op"], {"bytes": 0, "flops": 0})
        t["bytes"], t["flops"] = max(t["bytes"], w["bytes"]), max(t["flops"], w["flops"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    # heads of 64 or 128 as the presets have them, and narrow or odd ones (a 503-wide book layer is one head)
    kv, hd = rng.choice([(16, 64), (16, 64), (16, 128), (16, 128), (4, 128), (2, 64), (8, 40), (1, 503)])
    if op == "attention":
        nodes = 1 if rng.random() < 0.5 else _log_int(rng, 2, 64)
        c = dict(op=op, batch=_log_int(rng, 1, 64), heads=kv * (1 if kv in (1, 8, 16) else rng.choice([2, 3, 4])),
                 kv_heads=kv, head_dim=hd, dtype=dtype, length=_log_int(rng, 1, 66000), ragged=rng.random() < 0.5,
                 nodes=nodes, tree=nodes > 1 and rng.random() < 0.7, weights=rng.random() < 0.5)
    elif op == "evict":
        keep = _log_int(rng, 64, 8192)
        recent = rng.randint(0, keep // 2)
        c = dict(op=op, layers=_log_int(rng, 1, 24), batch=_log_int(rng, 1, 64), kv_heads=kv, head_dim=hd, dtype=dtype,
                 length=keep + _log_int(rng, 1, 8192), ragged=rng.random() < 0.5, keep=keep, recent=recent,
                 sinks=rng.randint(0, 8))
    else:
        nodes = _log_int(rng, 2, 64)
        c = dict(op=op, layers=_log_int(rng, 1, 24), batch=_log_int(rng, 1, 64), kv_heads=kv, head_dim=hd, dtype=dtype,
                 capacity=nodes + _log_int(rng, 64, 1024), nodes=nodes, accepted=rng.randint(1, max(1, nodes // 2)))
    while any(w > top[op][k] for k, w in work(c).items()) or _held(c) > 8e9:
        for k in ("batch", "layers", "length" if op == "attention" else "nodes"):
            if c.get(k, 1) > 1:
                c[k] = (c[k] + 1) // 2
                break
        else:
            break
        if op != "evict":
            c["tree"] = c["nodes"] > 1 and c.get("tree", False)
            if op == "commit":
                c["accepted"] = min(c["accepted"], max(1, c["nodes"] // 2))
                c.pop("tree")
    return c


def _lengths(c):
    """The cached tokens of every sequence: all `length`, or spread from a quarter of it (and one empty) up to it."""
    n, B = c["length"], c["batch"]
    if not c["ragged"]:
        return [n] * B
    ls = [max(1, n - (3 * n * b) // (4 * B)) for b in range(B)]
    if B >= 4 and c["op"] == "attention":
        ls[-1] = 0
    return ls


def _held(c):
    cap = c["capacity"] if c["op"] == "commit" else c["length"] + c.get("nodes", 0)
    return 2 * c.get("layers", 1) * c["batch"] * c["kv_heads"] * cap * c["head_dim"] * BYTES[c["dtype"]]


def work(case):
    c = case
    es, hd, kv, B = BYTES[c["dtype"]], c["head_dim"], c["kv_heads"], c["batch"]
    if c["op"] == "attention":
        T, nh = c["nodes"], c["heads"]
        total = sum(_lengths(c))
        byt = 2 * total * kv * hd * es                      # cached keys and values
        byt += 2 * 2 * B * T * kv * hd * es                 # new ones: read, stored into the cache
        byt += 2 * B * T * nh * hd * es                     # queries, outputs
        if c["weights"]:
            byt += 8 * kv * (total + B * T) + 4 * kv * B * T    # accumulated weights read and written, positions
        return {"bytes": float(byt), "flops": 4.0 * T * nh * hd * (total + B * (T + 1) / 2)}
    if c["op"] == "evict":
        units, cap = c["layers"] * kv, c["length"]
        byt = flops = 0.0
        for n in _lengths(c):
            byt += units * (8 * n + 8 * cap)                # weights and positions: read, written
            flops += units * n
            over = n - c["keep"]
            if over > 0:                                    # survivors behind the new end: their rows move
                moved = over if c["recent"] >= over else c["recent"] + (over - c["recent"]) * (
                    c["keep"] - c["recent"] - c["sinks"]) / (n - c["recent"] - c["sinks"])
                byt += units * moved * 2 * 2 * hd * es
        return {"bytes": byt, "flops": flops}
    rows = sum(_accepted(c)) - B                            # the root stays where it is
    byt = 4 * hd * es * rows * c["layers"] * kv + 20 * B * c["nodes"] + 8 * c["layers"] * kv * B * c["nodes"]
    return {"bytes": float(byt), "flops": float(B * c["nodes"])}


def _accepted(c):
    """How many drafted tokens every sequence accepts, the root among them."""
    return [1 + (7 * b + c["accepted"] - 1) % c["accepted"] for b in range(c["batch"])]


def _trees(B, T, gen):
    """Random trees: the parent of node i is a lower node, near i as often as not; node 0 is the root."""
    i = torch.arange(T, device=gen.device)
    u = torch.rand(B, T, generator=gen, device=gen.device)
    back = 1 + (u * u * i).floor().long().clamp_max(T)
    return torch.where(i > 0, (i - back).clamp_min(0), -torch.ones_like(i)).int()


def _ancestors(parents):
    """[B, T, T] truth values: row i has its ancestors and itself (the closure of the parent relation)."""
    B, T = parents.shape
    a = torch.eye(T, device=parents.device).expand(B, T, T) + torch.nn.functional.one_hot(
        parents.long().clamp_min(0), T) * (parents >= 0)[..., None]
    for _ in range(max(1, (T - 1).bit_length())):
        a = (a @ a).clamp_max(1)
    return a > 0


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=DTYPES[c["dtype"]])

    B, kv, hd = c["batch"], c["kv_heads"], c["head_dim"]
    if c["op"] == "attention":
        T, nh, S = c["nodes"], c["heads"], c["length"] + c["nodes"]
        ls = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
        s = dict(case=c, k_cache=rand(B, kv, S, hd), v_cache=rand(B, kv, S, hd),
                 lengths=ls[torch.randperm(B, generator=gen, device="cuda")])
        # projections of one matrix: q, k and v are strided views of its rows, some keys stand out
        qkv = rand(B, T, nh + 2 * kv, hd)
        s["q"], s["k_new"], s["v_new"] = qkv.split([nh, kv, kv], 2)
        s["q"].mul_(1.5)
        s["mask"] = _ancestors(_trees(B, T, gen)) if c["tree"] else None
        s["weight"] = torch.rand(B, kv, S, generator=gen, device="cuda") if c["weights"] else None
        if c["weights"]:                                    # nothing has looked behind the cached tokens yet
            slot = torch.arange(S, device="cuda", dtype=torch.int32)
            gone = (slot >= s["lengths"][:, None, None]).expand(B, kv, S)
            s["weight"].masked_fill_(gone, 0)
            s["seen"] = s["lengths"] + 1000
            s["positions"] = (slot + 1000).expand(B, kv, S).masked_fill(gone, -1)
        return s
    N, cap = c["layers"], c["capacity"] if c["op"] == "commit" else c["length"]
    s = dict(case=c, k_cache=rand(N, B, kv, cap, hd), v_cache=rand(N, B, kv, cap, hd))
    slot = torch.arange(cap, device="cuda", dtype=torch.int32)
    if c["op"] == "evict":
        ls = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
        s["lengths"] = ls[torch.randperm(B, generator=gen, device="cuda")]
        s["seen"] = s["lengths"] + 1000 * (1 + torch.arange(B, device="cuda", dtype=torch.int32))
        # heavy-tailed sums with many equal small ones; earlier evictions left the older slots out of order
        w = torch.randn(N, B, kv, cap, generator=gen, device="cuda").mul_(1.5).exp_()
        s["weight"] = torch.where(w < 0.25, (w * 16).floor() / 16, w)
        old = (s["lengths"].clamp_max(c["keep"]) - c["recent"]).clamp_min(0)[:, None, None]
        mix = torch.rand(N, B, kv, cap, generator=gen, device="cuda")
        mix = torch.where(slot < old, mix, slot + 1.0).argsort(-1).int()
        pos = mix + (s["seen"] - s["lengths"])[:, None, None]
        s["positions"] = torch.where((slot < c["sinks"]) & (pos > c["sinks"]), slot, pos)
        gone = slot >= s["lengths"][:, None, None]
        s["weight"].masked_fill_(gone, 0)
        s["positions"].masked_fill_(gone, -1)
        return s
    T = c["nodes"]
    s["lengths"] = torch.randint(0, cap - T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    s["seen"] = s["lengths"] + 500
    # the accepted path: node 0 and the lowest of random nodes; its tokens are the model's, the others are not
    n = torch.tensor(_accepted(c), device="cuda")[:, None]
    key = torch.rand(B, T, generator=gen, device="cuda")
    key[:, 0] = -1
    on = key.argsort(-1).argsort(-1) < n
    node = torch.arange(T, device="cuda").expand(B, T)
    last = torch.where(on, node, 0).cummax(-1).values       # the latest path node up to here
    before = torch.cat([torch.full_like(last[:, :1], -1), last[:, :-1]], 1)
    s["parents"] = torch.where(on, before.int(), _trees(B, T, gen))
    s["targets"] = torch.randint(0, 12288, (B, T), generator=gen, device="cuda")
    said = s["targets"].gather(1, s["parents"].long().clamp_min(0))
    s["tokens"] = torch.where(on, said, (said + 1 + node) % 12288)
    s["mask"] = _ancestors(s["parents"])
    s["weight"] = torch.rand(N, B, kv, cap, generator=gen, device="cuda")
    s["positions"] = (slot + 500).expand(N, B, kv, cap).contiguous()
    return s


def run(state):
    s, c = state, state["case"]
    if c["op"] == "attention":
        return _own_attention(s) if own else _plain_attention(s)
    if c["op"] == "evict":
        return _own_evict(s, c) if own else _plain_evict(s, c)
    return _own_commit(s) if own else _plain_commit(s)


def _own_attention(s):
    from sigma0_b200.ops.kv_cache import cache_attention
    o = cache_attention(s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["lengths"], mask=s["mask"],
                        weight=s["weight"], positions=s.get("positions"), seen=s.get("seen"))
    return dict(o=o, k_cache=s["k_cache"], v_cache=s["v_cache"], weight=s["weight"], positions=s.get("positions"))


def _own_evict(s, c):
    from sigma0_b200.ops.kv_cache import cache_evict
    weight, positions, lengths = cache_evict(s["k_cache"], s["v_cache"], s["weight"], s["positions"], s["lengths"],
                                             s["seen"], keep=c["keep"], recent=c["recent"], sinks=c["sinks"])
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"], weight=weight, positions=positions, lengths=lengths)


def _own_commit(s):
    from sigma0_b200.ops.kv_cache import tree_commit
    path, count, token = tree_commit(s["parents"], s["tokens"], s["targets"], s["k_cache"], s["v_cache"], s["lengths"],
                                     weight=s["weight"], positions=s["positions"], seen=s["seen"])
    return dict(path=path, count=count, token=token, k_cache=s["k_cache"], v_cache=s["v_cache"], weight=s["weight"],
                positions=s["positions"])


def _plain_attention(s):
    q, kc, vc, ls = s["q"], s["k_cache"], s["v_cache"], s["lengths"].long()
    B, T, nh, hd = q.shape
    kv, S = kc.shape[1], kc.shape[2]
    at = ls[:, None] + torch.arange(T, device=q.device)                       # slots of the new tokens
    to = at[:, None, :, None].expand(B, kv, T, hd)
    kc.scatter_(2, to, s["k_new"].transpose(1, 2))
    vc.scatter_(2, to, s["v_new"].transpose(1, 2))
    slot = torch.arange(S, device=q.device)
    among = (slot - ls[:, None]).clamp(0, T - 1)[:, None, :].expand(B, T, S)  # which new token a slot holds
    mask = s["mask"] if s["mask"] is not None else torch.ones(T, T, dtype=torch.bool, device=q.device).tril()
    seen = mask.expand(B, T, T).gather(2, among) & (slot < ls[:, None, None] + T) | (slot < ls[:, None, None])
    qf = q.float().reshape(B, T, kv, nh // kv, hd).permute(0, 2, 3, 1, 4)     # [B, kv, group, T, hd]
    sc = (qf @ kc.float()[:, :, None].transpose(-1, -2)) * hd ** -0.5
    sc = sc.masked_fill(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - top.clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = (p @ vc.float()[:, :, None]).permute(0, 3, 1, 2, 4).reshape(B, T, nh, hd).to(q.dtype)
    if s["weight"] is not None:
        s["weight"].add_(p.sum((2, 3)))
        now = (s["seen"].long()[:, None] + torch.arange(T, device=q.device)).int()
        s["positions"].scatter_(2, to[..., 0], now[:, None].expand(B, kv, T))
    return dict(o=o, k_cache=kc, v_cache=vc, weight=s["weight"], positions=s.get("positions"))


def _plain_evict(s, c):
    w, pos, seen = s["weight"], s["positions"], s["seen"][:, None, None]
    S, keep = w.shape[-1], c["keep"]
    slot = torch.arange(S, device=w.device)
    ls = s["lengths"].long()[:, None, None]
    new = ls.clamp_max(keep)
    held = (pos >= seen - c["recent"]) | (pos < c["sinks"])
    rank_by = w.masked_fill(held, float("inf")).masked_fill(slot >= ls, float("-inf"))
    order = torch.sort(rank_by, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    stays = rank < new
    hole, mover = (slot < new) & ~stays, (slot >= new) & stays
    movers = torch.where(mover, slot, S).sort(-1).values                      # in order of their slots
    src = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slot)
    k = min(keep, S)
    rows = src[..., :k, None].expand(*src.shape[:-1], k, s["k_cache"].shape[-1])
    s["k_cache"][..., :k, :] = s["k_cache"].gather(-2, rows)
    s["v_cache"][..., :k, :] = s["v_cache"].gather(-2, rows)
    gone = slot >= new
    src = src.clamp_max(S - 1)
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"], weight=w.gather(-1, src).masked_fill(gone, 0),
                positions=pos.gather(-1, src).masked_fill(gone, -1), lengths=s["lengths"].clamp_max(keep))


def _plain_commit(s):
    par, tok, tgt, kc, vc = s["parents"].long(), s["tokens"], s["targets"], s["k_cache"], s["v_cache"]
    B, T = tok.shape
    N, _, kv, S, hd = kc.shape
    node = torch.arange(T, device=tok.device)
    fits = (tok == tgt.gather(1, par.clamp_min(0))) & (par >= 0)
    rival = (par[:, :, None] == par[:, None, :]) & fits[:, None, :] & (node[None, :] < node[:, None])
    fits = fits & ~rival.any(-1) | (node == 0)                                # the lowest child that fits
    on = (fits[:, None, :] | ~s["mask"]).all(-1)                              # all of its root path fits
    count = on.sum(-1)
    path = torch.where(on, node, T).sort(-1).values
    path = torch.where(path < T, path, -1)
    token = tgt.gather(1, path.gather(1, count[:, None] - 1))[:, 0]
    ls = s["lengths"].long()
    src = ls[:, None] + torch.where(path >= 0, path, node)                    # dropped rows stay
    dst = ls[:, None] + node
    rows = src[None, :, None, :, None].expand(N, B, kv, T, hd)
    to = dst[None, :, None, :, None].expand(N, B, kv, T, hd)
    kc.scatter_(3, to, kc.gather(3, rows))
    vc.scatter_(3, to, vc.gather(3, rows))
    one, at = (x[None, :, None, :].expand(N, B, kv, T) for x in (src, dst))
    kept = (path >= 0)[None, :, None, :]
    s["weight"].scatter_(3, at, torch.where(kept, s["weight"].gather(3, one), 0))
    num = (s["seen"][:, None] + node)[None, :, None, :].int()
    s["positions"].scatter_(3, at, torch.where(kept, num, -1).expand(N, B, kv, T))
    return dict(path=path.int(), count=count.int(), token=token, k_cache=kc, v_cache=vc, weight=s["weight"],
                positions=s["positions"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    return _exact_evict(s, case) if case["op"] == "evict" else _exact_commit(s)


def _exact_attention(s):
    """One sequence at a time: softmax over the cached keys followed by the new ones, in 64 bits."""
    q, T = s["q"].double(), s["q"].shape[1]
    kv = s["k_cache"].shape[1]
    group = q.shape[2] // kv
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    weight = None if s["weight"] is None else s["weight"].double()
    causal = torch.ones(T, T, device=q.device).tril() > 0
    for b, n in enumerate(s["lengths"].tolist()):
        see = torch.cat([torch.ones(T, n, dtype=torch.bool, device=q.device),
                         causal if s["mask"] is None else s["mask"][b]], 1)
        for h in range(kv):
            k = torch.cat([s["k_cache"][b, h, :n], s["k_new"][b, :, h]]).double()
            v = torch.cat([s["v_cache"][b, h, :n], s["v_new"][b, :, h]]).double()
            for g in range(h * group, (h + 1) * group):
                x = torch.einsum("td,kd->tk", q[b, :, g], k) / math.sqrt(q.shape[-1])
                p = torch.softmax(x.masked_fill(~see, float("-inf")), -1)
                o[b, :, g] = torch.einsum("tk,kd->td", p, v)
                if weight is not None:
                    weight[b, h, :n + T] += p.sum(0)
    return dict(o=o, k_cache=None, v_cache=None, weight=weight, positions=None)


def _exact_evict(s, c):
    """One head at a time: the kept slots from their sorted list, survivors moved by hand."""
    W, P = s["weight"].double().cpu(), s["positions"].cpu()
    ls, seen = s["lengths"].tolist(), s["seen"].tolist()
    if W.numel() > 5e7 or W[..., 0].numel() > 10000:            # longer than some 20 seconds
        return None
    w2, p2 = torch.zeros_like(W), torch.full_like(P, -1)
    for u in range(W[..., 0].numel()):
        a, b = divmod(u, W.shape[1] * W.shape[2])
        b, h = divmod(b, W.shape[2])
        n, w, p = ls[b], W[a, b, h], P[a, b, h]
        m = min(n, c["keep"])
        first = ((p[:n] >= seen[b] - c["recent"]) | (p[:n] < c["sinks"])).to(torch.float64)
        key = torch.where(first > 0, torch.full_like(w[:n], 1e300), w[:n])
        best = torch.argsort(-key, stable=True)[:m]
        inside, outside = best[best < m], best[best >= m].sort().values
        free = torch.ones(m, dtype=torch.bool)
        free[inside] = False
        at = torch.arange(m)
        at[free.nonzero()[:, 0]] = outside
        w2[a, b, h, :m], p2[a, b, h, :m] = w[at], p[at]
    return dict(k_cache=None, v_cache=None, weight=w2.cuda(), positions=p2.cuda(),
                lengths=s["lengths"].clamp_max(c["keep"]))


def _exact_commit(s):
    """The walk down each tree, one node at a time; the weights of the rows that move."""
    par, tok, tgt = (s[k].tolist() for k in ("parents", "tokens", "targets"))
    weight, T = s["weight"].double(), len(tok[0])
    for b, n in enumerate(s["lengths"].tolist()):
        path, at = [0], 0
        while at is not None:
            at = next((i for i in range(1, T) if par[b][i] == path[-1] and tok[b][i] == tgt[b][path[-1]]), None)
            path += [] if at is None else [at]
        was = weight[:, b, :, n:n + T].clone()
        weight[:, b, :, n:n + T] = 0
        weight[:, b, :, n:n + len(path)] = was[:, :, path]
    return dict(path=None, count=None, token=None, k_cache=None, v_cache=None, weight=weight, positions=None)
