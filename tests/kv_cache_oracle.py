"""64-bit restatements of the cache operators, one sequence and head at a time, and the inputs their tests share."""
import torch

# unit roundoffs.  A 16-bit output is rounded once, and the probabilities may be rounded once to the same type before
# the second product: two relative errors of at most u each, so 2 u bounds the error's norm.  In float32 a score is
# hd <= 512 products of unit variance, scaled: its error is below sqrt(512) u 8 ~ 200 u for scores up to 8 in base 2,
# and p's relative error is the score's absolute one; 300 u covers the sums over the keys.
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def tolerance(dtype):
    return 300 * U[dtype] if dtype == torch.float32 else 2 * U[dtype]


# weights are sums of float32 probabilities whatever the cache's type
WEIGHT_TOL = 300 * 2.0 ** -24


def attention(q, k_new, v_new, kc, vc, lengths, mask, scale):
    """-> (o, weights added) in float64; lengths within the cache."""
    B, T, nh, hd = q.shape
    nkv, S = kc.shape[1], kc.shape[2]
    g = nh // nkv
    o = torch.zeros(B, T, nh, hd, dtype=torch.float64, device=q.device)
    w = torch.zeros(B, nkv, S + T, dtype=torch.float64, device=q.device)
    causal = torch.ones(T, T, device=q.device).tril() > 0
    for b in range(B):
        n = int(lengths[b])
        new = causal if mask is None else mask if mask.dim() == 2 else mask[b if mask.shape[0] > 1 else 0]
        see = torch.cat([torch.ones(T, n, dtype=torch.bool, device=q.device), new], 1)
        for h in range(nkv):
            k = torch.cat([kc[b, h, :n], k_new[b, :, h]]).double()
            v = torch.cat([vc[b, h, :n], v_new[b, :, h]]).double()
            for a in range(h * g, (h + 1) * g):
                s = (q[b, :, a].double() @ k.T * scale).masked_fill(~see, float("-inf"))
                e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)).masked_fill(~see, 0.0)
                p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
                o[b, :, a] = p @ v
                w[b, h, :n + T] += p.sum(0)
    return o, w[..., :S]


def evict(w, pos, n, seen, keep, recent, sinks):
    """One head -> (kept slots behind their new places, as a list: source of every new slot)."""
    key = []
    for i in range(n):
        held = pos[i] >= seen - recent or pos[i] < sinks
        key.append((2, 0.0) if held else (1, 0.0) if w[i] != w[i] else (0, w[i]))
    best = sorted(range(n), key=lambda i: (-key[i][0], -key[i][1], i))[:min(n, keep)]
    m, kept = len(best), set(best)
    src, movers = list(range(m)), sorted(i for i in best if i >= m)
    for hole in range(m):
        if hole not in kept:
            src[hole] = movers.pop(0)
    assert not movers
    return src


def random_tree(T, gen, chain=0.5):
    par = [-1]
    for i in range(1, T):
        near = torch.rand(1, generator=gen).item() < chain
        par.append(i - 1 if near else int(torch.randint(0, i, (1,), generator=gen)))
    return torch.tensor(par, dtype=torch.int32)


def rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()
