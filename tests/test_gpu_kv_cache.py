"""The cache kernels (csrc/kv_attention*.cu, csrc/kv_evict.cu) against 64-bit loops: element types, head
layouts, lengths from none to long, tiles that end early, masks that leave a row empty, stale NaN behind
the cached tokens, strided and huge caches, streams and graphs."""
import pytest
import torch

import kv_cache_oracle as K

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(seed, B, T, nh, nkv, hd, S, lengths, dtype, mask="causal", layout="heads"):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g).to("cuda").to(dtype)

    qkv = rand(B, T, nh + 2 * nkv, hd)
    q, kn, vn = qkv.split([nh, nkv, nkv], 2)
    if layout == "heads":
        kc, vc = rand(B, nkv, S, hd), rand(B, nkv, S, hd)
    elif layout == "tokens":                     # [B, S, nkv, hd] seen as [B, nkv, S, hd], K and V interleaved
        kv = rand(B, S, 2, nkv, hd)
        kc, vc = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    else:                                        # rows that start at odd elements
        kc, vc = rand(B, nkv, S, hd + 3)[..., 1:hd + 1], rand(B, nkv, S, hd + 1)[..., :hd]
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if mask == "causal":
        m = None
    elif mask == "tree":
        from sigma0_b200.ops.kv_cache import tree_mask
        m = torch.stack([tree_mask(K.random_tree(T, g)) for _ in range(B)]).cuda()
    elif mask == "shared":
        from sigma0_b200.ops.kv_cache import tree_mask
        m = tree_mask(K.random_tree(T, g)).cuda()
    else:                                        # rows that see no new token, not even themselves
        m = (torch.rand(B, T, T, generator=g) < 0.4).cuda()
        m[:, T // 2] = False
    for b, n in enumerate(lengths):              # what an earlier step left behind is never read
        kc[b, :, n:] = float("nan")
        vc[b, :, n:] = float("nan")
    return q, kn, vn, kc, vc, ls, m


def _check(args, dtype, lengths, weights=True, scale=None):
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, ls, m = args
    B, T, nh, hd = q.shape
    nkv, S = kc.shape[1], kc.shape[2]
    o64, w64 = K.attention(q, kn, vn, kc, vc, lengths, m, hd ** -0.5 if scale is None else scale)
    w = torch.rand(B, nkv, S, device="cuda") if weights else None
    pos = torch.full((B, nkv, S), -1, dtype=torch.int32, device="cuda") if weights else None
    w0, k0, v0 = None if w is None else w.clone(), kc.clone(), vc.clone()
    o = cache_attention(q, kn, vn, kc, vc, ls, mask=m, weight=w, positions=pos, seen=ls + 5 if weights else None, scale=scale)
    assert o.shape == q.shape and o.dtype == dtype and o.is_contiguous()
    assert torch.isfinite(o).all()
    assert K.rel(o, o64) < K.tolerance(dtype), K.rel(o, o64)
    # every row by itself: a lost row or head hides in the norm of all
    # (a row's error is bounded like the whole's; a dot product of few terms can be off by twice that)
    d = (o.double() - o64).norm(dim=-1) / o64.norm(dim=-1).clamp_min(1e-12)
    assert (d * (o64.norm(dim=-1) > 1e-9)).max() < 2 * K.tolerance(dtype), d.max()
    for b, n in enumerate(lengths):
        fit = max(0, min(T, S - n))
        assert torch.equal(kc[b, :, :n], k0[b, :, :n]) and torch.equal(vc[b, :, :n], v0[b, :, :n])
        assert torch.equal(kc[b, :, n:n + fit], kn[b, :fit].transpose(0, 1))
        assert torch.equal(vc[b, :, n:n + fit], vn[b, :fit].transpose(0, 1))
        assert torch.isnan(kc[b, :, n + fit:]).all() and torch.isnan(vc[b, :, n + fit:]).all()
        if weights:
            got, want = w[b].double() - 0, w0[b].double() + w64[b]
            assert K.rel(got[:, :n + fit], want[:, :n + fit]) < K.WEIGHT_TOL if n + fit else True
            assert torch.equal(w[b, :, n + fit:], w0[b, :, n + fit:])
            assert (pos[b, :, :n] == -1).all() and (pos[b, :, n + fit:] == -1).all()
            assert (pos[b, :, n:n + fit] == torch.arange(n + 5, n + 5 + fit, device="cuda")).all()
    return o


SHAPES = [  # B, T, nh, nkv, hd, S, lengths, mask
    (1, 1, 16, 16, 64, 500, [440], "causal"),
    (5, 1, 4, 4, 128, 1300, [0, 1, 63, 64, 1299], "causal"),
    (3, 1, 8, 2, 128, 700, [699, 128, 15], "causal"),
    (2, 1, 64, 1, 64, 300, [299, 17], "causal"),              # one key head for all
    (1, 1, 1, 1, 128, 20000, [19990], "causal"),              # one unit over many CTAs
    (4, 7, 6, 2, 64, 260, [0, 33, 128, 250], "tree"),
    (2, 22, 16, 16, 64, 600, [570, 1], "causal"),
    (2, 61, 16, 4, 128, 500, [0, 411], "tree"),
    (1, 64, 2, 2, 128, 4000, [3900], "shared"),
    (3, 16, 4, 4, 64, 200, [0, 100, 5], "holes"),             # rows that see nothing at all
    (2, 130, 4, 2, 64, 400, [129, 200], "tree"),              # more new tokens than a tile has rows or keys
    (2, 33, 3, 3, 40, 150, [100, 64], "tree"),                # a head narrower than the tensor-core tiles
    (1, 5, 1, 1, 503, 90, [80], "causal"),                    # one odd head
    (2, 3, 2, 2, 8, 50, [40, 0], "causal"),
    (2, 2, 2, 1, 512, 70, [65, 3], "causal"),
    (33, 1, 2, 2, 64, 90, list(range(0, 66, 2)), "causal"),   # one tile each
    (2, 9, 2, 2, 96, 0, [0, 0], "tree"),                      # no slots at all
    (2, 1000, 1, 1, 64, 1100, [7, 100], "causal"),
]


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"B{s[0]}T{s[1]}h{s[2]}.{s[3]}d{s[4]}S{s[5]}{s[7]}")
def test_attention(shape, dtype):
    B, T, nh, nkv, hd, S, lengths, mask = shape
    args = _case(B * 1000 + T + hd, B, T, nh, nkv, hd, S, lengths, dtype, mask)
    _check(args, dtype, lengths)
    _check(args, dtype, lengths, weights=False, scale=0.2)


@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,hd", [(1, 64), (20, 128)])
def test_attention_layouts(layout, dtype, T, hd):
    args = _case(T + hd, 2, T, 6, 3, hd, 200, [70, 128], dtype, "tree", layout)
    _check(args, dtype, [70, 128])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_past_the_last_slot_and_lengths_outside(dtype):
    """Rows that do not fit are attended to and dropped; a length outside the cache is one at its end."""
    args = _case(5, 3, 6, 2, 2, 64, 50, [46, 50, 0], dtype, "tree")
    _check(args, dtype, [46, 50, 0])
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, _, m = _case(6, 2, 6, 2, 2, 64, 50, [50, 0], dtype, "tree")
    o64, _ = K.attention(q, kn, vn, kc, vc, [50, 0], m, 64 ** -0.5)
    o = cache_attention(q, kn, vn, kc, vc, torch.tensor([5000, -3], dtype=torch.int32, device="cuda"), mask=m)
    assert K.rel(o, o64) < K.tolerance(dtype)


def test_attention_large_scores_and_infinities():
    """Scores far apart leave one key; an infinite or NaN key shows in the rows that see it and in no other."""
    from sigma0_b200.ops.kv_cache import cache_attention
    for dtype in (BF, F32):
        q, kn, vn, kc, vc, ls, m = _case(9, 2, 4, 2, 2, 64, 100, [90, 30], dtype, "tree")
        o64, _ = K.attention(q * 50, kn, vn, kc, vc, [90, 30], m, 1.0)
        o = cache_attention(q * 50, kn, vn, kc, vc, ls, mask=m, scale=1.0)
        # float32 scores around 400 carry an error of 400 2^-24 each, the exact products of 16-bit inputs as well
        assert K.rel(o, o64) < 2 * K.tolerance(dtype) + 2e-4
        kc[1, 0, 3, 5] = float("nan")
        o = cache_attention(q, kn, vn, kc, vc, ls, mask=m)
        assert torch.isnan(o[1, :, 0]).all() and torch.isfinite(o[0]).all() and torch.isfinite(o[1, :, 1]).all()
        # a new token that a row does not see
        q, kn, vn, kc, vc, ls, m = _case(10, 1, 3, 1, 1, 64, 100, [90], dtype, "causal")
        kn[0, 2, 0, 1], vn[0, 2, 0, 1] = float("inf"), float("nan")
        o = cache_attention(q, kn, vn, kc, vc, ls)
        assert torch.isfinite(o[0, :2]).all() and torch.isnan(o[0, 2]).any()


def test_attention_offsets_past_32_bits():
    """Slots that lie more than 2^31 elements apart."""
    from sigma0_b200.ops.kv_cache import cache_attention
    B, nkv, S, hd, far = 1, 2, 600, 64, 1 << 22
    buf = torch.empty(far * S, dtype=BF, device="cuda")
    kc = buf.as_strided((B, nkv, S, hd), (far * S, hd, far, 1))
    vc = buf.as_strided((B, nkv, S, hd), (far * S, hd, far, 1), storage_offset=4096)
    q, kn, vn, k1, v1, ls, m = _case(11, B, 3, 4, nkv, hd, S, [590], BF, "tree")
    kc.copy_(k1)
    vc.copy_(v1)
    o64, _ = K.attention(q, kn, vn, kc, vc, [590], m, hd ** -0.5)
    o = cache_attention(q, kn, vn, kc, vc, ls, mask=m)
    assert K.rel(o, o64) < K.tolerance(BF)
    assert torch.equal(kc[0, :, 590:593], kn[0].transpose(0, 1)) and torch.equal(vc[0, :, 590:593], vn[0].transpose(0, 1))


def test_attention_is_reproducible_on_streams_and_in_graphs():
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, ls, m = _case(12, 3, 9, 8, 4, 128, 3000, [2900, 100, 1500], BF, "tree")
    w = torch.zeros(3, 4, 3000, device="cuda")
    o = cache_attention(q, kn, vn, kc, vc, ls, mask=m, weight=w)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        w2 = torch.zeros_like(w)
        o2 = cache_attention(q, kn, vn, kc, vc, ls, mask=m, weight=w2)
    st.synchronize()
    assert torch.equal(o, o2) and torch.equal(w, w2)
    # a captured step follows the lengths on the device
    w3 = torch.zeros_like(w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o3 = cache_attention(q, kn, vn, kc, vc, ls, mask=m, weight=w3)
    ls.copy_(torch.tensor([17, 2000, 0], dtype=torch.int32))
    kc.normal_()
    vc.normal_()
    w3.zero_()
    g.replay()
    torch.cuda.synchronize()
    o64, w64 = K.attention(q, kn, vn, kc, vc, [17, 2000, 0], m, 128 ** -0.5)
    assert K.rel(o3, o64) < K.tolerance(BF) and K.rel(w3, w64) < K.WEIGHT_TOL


def test_attention_runs_the_kernel():
    from sigma0_b200.ops import _ext
    q, kn, vn, kc, vc, ls, m = _case(13, 1, 1, 2, 2, 64, 100, [90], BF)
    from sigma0_b200.ops.kv_cache import cache_attention
    _ext.reset_launch_count()
    cache_attention(q, kn, vn, kc, vc, ls)
    assert _ext.launch_count() > 0


def test_attention_refusals():
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, ls, m = _case(14, 2, 3, 4, 2, 64, 50, [40, 30], BF, "tree")
    w = torch.zeros(2, 2, 50, device="cuda")
    bad = [
        dict(q=q[:, :, :3]), dict(q=q.float()), dict(q=q[:1]), dict(kn=kn[:, :2]), dict(vn=vn.half()), dict(kc=kc.float()),
        dict(kc=kc[:, :, :40]), dict(ls=ls.long()), dict(ls=ls[:1]), dict(ls=ls.cpu()), dict(m=m.float()), dict(m=m[:, :2]),
        dict(m=m[:, :, :2]), dict(kc=kc.transpose(2, 3), vc=vc.transpose(2, 3)), dict(weight=w.half()), dict(weight=w[:, :, :49]),
        dict(positions=w.int()), dict(positions=w, seen=ls), dict(q=q.cpu()), dict(q=q.double(), kn=kn.double(), vn=vn.double(), kc=kc.double(), vc=vc.double()),
    ]
    for d in bad:
        a = dict(q=q, kn=kn, vn=vn, kc=kc, vc=vc, ls=ls, m=m) | d
        with pytest.raises(RuntimeError):
            cache_attention(a["q"], a["kn"], a["vn"], a["kc"], a["vc"], a["ls"], mask=a["m"], weight=a.get("weight"),
                            positions=a.get("positions"), seen=a.get("seen"))
    wide = torch.zeros(1, 1, 1, 513, device="cuda")
    with pytest.raises(RuntimeError):
        cache_attention(wide, wide, wide, wide, wide.clone(), ls[:1])
    with pytest.raises(RuntimeError):
        cache_attention(q.detach().requires_grad_(True), kn, vn, kc, vc, ls)
    assert cache_attention(q[:0], kn[:0], vn[:0], kc[:0], vc[:0], ls[:0]).shape == (0, 3, 4, 64)


# ---- eviction -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (F32, 40), (FH, 503), (BF, 6)])
@pytest.mark.parametrize("S,lengths,keep,recent,sinks", [
    (40, [40, 33, 7, 0], 16, 4, 2),
    (1500, [1500, 700, 1024, 513], 512, 100, 4),
    (1100, [1100, 1, 600, 601], 600, 600, 0),       # every survivor is recent
    (300, [300, 299, 298, 2], 1, 0, 0),
    (64, [64, 64, 64, 64], 500, 20, 4),             # a budget that nothing reaches
    (5000, [5000, 4097, 4999, 4100], 4096, 10, 3),
])
def test_evict(dtype, hd, S, lengths, keep, recent, sinks):
    from sigma0_b200.ops.kv_cache import cache_evict
    g = torch.Generator().manual_seed(S + keep)
    N, B, nkv = 2, len(lengths), 2
    kc, vc = (torch.randn(N, B, nkv, S, hd, generator=g).to("cuda").to(dtype) for _ in range(2))
    w = torch.randn(N, B, nkv, S, generator=g).mul_(2).exp_()
    w = torch.where(w < 1, (w * 4).floor() / 4, w)
    w[0, 0, 0, :3], w[1, 0, 1, 2], w[0, 1, 0, 1] = float("nan"), float("inf"), -0.0
    pos = torch.rand(N, B, nkv, S, generator=g).argsort(-1).int() + 50
    pos[..., :1] = 0
    ls = torch.tensor(lengths, dtype=torch.int32)
    seen = ls + 50
    dev = [x.cuda() for x in (w, pos, ls, seen)]
    k0, v0 = kc.cpu().clone(), vc.cpu().clone()
    w2, p2, l2 = cache_evict(kc, vc, *dev, keep, recent, sinks)
    assert l2.tolist() == [min(n, keep) for n in lengths]
    kc, vc, w2, p2 = kc.cpu(), vc.cpu(), w2.cpu(), p2.cpu()
    for n in range(N):
        for b in range(B):
            for h in range(nkv):
                src = K.evict(w[n, b, h].tolist(), pos[n, b, h].tolist(), lengths[b], lengths[b] + 50, keep, recent, sinks)
                m = len(src)
                assert torch.equal(p2[n, b, h, :m], pos[n, b, h, src]) and (p2[n, b, h, m:] == -1).all()
                assert torch.equal(w2[n, b, h, :m].view(torch.int32), w[n, b, h, src].view(torch.int32)) and (w2[n, b, h, m:] == 0).all()
                assert torch.equal(kc[n, b, h, :m], k0[n, b, h, src]) and torch.equal(vc[n, b, h, :m], v0[n, b, h, src])
                assert torch.equal(kc[n, b, h, m:], k0[n, b, h, m:]) and torch.equal(vc[n, b, h, m:], v0[n, b, h, m:])


def test_evict_in_place_in_a_graph_and_strided():
    from sigma0_b200.ops.kv_cache import cache_evict
    g = torch.Generator().manual_seed(4)
    N, B, nkv, S, hd = 3, 2, 4, 900, 64
    kv = torch.randn(N, B, S, 2, nkv, hd, generator=g).cuda().to(BF)
    kc, vc = kv[:, :, :, 0].transpose(2, 3), kv[:, :, :, 1].transpose(2, 3)
    w = torch.rand(N, B, nkv, S, generator=g).cuda()
    pos = torch.arange(S, dtype=torch.int32).expand(N, B, nkv, S).contiguous().cuda()
    ls = torch.tensor([900, 450], dtype=torch.int32, device="cuda")
    seen = ls.clone()
    k1, v1 = kc.clone(), vc.clone()
    want = cache_evict(k1, v1, w, pos, ls, seen, 300, 64, 4)
    saved = [x.clone() for x in (kv, w, pos, ls)]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = cache_evict(kc, vc, w, pos, ls, seen, 300, 64, 4, out=(w, pos, ls))
    for x, y in zip((kv, w, pos, ls), saved):
        x.copy_(y)
    gr.replay()
    torch.cuda.synchronize()
    assert got[0] is w and all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(kc, k1) and torch.equal(vc, v1)
    # once more: nothing is over the budget now
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kc, k1)


def test_evict_refusals():
    from sigma0_b200.ops.kv_cache import cache_evict
    kc, vc = torch.zeros(1, 2, 8, 4, device="cuda"), torch.zeros(1, 2, 8, 4, device="cuda")
    w, pos = torch.zeros(1, 2, 8, device="cuda"), torch.zeros(1, 2, 8, dtype=torch.int32, device="cuda")
    ls = torch.zeros(1, dtype=torch.int32, device="cuda")
    for a in [(kc, vc, w, pos, ls, ls, 0), (kc, vc, w, pos, ls, ls, 4, 4, 1), (kc, vc, w, pos, ls, ls, 4, -1),
              (kc, vc.half(), w, pos, ls, ls, 4), (kc, vc[:, :, :7], w, pos, ls, ls, 4), (kc, vc, w.double(), pos, ls, ls, 4),
              (kc, vc, w, pos.long(), ls, ls, 4), (kc, vc, w, pos, ls.long(), ls, 4), (kc, vc, w[:, :, ::2], pos[:, :, ::2], ls, ls, 4)]:
        with pytest.raises(RuntimeError):
            cache_evict(*a)


# ---- acceptance of drafts -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype,hd,layout", [(BF, 64, "heads"), (F32, 503, "heads"), (FH, 40, "tokens"), (BF, 7, "heads")])
@pytest.mark.parametrize("T,share", [(1, False), (2, False), (8, True), (33, False), (64, False), (200, False), (1024, True)])
def test_commit(dtype, hd, layout, T, share):
    from sigma0_b200.ops.kv_cache import tree_commit
    g = torch.Generator().manual_seed(T + hd)
    N, B, nkv, S = 2, 3, 3, T + 60
    if layout == "heads":
        kc, vc = (torch.randn(N, B, nkv, S, hd, generator=g).to("cuda").to(dtype) for _ in range(2))
    else:
        kv = torch.randn(N, B, S, 2, nkv, hd, generator=g).to("cuda").to(dtype)
        kc, vc = kv[:, :, :, 0].transpose(2, 3), kv[:, :, :, 1].transpose(2, 3)
    par = K.random_tree(T, g, 0.7) if share else torch.stack([K.random_tree(T, g, 0.9) for _ in range(B)])
    tgt = torch.randint(0, 3, (B, T), generator=g)                   # few tokens: long paths, equal siblings
    said = tgt.gather(1, par.expand(B, T).long().clamp_min(0))
    tok = torch.where(torch.rand(B, T, generator=g) < 0.95, said, torch.randint(0, 3, (B, T), generator=g))
    ls = torch.tensor([0, 17, 60], dtype=torch.int32)
    ls[2] = S - T // 2                                               # half of its nodes are past the last slot
    seen = ls + 9
    w, pos = torch.rand(N, B, nkv, S, generator=g), torch.randint(0, 99, (N, B, nkv, S), generator=g).int()
    from sigma0_b200.ops.kv_cache import tree_commit as commit
    host = [x.cpu().clone() for x in (kc, vc, w, pos)]
    want = commit(par, tok, tgt, host[0], host[1], ls, weight=host[2], positions=host[3], seen=seen)
    dw, dp = w.cuda(), pos.cuda()
    got = tree_commit(par.cuda(), tok.cuda(), tgt.cuda(), kc, vc, ls.cuda(), weight=dw, positions=dp, seen=seen.cuda())
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    for a, b in zip((kc, vc, dw, dp), host):
        assert torch.equal(a.cpu(), b)
    if T == 33:
        assert max(want[1].tolist()) > 3                             # the inputs do move rows


def test_commit_refusals_and_foreign_parents():
    from sigma0_b200.ops.kv_cache import tree_commit
    kc, vc = torch.zeros(1, 2, 8, 4, device="cuda"), torch.zeros(1, 2, 8, 4, device="cuda")
    ls = torch.zeros(1, dtype=torch.int32, device="cuda")
    par = torch.tensor([-1, 0, 1], dtype=torch.int32, device="cuda")
    t = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    for a in [(par.long(), t, t, kc, vc, ls), (par[:2], t, t, kc, vc, ls), (par, t.int(), t, kc, vc, ls), (par, t, t[:, :2], kc, vc, ls),
              (par, t, t, kc, vc.half(), ls), (par, t, t, kc, vc, ls.long()), (par[:0], t[:, :0], t[:, :0], kc, vc, ls)]:
        with pytest.raises(RuntimeError):
            tree_commit(*a)
    # parents that do not lie below their children, or are no node at all, are never reached
    odd = torch.tensor([0, 2, 77], dtype=torch.int32, device="cuda")
    path, count, token = tree_commit(odd, t, t, kc, vc, ls)
    assert path.tolist() == [[0, -1, -1]] and count.tolist() == [1] and token.tolist() == [0]
