"""More than 16 rows over a 16-bit cache: new tokens that are not finite, head sizes between 64 and 128, huge strides."""
import pytest
import torch

import kv_cache_oracle as K

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


def _case(seed, B, T, nh, nkv, hd, S, dtype):
    g = torch.Generator().manual_seed(seed)
    q, kn, vn = (torch.randn(B, T, n, hd, generator=g).to("cuda", dtype) for n in (nh, nkv, nkv))
    kc, vc = (torch.randn(B, nkv, S, hd, generator=g).to("cuda", dtype) for _ in range(2))
    from sigma0_b200.ops.kv_cache import tree_mask
    return q, kn, vn, kc, vc, torch.stack([tree_mask(K.random_tree(T, g)) for _ in range(B)]).cuda()


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T,nh,nkv,hd,S,lengths", [
    (40, 2, 2, 64, 300, [200, 0]),
    (40, 2, 2, 128, 300, [200, 0]),
    (20, 4, 2, 104, 150, [130, 1]),              # 40 rows; a head narrower than the tile
    (130, 2, 1, 64, 400, [129, 270]),            # 260 rows, two tiles of new tokens
    (130, 2, 2, 128, 30000, [29000, 5000]),      # units of several CTAs
    (5, 2, 2, 64, 300, [200, 0]),                # few rows
])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_new_tokens_that_are_not_finite(T, nh, nkv, hd, S, lengths, dtype, value):
    """What is not finite in the value (or the key) of a new token shows in the rows that see it, and the others are as without it."""
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, m = _case(T + hd, 2, T, nh, nkv, hd, S, dtype)
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o64, w64 = K.attention(q, kn, vn, kc, vc, lengths, m, hd ** -0.5)
    bad = [(0, T - 1, 0, 3), (0, T // 2, nkv - 1, hd - 1), (1, T // 3, 0, 0), (1, T // 3, 0, hd // 2)]   # book, token, head, channel
    g = nh // nkv
    # in a value: its channel of the rows that see it
    vbad, want, hit = vn.clone(), o64.clone(), torch.zeros_like(o64, dtype=torch.bool)
    for b, t, h, d in bad:
        vbad[b, t, h, d] = value
        hit[b, :, h * g:(h + 1) * g, d] |= m[b, :, t][:, None]
    w = torch.zeros(2, nkv, S, device="cuda")
    o = cache_attention(q, kn, vbad, kc.clone(), vc.clone(), ls, mask=m, weight=w)
    assert (torch.isnan(o[hit]).all() if value != value else (o[hit] == value).all())
    assert torch.isfinite(o[~hit]).all()
    assert K.rel(o.double().masked_fill(hit, 0), want.masked_fill(hit, 0)) < K.tolerance(dtype)
    assert K.rel(w, w64) < K.WEIGHT_TOL                      # the weights do not depend on values
    # in a key: whole rows that see it
    kbad, hit = kn.clone(), torch.zeros_like(hit)
    for b, t, h, d in bad:
        kbad[b, t, h, d] = float("nan")
        hit[b, :, h * g:(h + 1) * g] |= m[b, :, t][:, None, None]
    o = cache_attention(q, kbad, vn, kc.clone(), vc.clone(), ls, mask=m)
    assert torch.isnan(o[hit]).all() and torch.isfinite(o[~hit]).all()
    assert K.rel(o.double().masked_fill(hit, 0), want.masked_fill(hit, 0)) < K.tolerance(dtype)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("hd", [8, 56, 72, 80, 96, 120])
@pytest.mark.parametrize("T,nh,nkv,S,lengths", [(24, 2, 2, 400, [370, 0, 129]), (9, 8, 2, 2100, [2090, 1000, 77]), (200, 3, 1, 500, [128, 300, 5])])
def test_head_sizes(T, nh, nkv, S, lengths, hd, dtype):
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc, m = _case(T + hd, 3, T, nh, nkv, hd, S, dtype)
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths):
        kc[b, :, n:], vc[b, :, n:] = float("nan"), float("nan")
    o64, w64 = K.attention(q, kn, vn, kc, vc, lengths, m, hd ** -0.5)
    w = torch.zeros(3, nkv, S, device="cuda")
    o = cache_attention(q, kn, vn, kc, vc, ls, mask=m, weight=w)
    assert K.rel(o, o64) < K.tolerance(dtype) and K.rel(w, w64) < K.WEIGHT_TOL
    d = (o.double() - o64).norm(dim=-1) / o64.norm(dim=-1)
    assert d.max() < 2 * K.tolerance(dtype)
    for b, n in enumerate(lengths):
        assert torch.equal(kc[b, :, n:n + T], kn[b].transpose(0, 1)) and torch.equal(vc[b, :, n:n + T], vn[b].transpose(0, 1))


@pytest.mark.parametrize("T", [20, 130])
def test_offsets_past_32_bits(T):
    """Slots and queries that lie more than 2^31 elements apart."""
    from sigma0_b200.ops.kv_cache import cache_attention
    nkv, S, hd, far = 2, 600, 64, 1 << 22
    buf = torch.empty(far * S, dtype=BF, device="cuda")
    kc = buf.as_strided((1, nkv, S, hd), (far * S, hd, far, 1))
    vc = buf.as_strided((1, nkv, S, hd), (far * S, hd, far, 1), storage_offset=4096)
    q, kn, vn, k1, v1, m = _case(T, 1, T, 4, nkv, hd, S, BF)
    kc.copy_(k1)
    vc.copy_(v1)
    n = S - T
    # at 130 rows: q of the last token more than 2^31 elements behind the first
    qbuf = buf.as_strided(q.shape, (far * S, far * 4, hd, 1), storage_offset=8192)
    qbuf.copy_(q)
    o64, _ = K.attention(q, kn, vn, kc, vc, [n], m, hd ** -0.5)
    o = cache_attention(qbuf, kn, vn, kc, vc, torch.tensor([n], dtype=torch.int32, device="cuda"), mask=m)
    assert K.rel(o, o64) < K.tolerance(BF)
    assert torch.equal(kc[0, :, n:], kn[0].transpose(0, 1)) and torch.equal(vc[0, :, n:], vn[0].transpose(0, 1))
