"""What the cached attention of a 16-bit cache may lose: against 64-bit loops, next to the rounding of the output itself."""
import math

import pytest
import torch

import kv_cache_oracle as K

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


def _rand(seed, *shapes, dtype):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to("cuda").to(dtype) for s in shapes]


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("B,T,nh,nkv,hd,S,lengths", [
    (1, 1, 16, 16, 64, 500, [440]),
    (3, 1, 8, 2, 128, 700, [699, 128, 15]),
    (1, 1, 2, 2, 128, 20000, [19990]),           # one unit over several CTAs
    (2, 6, 4, 2, 64, 300, [250, 31]),            # twelve rows
    (2, 4, 8, 2, 96, 900, [890, 500]),           # sixteen
])
def test_up_to_16_rows_lose_the_output_rounding_only(B, T, nh, nkv, hd, S, lengths, dtype):
    """The products take the probabilities in two parts, 16 bits or more together, and sum in float32: beside the rounding of
    the output that leaves 2^-16 of its norm at most, and float32 sums of up to 20,000 terms another 2^-12 u."""
    from sigma0_b200.ops.kv_cache import cache_attention
    q, kn, vn, kc, vc = _rand(T * hd, (B, T, nh, hd), (B, T, nkv, hd), (B, T, nkv, hd), (B, nkv, S, hd), (B, nkv, S, hd), dtype=dtype)
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o64, _ = K.attention(q, kn, vn, kc, vc, lengths, None, hd ** -0.5)
    o = cache_attention(q, kn, vn, kc, vc, ls)
    assert K.rel(o, o64) < K.rel(o64.to(dtype), o64) + 2.0 ** -16 + 2.0 ** -12 * K.U[dtype]


@pytest.mark.parametrize("dtype", [FH, BF])
@pytest.mark.parametrize("T", [1, 12, 20])
@pytest.mark.parametrize("drop", [19.0, 25.2, 27.5, 30.0])
def test_one_dominant_token_beside_a_long_tail(T, drop, dtype):
    """Keys with 2^-drop of the largest probability each, 20,000 of them, and a largest one whose value is 0: the output is the tail's.

    The probabilities' absolute error is below 2^-36 of the largest each (fp16 keeps steps of 2^-24 and refers to 2^-11 of
    the largest; a bf16 one has a relative error only), and the outputs are rounded, below 2^-14 in fp16 to steps of 2^-24."""
    from sigma0_b200.ops.kv_cache import cache_attention
    # as many units as CTAs and more: most are walked by one of them
    B, nkv, hd, n = 2, 160, 64, 20000
    S = n + T
    kc = torch.zeros(B, nkv, S, hd, device="cuda", dtype=dtype)
    vc, = _rand(T, (B, nkv, S, hd), dtype=dtype)
    vc += 1
    kc[:, :, (0, 32, 64, 96), 0] = drop          # one in each warp's first keys
    vc[:, :, (0, 32, 64, 96)] = 0
    q = torch.zeros(B, T, nkv, hd, device="cuda", dtype=dtype)
    q[..., 0] = 8
    kn = torch.zeros_like(q)
    vn, = _rand(T + 1, q.shape, dtype=dtype)
    scale = math.log(2) / 8                      # scores of `drop` and 0 in base 2
    ls = torch.full((B,), n, dtype=torch.int32, device="cuda")
    o64, _ = K.attention(q, kn, vn, kc, vc, [n] * B, None, scale)
    o = cache_attention(q, kn, vn, kc, vc, ls, scale=scale).double()
    bound = 2 * K.U[dtype] * o64.abs()
    if dtype == FH:
        bound += 2.0 ** -25 + n * 2.0 ** -36 * 6  # |v| below 6
    assert ((o - o64).norm(dim=-1) <= bound.norm(dim=-1)).all(), ((o - o64).norm() / bound.norm()).item()


@pytest.mark.parametrize("dtype,e", [(BF, 4), (BF, 20), (BF, 52), (FH, 4), (FH, 15), (torch.float32, 20), (torch.float32, 52)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("T,n", [(1, 400), (1, 30000), (12, 3000), (40, 400), (40, 30000)])
def test_scores_of_any_size(T, n, sign, dtype, e):
    """Half of the keys have the score sign 2^(2 e + 3) exactly, the others one that is lower by 2^-7 of it or more: the output
    is the mean of the first half's values and their weights are equal, whatever the size of the scores."""
    from sigma0_b200.ops.kv_cache import cache_attention
    nkv, hd = 2, 64
    S = n + T
    q = torch.full((1, T, nkv, hd), 2.0 ** e, device="cuda", dtype=dtype)
    kc = torch.full((1, nkv, S, hd), sign * 2.0 ** e, device="cuda", dtype=dtype)
    kc[:, :, 1::2] = sign * 2.0 ** e * (1 - sign * 2.0 ** -7)
    kn = torch.full_like(q, sign * 2.0 ** e * (1 - sign * 2.0 ** -7))
    vc, vn = _rand(T, kc.shape, q.shape, dtype=dtype)
    ls = torch.tensor([n], dtype=torch.int32, device="cuda")
    o64, w64 = K.attention(q, kn, vn, kc, vc, [n], None, 0.125)
    w = torch.zeros(1, nkv, S, device="cuda")
    o = cache_attention(q, kn, vn, kc, vc, ls, scale=0.125, weight=w)
    assert K.rel(o, o64) < K.tolerance(dtype) and K.rel(w, w64) < K.WEIGHT_TOL
