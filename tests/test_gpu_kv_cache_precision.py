"""What the cached attention of a 16-bit cache may lose: against 64-bit loops, next to the rounding of the output itself."""
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
