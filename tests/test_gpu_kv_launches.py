"""launch_count counts the kernels that the cache operators launch: a join or a mover only where there is one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _attention(S, n, T=1, weights=False, dtype=torch.bfloat16):
    from sigma0_b200.ops.kv_cache import cache_attention
    q = torch.zeros(1, T, 2, 64, device="cuda", dtype=dtype)
    kc = torch.zeros(1, 2, S, 64, device="cuda", dtype=dtype)
    w = torch.zeros(1, 2, S, device="cuda") if weights else None
    cache_attention(q, q, q, kc, kc.clone(), torch.tensor([n], dtype=torch.int32, device="cuda"), weight=w)


def _evict(units, in_place):
    from sigma0_b200.ops.kv_cache import cache_evict
    kc = torch.zeros(1, units, 8, 4, device="cuda")
    w, ls = torch.zeros(1, units, 8, device="cuda"), torch.full((1,), 8, dtype=torch.int32, device="cuda")
    cache_evict(kc, kc.clone(), w, w.int(), ls, ls.clone(), 4, out=(w, w.int(), ls) if in_place else None)


def _commit():
    from sigma0_b200.ops.kv_cache import tree_commit
    kc, t = torch.zeros(1, 2, 8, 4, device="cuda"), torch.zeros(1, 1, dtype=torch.long, device="cuda")
    tree_commit(torch.full((1,), -1, dtype=torch.int32, device="cuda"), t, t, kc, kc.clone(), torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("call,kernels", [
    (lambda: _attention(500, 400), 1),                       # one CTA per unit, no join
    (lambda: _attention(500, 400, weights=True), 2),
    (lambda: _attention(20000, 19000), 2),
    (lambda: _attention(500, 400, T=40), 2),
    (lambda: _attention(400, 300, dtype=torch.float32), 1),
    (lambda: _evict(2, False), 2),                           # few units: a second kernel moves the rows
    (lambda: _evict(400, False), 1),
    (lambda: _evict(400, True), 2),                          # lengths in place
    (_commit, 1),
])
def test_launches(call, kernels):
    from sigma0_b200.ops import _ext
    from sigma0_b200.ops.kv_cache import status
    call()
    _ext.reset_launch_count()
    call()
    assert _ext.launch_count() == kernels
    status(torch.zeros(1, device="cuda"))
    assert _ext.launch_count() == kernels
