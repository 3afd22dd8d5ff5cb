"""The status word of the tcgen05 cache attention."""
import os
import subprocess
import sys

import pytest
import torch

import kv_cache_oracle as K

pytestmark = pytest.mark.gpu

FIRST_IN_A_CAPTURE = """
import torch
from sigma0_b200.ops import kv_cache as C
from sigma0_b200.ops._ext import ext
q = torch.randn(1, 40, 1, 64, device="cuda", dtype=torch.bfloat16)
kc, vc = (torch.randn(1, 1, 300, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
ls = torch.full((1,), 200, dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o = C.cache_attention(q, q, q, kc, vc, ls)
assert C.status(q) == 0, "set before anything ran"
ext().kv_status(q).fill_(1)                      # as a wait that ran out would
g.replay()
torch.cuda.synchronize()
assert C.status(q) == 1, "cleared by a replay"
ext().kv_status(q).zero_()
assert torch.equal(o, C.cache_attention(q, q, q, kc, vc, ls)) and C.status(q) == 0
print("as it should be")
"""


def test_a_first_call_inside_a_capture():
    """In a process of its own: the word is there before the call that a graph holds, and replays leave it alone."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as it should be" in r.stdout, r.stdout + r.stderr


@pytest.fixture
def no_waiting():
    """Every wait of the kernel gives up at once: nothing stays in flight, all roles leave, the GPU stays usable."""
    from sigma0_b200.ops import kv_cache as C
    C.wait_limit(0)
    yield
    C.wait_limit()
    torch.cuda.synchronize()
    C.ext().kv_status(torch.zeros(1, device="cuda")).zero_()


def _case(B, nkv, group, T, hd, S, dtype):
    g = torch.Generator().manual_seed(S)
    q, kn, vn = (torch.randn(B, T, n, hd, generator=g).to("cuda", dtype) for n in (nkv * group, nkv, nkv))
    kc, vc = (torch.randn(B, nkv, S, hd, generator=g).to("cuda", dtype) for _ in range(2))
    return q, kn, vn, kc, vc, torch.tensor([S - T - 3 * b for b in range(B)], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("B,nkv,group,T,hd,S,dtype", [
    (1, 2, 1, 40, 64, 5000, torch.bfloat16),     # units of several CTAs
    (4, 200, 1, 20, 64, 300, torch.float16),     # several units of a CTA
    (2, 3, 4, 30, 96, 900, torch.bfloat16),      # two row blocks
])
def test_a_wait_that_runs_out(no_waiting, B, nkv, group, T, hd, S, dtype, weights):
    from sigma0_b200.ops import kv_cache as C
    args = _case(B, nkv, group, T, hd, S, dtype)
    w = torch.zeros(B, nkv, S, device="cuda") if weights else None
    k0, v0 = args[3].clone(), args[4].clone()
    o = C.cache_attention(*args, weight=w)
    torch.cuda.synchronize()
    assert torch.isnan(o).all() and C.status(o) == 1
    with pytest.raises(RuntimeError, match="longer than its limit"):
        C.check(o)
    assert C.status(o) == 0
    C.check(o)
    if weights:
        for b, n in enumerate(args[5].tolist()):
            assert torch.isnan(w[b, :, :n + T]).all() and (w[b, :, n + T:] == 0).all()
    # the next call is none the worse for it
    C.wait_limit()
    got = C.cache_attention(args[0], args[1], args[2], k0, v0, args[5])
    want, _ = K.attention(args[0], args[1], args[2], k0, v0, args[5].tolist(), None, hd ** -0.5)
    assert K.rel(got, want) < K.tolerance(dtype) and C.status(o) == 0


def test_generation_says_so(no_waiting):
    from types import SimpleNamespace
    from sigma0_b200.infer.speculative import TreeDecoder, generate
    from sigma0_b200.models.registry import build_model
    from sigma0_b200.ops import kv_cache as C
    model = build_model(SimpleNamespace(architecture="transformer", d_model=128, n_heads=2, n_message_layers=1, n_layers=1, vocab_size=50,
                                        use_book_data=False, token_mode="22tok", dtype="bfloat16", impl="torch")).cuda().eval()
    prompt = torch.randint(0, 50, (2, 60), device="cuda")
    with pytest.raises(RuntimeError, match="longer than its limit"):
        generate(TreeDecoder(model, 2, 120), prompt, 10)
    C.wait_limit()
    assert generate(TreeDecoder(model, 2, 120), prompt, 10)[0].shape == (2, 10)


def test_limits():
    from sigma0_b200.ops import kv_cache as C
    for s in (-1, 61, float("nan")):
        with pytest.raises(RuntimeError):
            C.wait_limit(s)
