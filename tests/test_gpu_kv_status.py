"""The status word of the tcgen05 cache attention."""
import os
import subprocess
import sys

import pytest

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
