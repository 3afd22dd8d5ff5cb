"""Decoding over a key / value cache: CUDA-event times of attention, eviction and tree commit.

``python -m sigma0_b200.eval.kv_bench --batch 64 --length 11000`` prints one JSON line per operator: the time
of a call, the bytes that it cannot do without and the rate that they make.  Inputs beyond L2 (the default is
2.9 GB) need no flush between calls.
"""
from __future__ import annotations

import argparse
import json

import torch

from ..infer.speculative import chain_tree
from ..ops.kv_cache import cache_attention, cache_evict, tree_commit, tree_mask


def _time(fn, iters):
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(iters):
        fn()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / iters * 1e-3


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--batch", type=int, default=64)
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--kv_heads", type=int, default=16)
    p.add_argument("--hd", type=int, default=64)
    p.add_argument("--length", type=int, default=11000)
    p.add_argument("--width", type=int, default=0, help="chains of the drafted tree (0: one token)")
    p.add_argument("--depth", type=int, default=7)
    p.add_argument("--keep", type=int, default=2048)
    p.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float16", "float32"])
    p.add_argument("--weights", action="store_true", help="add up the softmax weight per slot")
    p.add_argument("--iters", type=int, default=20)
    a = p.parse_args(argv)
    dt = getattr(torch, a.dtype)
    par = chain_tree(a.width, a.depth, "cuda")
    T, mask = par.numel(), tree_mask(par)
    B, nkv, hd, S = a.batch, a.kv_heads, a.hd, a.length + par.numel()
    kc, vc = (torch.randn(B, nkv, S, hd, device="cuda", dtype=dt) for _ in range(2))
    q = torch.randn(B, T, a.heads, hd, device="cuda", dtype=dt)
    kn, vn = (torch.randn(B, T, nkv, hd, device="cuda", dtype=dt) for _ in range(2))
    ls = torch.full((B,), a.length, dtype=torch.int32, device="cuda")
    w = torch.rand(B, nkv, S, device="cuda")
    pos = torch.arange(S, dtype=torch.int32, device="cuda").expand(B, nkv, S).contiguous()
    es, out = kc.element_size(), []

    def say(op, seconds, byt):
        out.append({"op": op, "us": round(seconds * 1e6, 2), "bytes": byt, "gbs": round(byt / seconds / 1e9, 1), "batch": B,
                    "heads": a.heads, "kv_heads": nkv, "hd": hd, "length": a.length, "nodes": T, "dtype": a.dtype})
        print(json.dumps(out[-1]))

    t = _time(lambda: cache_attention(q, kn, vn, kc, vc, ls, mask=mask, weight=w if a.weights else None), a.iters)
    say("attention", t, 2 * B * nkv * a.length * hd * es + 4 * B * T * nkv * hd * es + 2 * B * T * a.heads * hd * es
        + (8 * B * nkv * S if a.weights else 0))
    t = _time(lambda: cache_evict(kc, vc, w, pos, ls, ls, keep=a.keep, recent=a.keep // 4), a.iters)
    over = max(0, a.length - a.keep)
    moved = min(over, a.keep // 4) + max(0, over - a.keep // 4) * (a.keep - a.keep // 4) / max(1, a.length - a.keep // 4)
    say("evict", t, int(B * nkv * (16 * S + 4 * hd * es * moved)))
    tgt = torch.zeros(B, T, dtype=torch.long, device="cuda")
    t = _time(lambda: tree_commit(par, tgt, tgt, kc, vc, ls), a.iters)
    say("commit", t, 4 * hd * es * B * nkv * min(T - 1, a.depth if a.width else 0))
    return out


if __name__ == "__main__":
    main()
