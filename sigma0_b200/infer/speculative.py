"""Greedy generation of transformer stacks with drafted trees and a token budget.

A step of :class:`TreeDecoder` takes the last token and a tree of drafts through the whole model at
once, accepts the path that the model itself would have produced, and cuts the caches to
their budget (:mod:`sigma0_b200.ops.kv_cache`).  Without a budget the tokens are those of one-by-one
greedy decoding; drafts only change how many of them a step yields.  Drafts come from the
sequence itself: what followed the latest earlier occurrences of its last two tokens, which order
flow with its repeated message skeletons offers often.  Several of them often begin alike; they share
the nodes of what they have in common, so that the model's path is in the tree if one of them has it.

``python -m sigma0_b200.infer.speculative --help`` runs it on a random-init model.  The reference
generates one token per model call (``src/base_model/inference/generate.py:870-1061``).
"""
from __future__ import annotations

import argparse
import json
import time

import torch

from ..models.transformer import TransformerBlock
from ..ops.kv_cache import KVCache, check, tree_depth


class TreeDecoder:
    """Decoding state of a :class:`~sigma0_b200.models.lob_model.LobModel` whose mixers are all transformer blocks."""

    def __init__(self, model, batch, slots, budget=None, recent=0, sinks=0):
        self.model = model
        book = [] if not model.use_book_data else model.book_encoder.pre_layers + model.book_encoder.post_layers
        layers = model.message_encoder.layers + book + model.fused_s5.layers
        if not all(isinstance(l.seq, TransformerBlock) for l in layers):
            raise ValueError("decoding over a KV cache needs transformer blocks in every layer")
        dev = next(model.parameters()).device
        # layers of one head shape share a cache (the book's pre-layers are narrower than the others)
        shapes = {}
        for l in layers:
            shapes.setdefault((l.seq.nh, l.seq.hd, l.seq.compute_dtype), []).append(l.seq)
        self.caches, self.place = [], {}
        for (nh, hd, dtype), blocks in shapes.items():
            c = KVCache(len(blocks), batch, nh, slots, hd, dtype, dev, budget, recent, sinks)
            self.caches.append(c)
            for i, blk in enumerate(blocks):
                self.place[id(blk)] = (c, i)

    @property
    def seen(self):
        return self.caches[0].seen

    def _layers(self, layers, x, positions, mask):
        for l in layers:
            cache, i = self.place[id(l.seq)]
            x = l.seq.decode(x, lambda q, k, v, m: cache.attend(i, q, k, v, m), positions, mask)
        return x

    @torch.no_grad()
    def forward(self, tokens, book=None, mask=None):
        """Logits (B, T, vocab) of T new tokens (B, T); ``book`` (B, T or 1, d_book) rows.  The caches hold the
        new tokens behind their ends until ``add`` or ``commit`` says which stay."""
        m, T = self.model, tokens.shape[1]
        depth = torch.arange(T, device=tokens.device) if mask is None else tree_depth(mask)
        positions = self.seen[:, None] + depth
        x = self._layers(m.message_encoder.layers, m.message_encoder.encoder(tokens), positions, mask)
        if m.use_book_data:
            be = m.book_encoder
            xb = self._layers(be.pre_layers, book.expand(-1, T, -1).float(), positions, mask)
            xb = self._layers(be.post_layers, be._project(xb), positions, mask)
            x = torch.cat([x, xb.to(x.dtype)], -1)
        x = self._layers(m.fused_s5.layers, m.fused_s5._encode(x), positions, mask)
        return m.decoder(x).float()

    def add(self, n):
        for c in self.caches:
            c.add(n)

    def commit(self, parents, tokens, targets):
        res = [c.commit(parents, tokens, targets) for c in self.caches]
        return res[0]

    def trim(self):
        for c in self.caches:
            c.trim()

    def _need(self, new, nodes=0):
        """Raises where ``new`` tokens behind the cached ones do not fit, or a step of ``nodes`` beyond a budget that they reach."""
        c = self.caches[0]
        if c.lengths.is_cuda and torch.cuda.is_current_stream_capturing():
            return                                                        # nothing is known on the host
        rows = int(c.lengths.max()) + new
        if c.budget:
            rows = min(rows, c.budget + nodes)
        if rows > c.slots:
            raise ValueError(f"{rows} slots are needed, the caches have {c.slots}")

    def prefill(self, tokens, book=None, chunk=512):
        """The prompt (B, L) in causal chunks that fit between budget and slots -> the model's next token (B,).

        Without a budget the prompt must fit behind the cached tokens (their number is read on the host, but not in the
        capture of a CUDA graph)."""
        c = self.caches[0]
        if not tokens.shape[1]:
            raise ValueError("a prompt of at least one token")
        chunk = min(chunk, 1024, c.slots - (c.budget or 0) if c.budget else c.slots)
        if chunk < 1:
            raise ValueError("no slots beyond the budget")
        self._need(tokens.shape[1])
        for s in range(0, tokens.shape[1], chunk):
            part = tokens[:, s:s + chunk]
            rows = None if book is None else book if book.shape[1] == 1 else book[:, s:s + chunk]
            logits = self.forward(part, rows)
            self.add(part.shape[1])
            self.trim()
        return logits[:, -1].argmax(-1)


def lookup_drafts(history, length, width, depth):
    """Drafts (B, width * depth) from the sequences themselves: what followed the ``width`` latest earlier
    occurrences of the last two of ``length`` (B,) tokens of ``history`` (B, L); -1 where there is nothing."""
    B, L = history.shape
    at = torch.arange(L, device=history.device)
    a, b = (history.gather(1, (length[:, None] - k).clamp_min(0)) for k in (2, 1))
    hit = torch.zeros_like(history, dtype=torch.bool)
    hit[:, 1:] = (history[:, :-1] == a) & (history[:, 1:] == b) & (at[1:] < length[:, None] - 1)
    end = torch.where(hit, at, -1).topk(width, dim=1).values                    # (B, width), latest first
    pos = end[:, :, None] + 1 + torch.arange(depth, device=history.device)
    ok = (end[:, :, None] >= 0) & (pos < length[:, None, None])
    drafts = history.gather(1, pos.clamp(0, L - 1).reshape(B, -1)).reshape(B, width, depth)
    return torch.where(ok, drafts, -1).reshape(B, -1)


def chain_tree(width, depth, device=None):
    """Parents (int32) of a root with ``width`` chains of ``depth`` nodes below it."""
    par = [-1]
    for w in range(width):
        par += [0 if d == 0 else 1 + w * depth + d - 1 for d in range(depth)]
    return torch.tensor(par, dtype=torch.int32, device=device)


def merge_tables(batch, width, depth, device=None):
    """What :func:`merged_tree` needs beside the drafts, which a generation makes once."""
    at = torch.arange(depth, device=device)
    parents = chain_tree(width, depth, device).repeat(batch, 1)
    mask = torch.zeros(batch, parents.shape[1], parents.shape[1], dtype=torch.bool, device=device)
    mask[:, :, 0] = True
    return at + 1, at <= at[:, None], torch.arange(width, device=device)[:, None], parents, mask


def merged_tree(drafts, width, depth, tables=None):
    """The ``width`` chains of ``drafts`` (B, width * depth) with equal beginnings merged, as
    :func:`chain_tree` numbers their nodes -> (parents int32 (B, T), mask bool (B, T, T), drafts).

    A node that repeats a lower chain's up to there is left out: its draft becomes -1, which no model says, and what
    follows hangs below the lower chain's.  So no two children of a node carry the same token, and the walk of
    :func:`~sigma0_b200.ops.kv_cache.tree_commit` misses no longer path."""
    B = drafts.shape[0]
    place, upto, chain, parents, mask = tables or merge_tables(B, width, depth, drafts.device)
    d = drafts.reshape(B, width, depth)
    first = (d[:, :, None] == d[:, None]).cumprod(-1).argmax(2)           # the lowest chain that agrees up to here
    node = torch.add(place, first, alpha=depth)                           # the node that stands for (chain, depth)
    parents, mask = parents.clone(), mask.clone()
    parents[:, 1:].unflatten(1, (width, depth))[..., 1:] = node[..., :-1]
    up = torch.where(upto, node[:, :, None], 0)                           # those of a chain down to here; the root
    mask[:, 1:].scatter_(2, up.reshape(B, width * depth, depth), True)
    return parents, mask, torch.where(first == chain, d, -1).reshape(B, -1)


@torch.no_grad()
def generate(decoder: TreeDecoder, prompt, n, book=None, width=2, depth=6, chunk=512):
    """Greedy tokens (B, n) after ``prompt`` (B, L) and the steps that they took.

    ``book`` (B, 1, d_book): one row for all of the tokens.  ``depth`` 0: no drafts, one token a step.  The caches
    need a slot for each token of the prompt and of the result but the last, with a budget one for each of the
    budget and of a step's 1 + width * depth nodes; ValueError where they have fewer.  RuntimeError if an attention
    kernel gave up (:func:`sigma0_b200.ops.kv_cache.check`)."""
    B, L = prompt.shape
    dev = prompt.device
    nodes = 1 + width * depth
    decoder._need(L + max(n, 1) - 1, nodes)
    history = torch.zeros(B, L + n + nodes, dtype=torch.long, device=dev)
    history[:, :L] = prompt
    length = torch.full((B,), L, dtype=torch.long, device=dev)
    last = decoder.prefill(prompt, book, chunk)
    parents, mask = chain_tree(width, depth, dev), None                   # the root alone
    tables = merge_tables(B, width, depth, dev)
    history[:, L] = last
    length += 1
    steps, at = 0, torch.arange(nodes, device=dev)
    while int((length - L).min()) < n:
        drafts = history.new_zeros(B, 0)
        if nodes > 1:
            parents, mask, drafts = merged_tree(lookup_drafts(history, length, width, depth), width, depth, tables)
        tokens = torch.cat([last[:, None], drafts], 1)
        logits = decoder.forward(tokens.clamp_min(0), book, mask)
        targets = logits.argmax(-1)
        path, count, last = decoder.commit(parents, tokens, targets)
        decoder.trim()
        # what the path's nodes were continued with: the accepted drafts and the token after them
        new = targets.gather(1, path.long().clamp_min(0))
        slot = length[:, None] + at
        keep = (at < count[:, None]) & (slot < history.shape[1])
        slot = slot.clamp_max(history.shape[1] - 1)
        history.scatter_(1, slot, torch.where(keep, new, history.gather(1, slot)))
        # sequences that are done keep going (their tokens are cut off) until the slowest is
        length = torch.minimum(length + count, torch.full_like(length, history.shape[1] - nodes))
        steps += 1
    check(history)
    return history[:, L:L + n], steps


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--d_model", type=int, default=1024)
    p.add_argument("--n_layers", type=int, default=6)
    p.add_argument("--n_heads", type=int, default=16)
    p.add_argument("--vocab_size", type=int, default=2112)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt", type=int, default=2200)
    p.add_argument("--tokens", type=int, default=220)
    p.add_argument("--width", type=int, default=2)
    p.add_argument("--depth", type=int, default=6)
    p.add_argument("--budget", type=int, default=0, help="tokens kept per layer and head (0: all)")
    p.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    from types import SimpleNamespace
    from ..models.registry import build_model
    torch.manual_seed(a.seed)
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    model = build_model(SimpleNamespace(architecture="transformer", d_model=a.d_model, n_heads=a.n_heads,
                                         n_message_layers=1, n_layers=a.n_layers, vocab_size=a.vocab_size,
                                         use_book_data=False, token_mode="22tok", dtype=a.dtype, impl="torch"))
    model = model.to(dev).eval()
    # a repetitive prompt: message skeletons of 22 tokens
    msg = torch.randint(0, a.vocab_size, (a.batch, 22), device=dev)
    prompt = msg.repeat(1, a.prompt // 22 + 1)[:, :a.prompt]
    nodes = 1 + a.width * a.depth
    slots = (a.budget + 512 if a.budget else a.prompt + a.tokens + 2 * nodes) + nodes
    out = {}
    for name, depth in (("one_by_one", 0), ("drafted", a.depth)):
        for run in range(2):                                       # the first run warms up
            dec = TreeDecoder(model, a.batch, slots, a.budget or None, a.budget // 4, 4 if a.budget >= 16 else 0)
            if dev.type == "cuda":
                torch.cuda.synchronize()
            t = time.perf_counter()
            toks, steps = generate(dec, prompt, a.tokens, width=a.width, depth=depth)
            if dev.type == "cuda":
                torch.cuda.synchronize()
            t = time.perf_counter() - t
        out[name] = {"steps": steps, "tokens_per_s": round(a.batch * a.tokens / t, 1),
                     "tokens_per_step": round(a.tokens / steps, 2)}
    print(json.dumps(out))
    return out


if __name__ == "__main__":
    main()
