"""Generation with drafted trees and a token budget against the model's own step-by-step decoding (CPU)."""
from types import SimpleNamespace

import pytest
import torch

import kv_cache_oracle as K
from sigma0_b200.infer.speculative import TreeDecoder, chain_tree, generate, lookup_drafts, main
from sigma0_b200.models.registry import build_model
from sigma0_b200.ops.kv_cache import KVCache, tree_mask


def _model(book=False, arch="transformer", seed=0):
    torch.manual_seed(seed)
    return build_model(SimpleNamespace(architecture=arch, d_model=32, n_heads=4, n_message_layers=1, n_layers=2, vocab_size=40,
                                        n_book_pre_layers=1, n_book_post_layers=1, d_book=13, use_book_data=book,
                                        token_mode="22tok", dtype="float32", impl="torch")).eval()


def _greedy(model, prompt, n, book):
    """One token at a time through the full forward."""
    toks = prompt
    for _ in range(n):
        rows = None if book is None else book.expand(-1, toks.shape[1], -1)
        with torch.no_grad():
            toks = torch.cat([toks, model(toks, rows)[:, -1].argmax(-1, keepdim=True)], 1)
    return toks[:, prompt.shape[1]:]


def _prompt(seed, B=3, L=30, vocab=40):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (B, 7), generator=g).repeat(1, L // 7 + 1)[:, :L]


@pytest.mark.parametrize("book", [False, True])
@pytest.mark.parametrize("depth,chunk", [(0, 512), (3, 512), (4, 11)])
def test_generation_is_greedy_decoding(book, depth, chunk):
    model = _model(book)
    prompt = _prompt(1)
    row = torch.randn(3, 1, 13, generator=torch.Generator().manual_seed(2)) if book else None
    want = _greedy(model, prompt, 25, row)
    got, steps = generate(TreeDecoder(model, 3, 90), prompt, 25, row, width=2, depth=depth, chunk=chunk)
    assert torch.equal(got, want)
    assert steps == 24 if depth == 0 else steps <= 24


def test_drafts_are_accepted():
    """A model that repeats its input accepts what it has said before: fewer steps than tokens."""
    model = _model(seed=3)
    prompt = _prompt(5, L=60)
    got, steps = generate(TreeDecoder(model, 3, 400), prompt, 120, width=2, depth=5)
    assert torch.equal(got, _greedy(model, prompt, 120, None))
    assert steps < 119


def test_tree_forward_is_the_forward_of_every_branch():
    model = _model()
    prompt = _prompt(7, B=2, L=9)
    dec = TreeDecoder(model, 2, 40)
    dec.prefill(prompt)
    g = torch.Generator().manual_seed(8)
    par = K.random_tree(7, g)
    mask = tree_mask(par)
    tokens = torch.randint(0, 40, (2, 7), generator=g)
    got = torch.log_softmax(dec.forward(tokens, mask=mask), -1)
    for i in range(7):
        branch = [j for j in range(7) if mask[i, j]]
        with torch.no_grad():
            want = model(torch.cat([prompt, tokens[:, branch]], 1))[:, -1]
        # float32 sums in another order through three layers: a few hundred roundings of values around 10
        assert (got[:, i] - want).abs().max() < 10 * 300 * K.U[torch.float32] * 10


def test_budget_keeps_the_caches_short():
    model = _model()
    prompt = _prompt(9, L=50)
    dec = TreeDecoder(model, 3, 40, budget=24, recent=8, sinks=2)
    got, _ = generate(dec, prompt, 30, width=2, depth=3, chunk=16)
    assert got.shape == (3, 30)
    for c in dec.caches:
        assert (c.lengths <= 24).all() and (c.seen >= 79).all()
        # the first and the latest tokens are there, in every layer and head
        live = c.positions.masked_fill(torch.arange(c.slots) >= c.lengths[:, None, None], -1)
        assert ((live == 0).any(-1) & (live == 1).any(-1)).all()
        for k in range(1, 9):
            assert (live == c.seen[:, None, None] - k).any(-1).all()
        assert (c.weight >= 0).all() and (c.weight.sum(-1) > 0).all()
    # a budget that is never reached changes nothing
    a, _ = generate(TreeDecoder(model, 3, 140, budget=100, recent=8), prompt, 20, width=2, depth=3)
    assert torch.equal(a, _greedy(model, prompt, 20, None))


def test_lookup_and_tree():
    h = torch.tensor([[5, 1, 2, 9, 1, 2, 7, 8, 1, 2, 0, 0], [1, 2, 3, 0, 0, 0, 0, 0, 0, 0, 0, 0]])
    d = lookup_drafts(h, torch.tensor([10, 3]), 2, 3)
    assert d.tolist() == [[7, 8, 1, 9, 1, 2], [-1] * 6]
    assert chain_tree(2, 3).tolist() == [-1, 0, 1, 2, 0, 4, 5] and chain_tree(2, 0).tolist() == [-1]


def test_refusals_and_command():
    with pytest.raises(ValueError):
        TreeDecoder(_model(arch="s5"), 1, 10)
    with pytest.raises(ValueError):
        KVCache(1, 1, 1, 10, 4, budget=11)
    with pytest.raises(ValueError):
        TreeDecoder(_model(), 1, 24, budget=24).prefill(torch.zeros(1, 4, dtype=torch.long))
    out = main(["--d_model", "16", "--n_layers", "1", "--n_heads", "2", "--vocab_size", "30", "--batch", "2", "--prompt", "44",
                "--tokens", "12", "--dtype", "float32", "--depth", "2"])
    assert set(out) == {"one_by_one", "drafted"} and out["drafted"]["steps"] <= out["one_by_one"]["steps"]
