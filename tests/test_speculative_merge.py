"""Drafts that begin alike share their nodes: the tree has no equal siblings, and the longest fitting draft is accepted."""
from types import SimpleNamespace

import pytest
import torch

from sigma0_b200.infer.speculative import TreeDecoder, chain_tree, generate, merged_tree
from sigma0_b200.models.registry import build_model
from sigma0_b200.ops.kv_cache import KVCache, tree_mask


def test_equal_beginnings():
    d = torch.tensor([[5, 6, 7, 5, 6, 8, 5, 9, 8], [1, 2, 3, 1, 2, 3, 4, 2, 3], [1, 2, 3, 4, 5, 6, -1, -1, -1]])
    par, mask, drafts = merged_tree(d, 3, 3)
    assert drafts.tolist() == [[5, 6, 7, -1, -1, 8, -1, 9, 8], [1, 2, 3, -1, -1, -1, 4, 2, 3], [1, 2, 3, 4, 5, 6, -1, -1, -1]]
    assert par.tolist() == [[-1, 0, 1, 2, 0, 1, 2, 0, 1, 8], [-1, 0, 1, 2, 0, 1, 2, 0, 7, 8], [-1, 0, 1, 2, 0, 4, 5, 0, 7, 8]]
    tree = tree_mask(par)
    live = torch.cat([torch.ones(3, 1, dtype=torch.bool), drafts >= 0], 1)
    assert torch.equal(mask[live], tree[live])
    assert torch.equal(mask.sum(-1) - 1, torch.tensor([0] + [1, 2, 3] * 3).expand(3, 10))   # every node's depth
    assert torch.equal(par[2], chain_tree(3, 3))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_longer_draft_behind_an_equal_first_token(dev):
    """Chains 7 1 1 and 7 5 6, the model says 7 5 6 2: three drafts are accepted, two of them the second chain's."""
    par, mask, drafts = merged_tree(torch.tensor([[7, 1, 1, 7, 5, 6]], device=dev), 2, 3)
    tokens = torch.cat([torch.tensor([[3]], device=dev), drafts], 1)
    says = {0: 7, 1: 5, 5: 6, 6: 2}
    targets = torch.tensor([[says.get(i, 9) for i in range(7)]], device=dev)
    c = KVCache(1, 1, 1, 16, 8, torch.float32, dev)
    x = torch.arange(7.0, device=dev)[None, :, None, None].expand(1, 7, 1, 8).contiguous()
    c.attend(0, x, x, x, mask)
    path, count, token = c.commit(par, tokens, targets)
    assert path.tolist() == [[0, 1, 5, 6, -1, -1, -1]] and count.tolist() == [4] and token.tolist() == [2]
    assert c.k[0, 0, 0, :4, 0].tolist() == [0, 1, 5, 6]


@pytest.mark.parametrize("width,depth", [(1, 4), (4, 3), (0, 3), (3, 0)])
def test_generation(width, depth):
    """Greedy decoding whatever the tree, and no more steps than with one draft."""
    torch.manual_seed(3)
    model = build_model(SimpleNamespace(architecture="transformer", d_model=32, n_heads=4, n_message_layers=1, n_layers=2, vocab_size=40,
                                        n_book_pre_layers=1, n_book_post_layers=1, d_book=13, use_book_data=False,
                                        token_mode="22tok", dtype="float32", impl="torch")).eval()
    prompt = torch.randint(0, 40, (3, 7), generator=torch.Generator().manual_seed(5)).repeat(1, 9)[:, :60]
    toks = prompt
    for _ in range(40):
        with torch.no_grad():
            toks = torch.cat([toks, model(toks, None)[:, -1].argmax(-1, keepdim=True)], 1)
    got, steps = generate(TreeDecoder(model, 3, 200), prompt, 40, width=width, depth=depth)
    assert torch.equal(got, toks[:, 60:])
    assert steps == 39 if not width * depth else steps <= 39
