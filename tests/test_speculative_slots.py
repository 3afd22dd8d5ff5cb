"""Generation over caches with too few slots is refused, over just enough of them it is greedy decoding."""
from types import SimpleNamespace

import pytest
import torch

from sigma0_b200.infer.speculative import TreeDecoder, generate
from sigma0_b200.models.registry import build_model


def _model(seed=3):
    torch.manual_seed(seed)
    return build_model(SimpleNamespace(architecture="transformer", d_model=32, n_heads=4, n_message_layers=1, n_layers=2, vocab_size=40,
                                        n_book_pre_layers=1, n_book_post_layers=1, d_book=13, use_book_data=False,
                                        token_mode="22tok", dtype="float32", impl="torch")).eval()


def _prompt(L, B=3):
    g = torch.Generator().manual_seed(5)
    return torch.randint(0, 40, (B, 7), generator=g).repeat(1, L // 7 + 1)[:, :L]


def _greedy(model, prompt, n):
    toks = prompt
    for _ in range(n):
        with torch.no_grad():
            toks = torch.cat([toks, model(toks, None)[:, -1].argmax(-1, keepdim=True)], 1)
    return toks[:, prompt.shape[1]:]


@pytest.mark.parametrize("depth", [0, 3, 5])
def test_just_enough_slots(depth):
    """prompt + tokens - 1 slots: the last steps' trees pass the end of the cache, the tokens stay the model's."""
    model, prompt = _model(), _prompt(30)
    got, _ = generate(TreeDecoder(model, 3, 30 + 40 - 1), prompt, 40, width=2, depth=depth)
    assert torch.equal(got, _greedy(model, prompt, 40))


@pytest.mark.parametrize("slots,budget,L,n", [(68, None, 30, 40), (29, None, 30, 1), (10, None, 30, 40), (34, 24, 30, 20),
                                               (26, 24, 60, 20), (36, 32, 60, 20)])
def test_too_few_slots(slots, budget, L, n):
    with pytest.raises(ValueError):
        generate(TreeDecoder(_model(), 3, slots, budget=budget), _prompt(L), n, width=2, depth=5)


def test_prefill_that_does_not_fit():
    dec = TreeDecoder(_model(), 3, 40)
    dec.prefill(_prompt(25))
    with pytest.raises(ValueError):
        dec.prefill(_prompt(16))
    dec.prefill(_prompt(15))
    with pytest.raises(ValueError):
        dec.prefill(_prompt(0))


def test_a_budget_that_is_not_reached_needs_no_slots_beyond_it():
    model, prompt = _model(), _prompt(30)
    got, _ = generate(TreeDecoder(model, 3, 60, budget=58, recent=8), prompt, 20, width=2, depth=5)
    assert torch.equal(got, _greedy(model, prompt, 20))


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [None, 40])
def test_prefill_can_be_captured(budget):
    """In a CUDA graph, where nothing can be read on the host: the replay does what the eager call does."""
    model, prompt = _model().cuda(), _prompt(90).cuda()
    runs = []
    for graphed in (False, True):
        dec = TreeDecoder(model, 3, 120, budget=budget, recent=8)
        state = [x for c in dec.caches for x in (c.k, c.v, c.lengths, c.seen, c.weight, c.positions) if x is not None]
        saved = [x.clone() for x in state]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            token = dec.prefill(prompt, chunk=30)
        torch.cuda.current_stream().wait_stream(st)
        if graphed:
            g = torch.cuda.CUDAGraph()
            for x, y in zip(state, saved):
                x.copy_(y)
            with torch.cuda.graph(g):
                token = dec.prefill(prompt, chunk=30)
            g.replay()
        torch.cuda.synchronize()
        runs.append([token] + [x.clone() for x in state])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
