"""Drafted generation over the cache kernels: the tokens of step-by-step greedy decoding, a budget, a captured step."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dtype, d_model=256, n_heads=4, book=False):
    from sigma0_b200.models.registry import build_model
    torch.manual_seed(1)
    m = build_model(SimpleNamespace(architecture="transformer", d_model=d_model, n_heads=n_heads, n_message_layers=1, n_layers=2,
                                    n_book_pre_layers=1, n_book_post_layers=1, d_book=13, vocab_size=200, use_book_data=book,
                                    token_mode="22tok", dtype=dtype, impl="torch"))
    return m.cuda().eval()


def _prompt(B=3, L=300):
    g = torch.Generator().manual_seed(4)
    return torch.randint(0, 200, (B, 22), generator=g).repeat(1, L // 22 + 1)[:, :L].cuda()


@pytest.mark.parametrize("book", [False, True])
def test_drafted_generation_float32(book):
    """In float32 the drafted tokens are the model's own: its full forward over prompt and tokens says the same."""
    from sigma0_b200.infer.speculative import TreeDecoder, generate
    from sigma0_b200.ops import _ext
    model = _model("float32", book=book)
    prompt = _prompt()
    row = torch.randn(3, 1, 13, device="cuda") if book else None
    _ext.reset_launch_count()
    toks, steps = generate(TreeDecoder(model, 3, 400), prompt, 40, row, width=2, depth=6)
    assert _ext.launch_count() > 0 and steps <= 39
    seq = torch.cat([prompt, toks], 1)
    with torch.no_grad():
        lp = model(seq, None if row is None else row.expand(-1, seq.shape[1], -1))[:, prompt.shape[1] - 1:-1]
    # each token is the argmax up to what float32 sums in another order can change (values around 10)
    best, took = lp.max(-1).values, lp.gather(-1, toks[..., None])[..., 0]
    assert (best - took).max() < 1e-3


@pytest.mark.parametrize("heads", [4, 2])
def test_drafted_generation_bf16_with_a_budget(heads):
    from sigma0_b200.infer.speculative import TreeDecoder, generate
    model = _model("bfloat16", n_heads=heads)
    dec = TreeDecoder(model, 3, 400, budget=200, recent=64, sinks=4)
    toks, steps = generate(dec, _prompt(), 40, width=3, depth=6, chunk=128)
    assert toks.shape == (3, 40) and (toks >= 0).all() and (toks < 200).all()
    for c in dec.caches:
        assert (c.lengths <= 200).all()
        live = c.positions.masked_fill(torch.arange(c.slots, device="cuda") >= c.lengths[:, None, None], -1)
        for k in list(range(1, 65)):
            assert (live == c.seen[:, None, None] - k).any(-1).all()
        # the slots of a head hold different tokens
        srt = live.sort(-1).values
        assert ((srt[..., 1:] != srt[..., :-1]) | (srt[..., 1:] < 0)).all()


def test_decode_step_in_a_graph():
    """A captured step (forward, acceptance, trimming) follows the state on the device."""
    from sigma0_b200.infer.speculative import TreeDecoder, chain_tree
    from sigma0_b200.ops.kv_cache import tree_mask
    model = _model("bfloat16")
    prompt = _prompt()
    par = chain_tree(2, 3, "cuda")
    mask = tree_mask(par)
    runs = []
    for graphed in (False, True):
        dec = TreeDecoder(model, 3, 330, budget=280, recent=32, sinks=2)
        dec.prefill(prompt, chunk=40)
        tokens = torch.zeros(3, 7, dtype=torch.long, device="cuda")
        out = torch.zeros(3, dtype=torch.long, device="cuda")

        def step():
            targets = dec.forward(tokens, mask=mask).argmax(-1)
            out.copy_(dec.commit(par, tokens, targets)[2])
            dec.trim()
        saved = [x.clone() for c in dec.caches for x in (c.k, c.v, c.lengths, c.seen, c.weight, c.positions)]
        if graphed:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                step()
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
            for x, y in zip([x for c in dec.caches for x in (c.k, c.v, c.lengths, c.seen, c.weight, c.positions)], saved):
                x.copy_(y)
        got = []
        for k in range(6):
            tokens.copy_((torch.arange(21, device="cuda").reshape(3, 7) * (k + 3)) % 200)
            g.replay() if graphed else step()
            got += [out.clone(), dec.caches[0].lengths.clone()]
        torch.cuda.synchronize()
        runs.append(torch.stack(got))
    assert torch.equal(runs[0], runs[1])


def test_status_word_is_clear():
    from sigma0_b200.ops.kv_cache import status
    assert status(torch.zeros(1, device="cuda")) == 0


def test_bench_command():
    from sigma0_b200.eval.kv_bench import main
    out = main(["--batch", "2", "--heads", "4", "--kv_heads", "2", "--length", "300", "--keep", "64", "--width", "2", "--depth", "3",
                "--weights", "--iters", "2"])
    assert [r["op"] for r in out] == ["attention", "evict", "commit"] and all(r["us"] > 0 for r in out)
