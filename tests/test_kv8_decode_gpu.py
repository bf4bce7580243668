"""The 8-bit cache inside the cached Transformer decode, and scoring what it
generates: generate(mode="cached", kv="fp8") -> score(...), as a program uses them."""
import random

import numpy as np
import pytest
import torch

from oracle import kv8 as okv
from oracle import transformer as otr
from oracle.fill import REAL, TINY, grammar_tokens
from midiseq.config import Discretization, Grammar
from midiseq.generate import generate, score
from midiseq.loss import filtered_cross_entropy, filtered_logit, token_logprobs
from midiseq.mamba import Mamba
from midiseq.transformer import Transformer, TransformerConfig

pytestmark = pytest.mark.gpu
META = torch.tensor([[519, 279, 202, 202, 202, 178], [432, 277, 202, 202, 202, 173]])


def model(hp, precision, vocab=REAL, mv=568):
    cfg = TransformerConfig(vocab_size=vocab.size, metadata_vocab_size=mv, precision=precision, dropout=0.0, **hp)
    m = Transformer(cfg).to("cuda").eval()
    m.load_state_dict(otr.filled_params(otr.param_shapes(hp["n_embd"], hp["n_heads"], hp["n_layer"], hp["block_len"],
                                                         vocab.size, mv)))
    return m


def tokens(B, T, seed, vocab=REAL):
    g = np.random.default_rng(seed)
    return torch.from_numpy(np.stack([grammar_tokens(g, vocab, T) for _ in range(B)]))


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_step_attends_to_the_cache(precision):
    """Teacher-forced steps round a ring of 50: after each, the last layer's attention output equals
    the oracle's over what kv8_read returns; layer 0's keys and values (the same tokens' in both
    caches) equal the engine's own cache rounded: each off by half a step (2^-4 relative) or by half the smallest
    code (2^-10) of the block's scale, which is at most amax / 224."""
    hp = dict(n_embd=256, n_heads=2, n_layer=2, block_len=50)
    m = model(hp, precision)
    eng, B, T0, steps, ctx = m.engine, 2, 30, 35, 50
    toks, meta = tokens(B, T0 + steps, 1), META
    c8, c16 = eng.decode_cache(B, ctx, kv="fp8"), eng.decode_cache(B, ctx)
    with torch.no_grad():
        for c in (c8, c16):
            eng.forward(toks[:, :T0].cuda(), meta.cuda(), save=False, cache=c)
        R = eng.W["1.R"].double().cpu().numpy()  # (the bf16 copy is made by the first forward)
        for t in range(T0, T0 + steps):
            for c in (c16, c8):
                eng.step(toks[:, t].contiguous().cuda(), c)
            if t % 7 and t != ctx:
                continue
            q = c8.qkv.view(B, 3, 2, 128)[:, 0].double().cpu().numpy()
            k, v = (x.double().cpu().numpy() for x in c8.window_kv(1, torch.float32))
            assert k.shape[2] == 6 + min(t + 1, ctx)
            got = c8.o.view(B, 2, 128).double().cpu().numpy()
            for b in range(B):
                want = okv.attend(q[b], k[b], v[b], R, 256 ** -0.5)
                mag = np.abs(q[b]).max() * (np.abs(k[b]).max() + np.abs(R).max()) * 128 * 256 ** -0.5
                tol = 2 * np.abs(v[b]).max() * (136 * 2.0 ** -24 * mag + 2.0 ** -20) + 2.0 ** -8 * np.abs(want) * (precision == "bf16")
                off = float((np.abs(got[b] - want) / tol).max())
                assert off <= 1, (t, b, off)
            for x8, x16 in zip(c8.window_kv(0), c16.window_kv(0)):
                x8, x16 = x8.double(), x16.double()
                assert x8.shape == x16.shape
                assert ((x8 - x16).abs() <= 2.0 ** -4 * x16.abs() + 2.0 ** -10 * x16.abs().amax() / 224).all()


def test_graph_steps_equal_eager_steps():
    hp = dict(n_embd=256, n_heads=2, n_layer=2, block_len=64)
    m = model(hp, "bf16")
    eng, toks = m.engine, tokens(2, 100, 3)
    rows = []
    try:
        for graphs in (True, False):
            eng.step_graphs = graphs
            c = eng.decode_cache(2, 64, kv="fp8")
            with torch.no_grad():
                eng.forward(toks[:, :60].cuda(), META.cuda(), save=False, cache=c)
                rows.append(torch.stack([eng.step(toks[:, t].contiguous().cuda(), c).clone() for t in range(60, 100)]))
    finally:
        del eng.step_graphs
    assert torch.equal(rows[0], rows[1])


def test_generate_then_score():
    """The whole run: the prompt's first token equals the exact mode's, the rest are generated over the
    8-bit cache past the window's end; the rows are then scored: the mean of -logprob is the training
    loss, the given token never beats the best alternative, and a token's own alternative agrees."""
    vocab, mv = TINY, 10
    hp = dict(n_embd=64, n_heads=2, n_layer=2, block_len=24)
    m = model(hp, "fp32", vocab, mv)
    d = vocab.disc
    gr = Grammar(Discretization(**{k: d[k] for k in ("pitch", "channel", "dyn", "length", "time", "tempo")}))
    src, meta = tokens(3, 20, 9, vocab), torch.randint(0, mv, (3, 6), generator=torch.Generator().manual_seed(1))
    us = np.random.default_rng(2).random(3 * 30).tolist()

    def run(n, **kw):
        return generate(m, 24, src, meta, num_tokens=n, rng=random.Random(4), uniforms=iter(us), grammar=gr,
                        return_tensor=True, **kw)

    got = run(30, mode="cached", kv="fp8")
    assert got.shape == (3, 50) and torch.equal(got, run(30, mode="cached", kv="fp8"))
    assert torch.equal(got[:, :21], run(1))
    assert (0 <= got).all() and (got < vocab.size).all()
    rows = got[:, -25:]
    r = score(m, rows, meta, top=3, grammar=gr)
    assert r.logprob.shape == (3, 24) and r.top_ids.shape == (3, 24, 3)
    with torch.no_grad():
        logits = m(rows[:, :-1].contiguous(), meta.cuda())
        loss = filtered_cross_entropy(rows[:, :-1].contiguous(), logits, rows[:, 1:].contiguous(), gr)
    # two fp32 evaluations of the mean of 72 terms of some units
    assert abs(loss.item() + r.logprob.mean().item()) < 1e-5 * max(1.0, loss.item())
    assert (r.logprob <= r.top_logprobs[..., 0] + 1e-6).all()
    hit = r.top_ids == rows[:, 1:, None]
    assert torch.equal(r.top_logprobs[hit], r.logprob[..., None].expand_as(hit)[hit])
    assert (r.entropy >= 0).all() and (r.entropy <= np.log(vocab.size) + 1e-5).all()


def test_score_has_a_gradient():
    """-mean(logprob) through filtered_logit and the model: the gradient of filtered_cross_entropy."""
    vocab, mv = TINY, 10
    hp = dict(n_embd=64, n_heads=2, n_layer=1, block_len=24)
    m = model(hp, "fp32", vocab, mv)
    d = vocab.disc
    gr = Grammar(Discretization(**{k: d[k] for k in ("pitch", "channel", "dyn", "length", "time", "tempo")}))
    w, meta = tokens(2, 25, 4, vocab).cuda(), torch.zeros(2, 6, dtype=torch.int64, device="cuda")
    src, trg = w[:, :-1].contiguous(), w[:, 1:].contiguous()
    grads = []
    for own in (True, False):
        logits = m(src, meta)
        loss = -token_logprobs(filtered_logit(src, logits, gr), trg).logprob.mean() if own else \
            filtered_cross_entropy(src, logits, trg, gr)
        (g,) = torch.autograd.grad(loss, m.flat)
        grads.append(g)
    # fp32 on both sides, sums of some hundred terms: well within 1e-4 of the largest
    assert ((grads[0] - grads[1]).abs().max() <= 1e-4 * grads[1].abs().max()).item()


def test_score_of_a_mamba_model():
    vocab, mv = TINY, 10
    m = Mamba(d_model=128, n_layers=2, vocab_size=vocab.size, metadata_vocab_size=mv, precision="fp32").to("cuda").eval()
    d = vocab.disc
    gr = Grammar(Discretization(**{k: d[k] for k in ("pitch", "channel", "dyn", "length", "time", "tempo")}))
    w, meta = tokens(2, 40, 6, vocab), torch.zeros(2, 6, dtype=torch.int64)
    r = score(m, w, meta, grammar=gr)
    with torch.no_grad():
        logits = m(w[:, :-1].contiguous().cuda(), meta.cuda())
        loss = filtered_cross_entropy(w[:, :-1].contiguous().cuda(), logits, w[:, 1:].contiguous().cuda(), gr)
    assert r.top_ids is None and abs(loss.item() + r.logprob.mean().item()) < 1e-5 * max(1.0, loss.item())
    with pytest.raises(ValueError, match="Transformer"):
        generate(m, 24, w, meta, num_tokens=1, mode="cached", kv="fp8")


def test_refusals():
    m = model(dict(n_embd=64, n_heads=2, n_layer=1, block_len=24), "fp32", TINY, 10)
    src, meta = tokens(1, 8, 1, TINY), torch.zeros(1, 6, dtype=torch.int64)
    with pytest.raises(ValueError, match="cached"):
        generate(m, 24, src, meta, num_tokens=1, kv="fp8")
    with pytest.raises(ValueError, match="fp8"):
        generate(m, 24, src, meta, num_tokens=1, mode="cached", kv="int8")
    with pytest.raises(ValueError, match="two tokens"):
        score(m, src[:, :1], meta)
    with pytest.raises(ValueError, match="head size"):
        model(dict(n_embd=24, n_heads=2, n_layer=1, block_len=24), "fp32", TINY, 10).engine.decode_cache(1, 24, kv="fp8")


@pytest.mark.parametrize("kv", [None, "fp8"])
def test_a_refused_prefill_leaves_the_cache(kv):
    """A prompt that the cache cannot hold is refused before a key of it is written: the next step is
    what it would have been."""
    hp = dict(n_embd=64, n_heads=2, n_layer=2, block_len=40)
    m = model(hp, "fp32", TINY, 10)
    eng, toks, meta = m.engine, tokens(2, 40, 8, TINY).cuda(), torch.zeros(2, 6, dtype=torch.int64, device="cuda")
    rows = []
    with torch.no_grad():
        for disturbed in (False, True):
            c = eng.decode_cache(2, 20, kv)
            eng.forward(toks[:, :20], meta, save=False, cache=c)
            if disturbed:
                with pytest.raises(ValueError, match="prefill"):
                    eng.forward(toks[:, 5:30], meta, save=False, cache=c)
                with pytest.raises(RuntimeError, match="size"):  # three rows for two
                    eng.forward(toks[[0, 1, 0], 1:21], meta[[0, 1, 0]], save=False, cache=c)
            rows.append(torch.stack([eng.step(toks[:, t].contiguous(), c).clone() for t in range(20, 24)]))
    assert torch.equal(rows[0], rows[1])


@pytest.mark.parametrize("kv", [None, "fp8"])
def test_one_prompt_for_all_rows(kv):
    """One prompt prefills every row of a cache."""
    hp = dict(n_embd=64, n_heads=2, n_layer=2, block_len=40)
    m = model(hp, "fp32", TINY, 10)
    eng, toks, meta = m.engine, tokens(1, 24, 8, TINY).cuda(), torch.zeros(3, 6, dtype=torch.int64, device="cuda")
    rows = []
    with torch.no_grad():
        for n in (1, 3):
            c = eng.decode_cache(3, 30, kv)
            eng.forward(toks[:, :20].expand(n, 20), meta[:n], save=False, cache=c)
            rows.append(torch.stack([eng.step(toks[:, t].expand(3).contiguous(), c).clone() for t in range(20, 24)]))
    assert torch.equal(rows[0], rows[1])


def test_score_in_a_graph():
    """Captured, the ids are not looked at; replays over other rows equal the eager calls."""
    m = model(dict(n_embd=64, n_heads=2, n_layer=2, block_len=24), "fp32", TINY, 10)
    d = TINY.disc
    gr = Grammar(Discretization(**{k: d[k] for k in ("pitch", "channel", "dyn", "length", "time", "tempo")}))
    sets = [tokens(3, 25, s, TINY).cuda() for s in range(5)]
    rows, meta = sets[0].clone(), torch.zeros(3, 6, dtype=torch.int64, device="cuda")
    score(m, rows, meta, 2, gr)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = score(m, rows, meta, 2, gr)
    for s in sets:
        rows.copy_(s)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, score(m, s, meta, 2, gr)):
            assert torch.equal(a, b)
