"""A search with beams, and a cache of 8-bit integers, against the oracle model, which computes every sequence anew in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout, init_flat
from cme213_final_project_b200.config import ModelConfig
from cme213_final_project_b200.generate import CacheFull, Generator, Sampling, main
from cme213_final_project_b200.models.reference import forward

PROMPTS = [[1, 2, 3, 4, 5], list(range(40)), [(i * 7) % 65 for i in range(32)]]


def model(dtype, hidden=128, heads=4, layers=2, vocab=65, seq_len=96):
    cfg = ModelConfig(mode="gpt", vocab_size=vocab, seq_len=seq_len, hidden=hidden, heads=heads, ff=2 * hidden, layers=layers, batch_size=1,
                      activation="gelu", causal=True, head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg, align=64)
    flat = init_flat(layout, 3)
    flat *= 4.0                                            # (with the small weights of a fresh model all logits are nearly the same)
    return cfg, layout, flat.to(dtype).cuda()


def oracle(cfg, layout, params, tokens):
    """Logits after each token, in 64 bits."""
    P = {k: v.double().cpu() for k, v in layout.views(params).items()}
    one = ModelConfig(**{**cfg.__dict__, "seq_len": len(tokens)})
    P["pos_embed"] = P["pos_embed"][:len(tokens)]
    return forward(P, one, torch.tensor(tokens, dtype=torch.int32), None)[1]


def search(cfg, layout, params, prompt, n, steps, end, allowed):
    """[(score, tokens)] of the best n, each from scratch."""
    beams = [(0.0, [], False)]
    for _ in range(steps):
        found = []
        for i, (score, tokens, over) in enumerate(beams):
            if over:
                found.append((score, tokens, True))
                continue
            x = oracle(cfg, layout, params, prompt + tokens)[-1]
            if allowed is not None:
                hidden = torch.ones(len(x), dtype=torch.bool)
                hidden[allowed] = False
                x = x.masked_fill(hidden, -math.inf)
            lp = torch.log_softmax(x, 0)
            found += [(score + float(lp[t]), tokens + [t], t == end) for t in lp.topk(min(n, len(lp))).indices.tolist() if lp[t] > -math.inf]
        beams = sorted(found, key=lambda f: -f[0])[:n]
    return [(s, t) for s, t, _ in beams]


@pytest.mark.parametrize("beams,page,heads", [(1, 16, 4), (3, 8, 2), (4, 16, 1), (8, 16, 4)])
@pytest.mark.parametrize("end,allowed", [(None, None), (11, None), (7, [3, 7, 11, 19, 64])])
def test_the_beams_of_the_oracle(beams, page, heads, end, allowed):
    cfg, layout, params = model(torch.float32, heads=heads)
    gen = Generator(cfg, layout, params, len(PROMPTS) * beams, page=page, beams=beams)
    tokens, scores = gen.beam_search(PROMPTS, 12, end, allowed, chunk=13)
    for g, prompt in enumerate(PROMPTS):
        want = search(cfg, layout, params, prompt, beams, 12, end, allowed)
        for row, score, (w_score, w_tokens) in zip(tokens[g].tolist(), scores[g].tolist(), want):
            assert [t for t in row if t >= 0] == w_tokens
            assert abs(score - w_score) < 2e-3             # twelve logits, each off by some 1e-4 of a spread of one
    assert ops.attention_check_status() == 0 and ops.gemm_check_status() == 0


@pytest.mark.parametrize("dtype,cache8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, True)])
def test_a_search_is_what_its_steps_are(dtype, cache8):
    """With a CUDA graph or without, call after call; the scores are those of the tokens."""
    cfg, layout, params = model(dtype)
    gen = Generator(cfg, layout, params, len(PROMPTS) * 4, beams=4, cache8=cache8)
    runs = [gen.beam_search(PROMPTS, 20, end=9, cuda_graph=g) for g in (True, False, True)]
    for r in runs[1:]:
        assert torch.equal(runs[0][0], r[0]) and torch.equal(runs[0][1], r[1])
    tokens, scores = runs[0]
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    for prompt, found, best in zip(PROMPTS, tokens.tolist(), scores.tolist()):
        assert len({tuple(r) for r in found}) == 4
        for row, score in zip(found, best):
            row = [t for t in row if t >= 0]
            assert 9 not in row[:-1] and (len(row) == 20 or row[-1] == 9)
            logits = oracle(cfg, layout, params, prompt + row)[len(prompt) - 1:-1]
            lp = torch.log_softmax(logits, 1).gather(1, torch.tensor(row)[:, None]).sum()
            # as for a run without beams: a bf16 model's (or cache's) log-probabilities are off by up to a fifth of the logits' spread
            assert abs(float(lp) - score) <= 0.2 * float(logits.std()) * math.sqrt(len(row))
    by_length = gen.beam_search(PROMPTS, 20, end=9, length_power=1.0)
    rate = by_length[1] / (by_length[0] >= 0).sum(2)
    assert bool((rate[:, :-1] >= rate[:, 1:]).all())


def values(cache, b):
    """What an 8-bit cache holds of a sequence: keys and values ``[layers, positions, heads, head size]`` in 64 bits."""
    pages, n, out = cache.table[b][cache.table[b] >= 0].long(), cache.lengths[b], []
    for q, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x = q[:, pages].double() * s[:, pages].double().repeat_interleave(q.shape[3] // s.shape[3], 3)[..., None]
        out.append(x.transpose(2, 3).flatten(1, 2)[:, :n].cpu())
    return out


def last_logits(cfg, layout, params, token, cache, b):
    """Logits after a sequence's last token in 64 bits, its keys and values being those of the cache; and its own of the first layer."""
    P = {k: v.double().cpu() for k, v in layout.views(params).items()}
    keys, vals = values(cache, b)
    norm = lambda x, g, c: torch.nn.functional.layer_norm(x, x.shape[-1:], g, c, cfg.ln_eps)
    x, H, first = P["tok_embed"][token] + P["pos_embed"][cache.lengths[b] - 1], cfg.heads, None
    for l in range(cfg.layers):
        w = lambda name: P[f"h{l}.{name}"]
        q, k, v = (norm(x, w("ln1_gamma"), w("ln1_beta")) @ w("Wqkv")).view(3, H, -1)
        first = (k, v) if first is None else first
        p = torch.softmax(torch.einsum("hd,thd->ht", q, keys[l]) * cfg.head_dim ** -0.5, 1)
        x = x + torch.einsum("ht,thd->hd", p, vals[l]).flatten() @ w("Wo")
        h = norm(x, w("ln2_gamma"), w("ln2_beta")) @ w("W1") + w("b1")
        x = x + torch.nn.functional.gelu(h, approximate="tanh") @ w("W2") + w("b2")
    return norm(x, P["lnf_gamma"], P["lnf_beta"]) @ P["tok_embed"].T, first


def test_the_cache_in_8_bits():
    """Logits after prompts in chunks, against a model whose keys and values are those that the cache stands for: held to 1 % of their spread, as
    with a cache in fp32.  What the cache stands for is off by half a scale, and by as much for each later rounding in its block: chunks of 7
    come to a block of 16 slots in 4 calls at the most, and a scale only grows."""
    cfg, layout, params = model(torch.float32)
    gen = Generator(cfg, layout, params, len(PROMPTS), cache8=True)
    assert gen.cache.k.dtype == torch.int8 and gen.cache.k_scales.shape == (2, len(PROMPTS) * 6, 4, 1)
    for chunk in (512, 7):
        logits = gen.prefill(PROMPTS, chunk)
        for b, p in enumerate(PROMPTS):
            want, first = last_logits(cfg, layout, params, p[-1], gen.cache, b)
            assert float((logits[b].cpu().double() - want).abs().max()) < 0.01 * float(want.std())
            page = int(gen.cache.table[b, (len(p) - 1) // 16])
            for x, held, s in zip(first, values(gen.cache, b), (gen.cache.k_scales, gen.cache.v_scales)):
                step = s[0, page, :, 0].double().cpu()[:, None]
                assert bool(((held[0, -1] - x).abs() <= (0.5 if chunk > 40 else 2.0) * step * 1.001).all())
    # a run's picks are the best of such a model: the last of 2 to 12 tokens
    for n in (2, 5, 12):
        tokens, _ = gen.generate(PROMPTS, n)
        for b, row in enumerate(tokens.tolist()):
            want, _ = last_logits(cfg, layout, params, row[-2], gen.cache, b)
            assert float(want.max() - want[row[-1]]) < 0.02 * float(want.std())
    sampled = [gen.generate(PROMPTS, 12, Sampling(1.0), seed=s)[0] for s in (1, 1)]
    assert torch.equal(*sampled)


def test_a_search_then_a_run_then_a_search():
    cfg, layout, params = model(torch.bfloat16)
    gen = Generator(cfg, layout, params, 4, beams=2)
    first = gen.beam_search(PROMPTS[:2], 9)
    run = gen.generate(PROMPTS[:2] * 2, 9)
    again = gen.beam_search(PROMPTS[:2], 9)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert torch.equal(run[0][:2], run[0][2:])
    with pytest.raises(ValueError):
        gen.beam_search(PROMPTS, 9)
    assert gen.cache.shared
    assert torch.equal(gen.beam_search(PROMPTS[:2], 9)[0], first[0])


def test_pages_run_out():
    cfg, layout, params = model(torch.bfloat16)
    need = 0 + 4 * (2 - 0 + 1)                             # 5 + 19 tokens: no full page is shared, two pages and a spare one each
    assert Generator(cfg, layout, params, 4, pages=need, beams=4).beam_search(PROMPTS[:1], 20)[0].shape == (1, 4, 20)
    with pytest.raises(CacheFull):
        Generator(cfg, layout, params, 4, pages=need - 1, beams=4).beam_search(PROMPTS[:1], 20)
    shared = 2 + 4 * (3 - 2 + 1)                           # 32 + 8 tokens: two full pages are shared
    assert Generator(cfg, layout, params, 4, pages=shared, beams=4).beam_search([PROMPTS[2]], 9)[0].shape == (1, 4, 9)
    Generator(cfg, layout, params, 4, beams=4).beam_search(PROMPTS[:1], 92)      # up to the last position, with the default's pages


def test_commands(tmp_path, capsys):
    """A few steps on a text of one phrase, a checkpoint, and the phrase comes back: as the best beam, and out of 8 bits."""
    from cme213_final_project_b200.train import main as train
    text, ck = tmp_path / "text.txt", tmp_path / "model.ck"
    text.write_text("the quick brown fox jumps over the lazy dog. " * 400)
    assert train([str(text), "--preset", "tiny-gpt", "--epochs", "8", "--lr", "3e-3", "--save-checkpoint", str(ck)]) == 0
    capsys.readouterr()
    common = ["--checkpoint", str(ck), "--data", str(text), "--prompt", "the quick", "--prompt", "jumps over", "--max-new", "30"]
    assert main(common + ["--beams", "3", "--end", ".", "--cache-dtype", "int8"]) == 0
    out = capsys.readouterr().out
    assert out.count("log-probability") == 6 and "jumps over the lazy dog.\n" in out
    assert main(common + ["--temperature", "0", "--cache-dtype", "int8"]) == 0
    out = capsys.readouterr().out
    assert "the quick brown fox jumps over the" in out and "jumps over the lazy dog. the" in out
    for more in (["--beams", "33"], ["--beams", "2", "--temperature", "0.5"], ["--beams", "2", "--end", "the"], ["--end", "."], ["--beams", "2", "--end", "%"]):
        assert main(common + more) == 1
