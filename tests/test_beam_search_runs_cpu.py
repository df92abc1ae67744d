"""Searches with beams on the CPU, with the operators replaced by plain torch."""
import math

import pytest
import torch

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout, init_flat
from cme213_final_project_b200.config import ModelConfig
from cme213_final_project_b200.generate import Generator
from test_generate_runs_cpu import plain_append, plain_attention, plain_gemm, plain_layernorm

PROMPTS = [[1, 2, 3, 4, 5], list(range(20))]


def plain_beam_step(logits, scores, width=None, *, finished=None, allowed=None):
    B, n = scores.shape
    width, V = width or n, logits.shape[1]
    parents, tokens = torch.arange(width).remainder(n).expand(B, -1).clone(), torch.full((B, width), -1)
    out = torch.full((B, width), -math.inf)
    lp = logits.double().view(B, n, V)
    if allowed is not None:
        t = torch.arange(V)
        lp = lp.masked_fill((allowed[0, t // 32] >> t % 32) & 1 == 0, -math.inf)
    lp = scores.double()[..., None] + (lp - torch.logsumexp(lp, 2, keepdim=True))
    for b in range(B):
        found = []
        for i in range(n):
            if not math.isfinite(scores[b, i]):
                continue
            if finished is not None and finished[b, i]:
                found.append((-float(scores[b, i]), i, -1))
            elif bool(lp[b, i].isfinite().any()):
                found += [(-float(v), i, t) for t, v in enumerate(lp[b, i]) if v > -math.inf]
        for k, (v, i, t) in enumerate(sorted(found)[:width]):
            parents[b, k], tokens[b, k], out[b, k] = i, t, -v
    return parents.to(torch.int32), tokens.to(torch.int32), out


def plain_reorder(cache_k, cache_v, pages, spare, parents, lengths):
    B, n = parents.shape
    slots, table, new_spare = cache_k.shape[3], pages.clone(), spare.clone()
    old_k, old_v = cache_k.clone(), cache_v.clone()
    for b in range(B):
        full, rest = divmod(int(lengths[b]), slots)
        for i in range(n):
            own, of = b * n + i, b * n + int(parents[b, i])
            table[own, :full] = pages[of, :full]
            if rest and own != of:
                to = int(spare[own])
                assert to >= 0
                cache_k[:, to, :, :rest], cache_v[:, to, :, :rest] = (c[:, pages[of, full], :, :rest] for c in (old_k, old_v))
                table[own, full], new_spare[own] = to, pages[own, full]
    return table, new_spare


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    for name, f in (("add", torch.add), ("layernorm_fwd", plain_layernorm), ("gemm", plain_gemm), ("cache_append", plain_append),
                    ("paged_attention", plain_attention), ("beam_step", plain_beam_step), ("cache_reorder", plain_reorder)):
        monkeypatch.setattr(ops, name, f)


def generator(beams, **kw):
    cfg = ModelConfig(mode="gpt", vocab_size=33, seq_len=48, hidden=64, heads=2, ff=64, layers=2, batch_size=1, activation="gelu",
                      causal=True, head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg)
    return Generator(cfg, layout, init_flat(layout, 3) * 6.0, len(PROMPTS) * beams, page=8, beams=beams, **kw)


@pytest.mark.parametrize("beams", [2, 4])
@pytest.mark.parametrize("from_step", [1, 3, 5])
@pytest.mark.parametrize("token", [None, 1])
def test_places_that_lose_their_continuation_are_empty(beams, from_step, token, monkeypatch):
    """From some step on all logits are NaN, or those after one of the tokens that are common among the beams: a place that no beam takes says nothing."""
    g = generator(beams)
    clean, best = g.beam_search(PROMPTS, 8, cuda_graph=False)
    bad = token if token is None else int(clean[0, 0, from_step - 1])
    forward, calls = Generator.forward, [0]

    def broken(self, tokens, positions, offsets, lengths, last):
        logits = forward(self, tokens, positions, offsets, lengths, last)
        calls[0] += 1
        if calls[0] > from_step:                                       # (the first call is the prompts')
            logits = logits.masked_fill(torch.ones_like(tokens[last], dtype=torch.bool)[:, None] if bad is None else (tokens[last] == bad)[:, None],
                                        math.nan)
        return logits

    monkeypatch.setattr(Generator, "forward", broken)
    tokens, scores = g.beam_search(PROMPTS, 8, cuda_graph=False)
    empty = scores == -math.inf
    assert bool((tokens[empty] == -1).all()) and bool((tokens[~empty] >= 0).all())
    if bad is None:
        assert bool(empty.all())
    for row, score in zip(tokens[~empty].tolist(), scores[~empty].tolist()):
        assert math.isfinite(score) and bad not in row[from_step - 1:-1]


def test_few_tokens_at_first():
    """Fewer continuations than beams: the places fill up when there are more."""
    g = generator(4)
    tokens, scores = g.beam_search(PROMPTS, 1, allowed=[3, 7], cuda_graph=False)
    assert bool((scores[:, :2] > -math.inf).all()) and bool((scores[:, 2:] == -math.inf).all()) and bool((tokens[:, 2:] == -1).all())
    tokens, scores = g.beam_search(PROMPTS, 3, allowed=[3, 7], cuda_graph=False)
    assert bool((scores > -math.inf).all()) and set(tokens.unique().tolist()) == {3, 7}


@pytest.mark.parametrize("beams", [1, 2, 4])
def test_up_to_the_last_position_with_the_pages_of_the_default(beams):
    g = generator(beams)
    tokens, _ = g.beam_search([PROMPTS[0], [1] * 5], 48 - 5 + 1, cuda_graph=False)
    assert tokens.shape == (2, beams, 44) and bool((tokens >= 0).all())
    g.beam_search([PROMPTS[0], [1] * 48], 1, cuda_graph=False)                   # a prompt that fills it


def test_one_beam_is_a_run():
    """Of one beam the best continuation goes on, as in a run without sampling; it needs no spare page."""
    g = generator(1)
    tokens, scores = g.beam_search(PROMPTS, 9, cuda_graph=False)
    for row, p in zip(tokens[:, 0].tolist(), PROMPTS):
        one = generator(1)
        for t in row:
            assert int(one.prefill([p, [0]])[0].argmax()) == t
            p = p + [t]


def test_books_of_one_beam():
    g = generator(1)
    c = g.cache
    c.grow([9, 17])
    free = len(c.free)
    spare = c.fork(1, 8)
    assert spare.tolist() == [-1, -1] and len(c.free) == free - 2 and [len(o) for o in c.owned] == [3, 4]
    c.clear()
    assert c.forked([9, 17], 1, 8) == 7 and sorted(c.free) == list(range(c.k.shape[1]))
