"""A search with one beam up to the last position, and places without a continuation in a captured step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops
from cme213_final_project_b200.generate import Generator
from test_beam_search_gpu import PROMPTS, model


@pytest.mark.parametrize("dtype,cache8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_one_beam_up_to_the_last_position(dtype, cache8):
    """The most likely token every time, as in a run without sampling."""
    cfg, layout, params = model(dtype)
    gen = Generator(cfg, layout, params, 3, beams=1, cache8=cache8)
    prompts = [p[:5] for p in PROMPTS]
    tokens, scores = gen.beam_search(prompts, 92)
    assert tokens.shape == (3, 1, 92)
    run, logprobs = gen.generate(prompts, 92)
    assert torch.equal(tokens[:, 0], run)
    # sums of 92 log-probabilities, each rounded to 32 bits
    assert bool(((scores[:, 0] - logprobs.double().sum(1)).abs() <= 92 * 2 ** -23 * scores[:, 0].abs() + 92 * 1e-5).all())
    assert ops.attention_check_status() == 0 and ops.gemm_check_status() == 0


@pytest.mark.parametrize("cuda_graph", [True, False])
def test_places_that_lose_their_continuation_are_empty(cuda_graph, monkeypatch):
    cfg, layout, params = model(torch.bfloat16)
    gen = Generator(cfg, layout, params, 12, beams=4)
    clean, _ = gen.beam_search(PROMPTS, 10, cuda_graph=cuda_graph)
    bad = int(clean[0, 0, 6])
    forward = Generator.forward

    def broken(self, tokens, positions, offsets, lengths, last):
        logits = forward(self, tokens, positions, offsets, lengths, last)
        return logits.masked_fill((tokens[last] == bad)[:, None] & (positions[last] > 40)[:, None], math.nan)

    monkeypatch.setattr(Generator, "forward", broken)
    tokens, scores = gen.beam_search(PROMPTS, 10, cuda_graph=cuda_graph)
    empty = scores == -math.inf
    assert bool((tokens[empty] == -1).all()) and bool((tokens[~empty] >= 0).all()) and bool(scores[~empty].isfinite().all())
